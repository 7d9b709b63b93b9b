// Gated scan: the diagonal gated linear recurrence
//
//   h_t = e^{g_t} h_{t-1} + s_t x_t        s_t = 1, or 1 - e^{g_t} (complement)
//
// per channel of [B][T][C] (or of packed sequences), and its adjoint
//
//   l_t = dh_t + e^{g_{t+1}} l_{t+1},  dx_t = s_t l_t,
//   dg_t = e^{g_t} (h_{t-1} [- x_t]) l_t,  dstate = e^{g_0} l_0.
//
// Both are bound by HBM with the issue rate close behind (some twenty
// instructions for 8 to 14 bytes a value): a forward reads x and g and writes
// h, a backward reads x, g and dh and writes dx and dg.  So each value is
// read once and its decay computed once, between the load and the store, in
// packed pairs of channels: a warp holds RUN tokens of 64 channels in
// registers, reduces them to the affine map c -> A c + H of the run, the maps of
// a block's runs are joined through shared memory, and the block walks its
// channels' time axis, the loads of the next step in flight meanwhile.  8 x 4096
// x 2048, bf16 x and f32 g: 101 us forward and 151 us backward, 81 % and 95 % of
// what a copy of as many bytes reaches.
//
// With few chains (sequences times sets of channels) the time axis is cut
// into segments as well: a first launch reduces every segment to its map, the
// second starts each segment from the maps before it.  That reads the inputs
// twice, and pays below about 80 chains, where one block each would leave the
// memory system idle.  The first launch walks its segments against the
// direction of the scan: it ends where the second begins, so L2 still holds
// that part of the inputs, and it stops at a packed sequence's boundary, since
// nothing passes it.  The joining order is fixed by the sizes: results do not
// depend on timing.  1 x 65536 x 1024 bf16: 63 + 84 us forward, 58 + 126 us
// backward, where a copy of every input and output once would take 125 us.
#pragma once

#include <cfloat>
#include <type_traits>

#include "sequence.cuh"

namespace gdn2 {

static_assert(RUN == 16, "the spacing of the states a backward starts from is part of the interface");
constexpr int MAX_SEGMENTS = 128;

struct ScanParams {
  int B, T, C;      // dense: B sequences of T; packed: N sequences in T rows
  int sets;         // sets of 64 channels
  int steps;        // tiles of a segment
  int segments;
  const int* cu;
  DView x, g, h;    // forward: h out.  backward: h = dh
  DView dx, dg;
  const float* state_in;
  float* state_out;
  const float* d_state_out;
  float* d_state_in;
  float* carry;     // [B or 1][ceil(T / RUN)][C]: state before every RUN-th token
  ulonglong2* maps; // [chain][segment][32 lanes] maps of the segments, or null (one segment)
  int* map_cuts;    // [chain][segment]: a sequence begins (adjoint: ends) in the segment
};

// Bytes of a run's staged rows, and blocks that an SM holds: by their shared
// memory, and by registers 16 warps of a forward (128 a thread) and 12 of a
// backward (168).
template <typename TX, typename TG, RowMode MODE>
constexpr int stage_bytes(bool bwd) {
  return (bwd ? 2 : 1) * Rows<TX, MODE>::BYTES + Rows<TG, MODE>::BYTES;
}
template <typename TX, typename TG, RowMode MODE>
constexpr int resident_blocks(int warps, bool bwd) {
  const int smem = warps * (STAGES * stage_bytes<TX, TG, MODE>(bwd) + 1040) + 1024;
  const int by_smem = 227 * 1024 / smem, by_regs = (bwd ? 12 : 16) / warps;
  return by_smem < by_regs ? by_smem : by_regs;
}

// The maps of a step's runs, twice for alternating steps.  cut: a sequence
// begins (adjoint: ends) in the run, so that nothing from before it comes
// through, not even an infinity or NaN times zero.
template <int NW>
struct ScanMaps {
  ulonglong2 run[2][NW][32];  // (A, H) pairs
  int cut[2][NW];
};

// A span's map of the state before it.  A state of zero stays out of the
// product, which growth (g > 0) may have taken to infinity.
__device__ __forceinline__ f32x2 through(f32x2 A, f32x2 c, f32x2 H) {
  float c0, c1, h0, h1, v0, v1;
  f2un(c, c0, c1);
  f2un(H, h0, h1);
  f2un(f2fma(A, c, H), v0, v1);
  return f2pk(c0 == 0.f ? h0 : v0, c1 == 0.f ? h1 : v1);
}

__device__ __forceinline__ bool not_number(f32x2 v) {
  float v0, v1;
  f2un(v, v0, v1);
  return v0 != v0 || v1 != v1;
}

// Product of the decays of two neighbouring spans.  A reset leaves zero beside
// growth beyond f32 as well: a state that it cut off has nothing to grow from.
__device__ __forceinline__ f32x2 chained(f32x2 a, f32x2 b) {
  const f32x2 v = f2mul(a, b);
  if (!not_number(v)) return v;
  float v0, v1, s0, s1;
  f2un(v, v0, v1);
  f2un(f2add(a, b), s0, s1);  // NaN where a factor is: both are at least 0
  return f2pk(v0 != v0 && s0 == s0 ? 0.f : v0, v1 != v1 && s1 == s1 ? 0.f : v1);
}

// The same of a segment's tiles, the latest one's runs being in `sh` and their
// product `tile`; a product of all that is a number has met no such pair.
template <int NW>
__device__ __forceinline__ f32x2 chained(const ScanMaps<NW>& sh, int buf, int lane, f32x2 all, f32x2 tile) {
  const f32x2 v = f2mul(all, tile);
  if (!not_number(v)) return v;
  #pragma unroll 1
  for (int w = 0; w < NW; ++w) all = chained(all, sh.run[buf][w][lane].x);
  return all;
}

// e c + in for an e = e^g (or 1 - e^g) that may be beyond f32 although g is
// not: nothing grows out of nothing.  SURE: e is a number.
template <bool SURE>
__device__ __forceinline__ f32x2 grow(f32x2 e, f32x2 g, f32x2 c, f32x2 in) {
  const f32x2 v = f2fma(e, c, in);
  if (SURE) return v;
  float g0, g1, c0, c1, i0, i1, v0, v1;
  f2un(g, g0, g1);
  f2un(c, c0, c1);
  f2un(in, i0, i1);
  f2un(v, v0, v1);
  return f2pk(c0 == 0.f && g0 <= FLT_MAX ? i0 : v0, c1 == 0.f && g1 <= FLT_MAX ? i1 : v1);
}
template <bool SURE>
__device__ __forceinline__ f32x2 grow(f32x2 e, f32x2 g, f32x2 c) {
  return SURE ? f2mul(e, c) : grow<false>(e, g, c, f2pk(0.f, 0.f));
}

// From the state `c` before the step's first token (after its last, in the
// adjoint), the state before this warp's run; c becomes the state after the
// step, and the maps join to `A` of the whole (with SUM).  wild: a product of
// the step is beyond f32.
template <int NW, bool PACKED, bool SUM>
__device__ __forceinline__ f32x2 join(ScanMaps<NW>& sh, int buf, int warp, int lane, f32x2 A, f32x2 H, bool cut,
                                      f32x2& c, f32x2& all, bool& any_cut, bool& wild) {
  float a0, a1;
  f2un(A, a0, a1);
  sh.run[buf][warp][lane] = make_ulonglong2(A, H);
  if (PACKED && lane == 0) sh.cut[buf][warp] = cut;
  wild = __syncthreads_or(!(a0 <= FLT_MAX && a1 <= FLT_MAX));
  f32x2 cin = c;
  #pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w == warp) cin = c;
    const ulonglong2 m = sh.run[buf][w][lane];
    const bool stop = PACKED && sh.cut[buf][w];
    c = stop ? m.y : wild ? through(m.x, c, m.y) : f2fma(m.x, c, m.y);
    if (SUM) {
      all = f2mul(all, m.x);
      any_cut |= stop;
    }
  }
  return cin;
}

// Decays of a run: a = e^g, and k = 1 - e^g where it is wanted.  False where
// some |g| is beyond the range of exp_pair: a reset (-inf), a decay below
// every f32, or growth.
template <bool COMP, typename View>
__device__ __forceinline__ bool decays(const View& rows, f32x2 (&a)[RUN], f32x2 (&k)[RUN]) {
  float far = 0.f;
  #pragma unroll
  for (int i = 0; i < RUN; ++i) {
    const f32x2 g = rows.get(i);
    float g0, g1;
    f2un(g, g0, g1);
    far = fmaxf(far, fmaxf(fabsf(g0), fabsf(g1)));
    exp_pair<COMP>(g, a[i], k[i]);
  }
  return __all_sync(0xffffffffu, far <= kExpRange);
}
// One token's, any g.
template <bool COMP>
__device__ __forceinline__ void decay_any(f32x2 g, f32x2& a, f32x2& k) {
  float v[2], e[2], m[2];
  f2un(g, v[0], v[1]);
  exp_pair<COMP>(g, a, k);
  f2un(a, e[0], e[1]);
  if (COMP) f2un(k, m[0], m[1]);
  #pragma unroll
  for (int i = 0; i < 2; ++i)
    if (fabsf(v[i]) > kExpRange) {
      e[i] = expf(v[i]);
      m[i] = -expm1f(v[i]);
    }
  a = f2pk(e[0], e[1]);
  if (COMP) k = f2pk(m[0], m[1]);
}

// Which of a run's tokens open or close a sequence or lie in one, one bit a
// token; seq: in lane i the sequence of token i, -1 outside (sequence(i): for all lanes).
constexpr unsigned ALL = (1u << RUN) - 1;
struct RunMasks {
  unsigned start, last, valid;
  int seq;
  __device__ __forceinline__ int sequence(int i) const { return __shfl_sync(0xffffffffu, seq, i); }
};
// The packed sequence on the far side (token SIDE) of a warp's latest run;
// most runs lie in that of the run before, and need no search.
template <int SIDE>
struct SequenceCursor {
  int n = -1, from = 0, to = 0;
  __device__ __forceinline__ RunMasks masks(const int* __restrict__ cu, int N, int T, int t0, int lane) {
    RunMasks k;
    if (n >= 0 && t0 >= from && t0 + RUN <= to) {
      k.start = t0 == from;
      k.last = t0 + RUN == to ? 1u << (RUN - 1) : 0u;
      k.valid = ALL;
      k.seq = n;
      return k;
    }
    const int t = t0 + lane;
    int first = 0, end = 0;
    k.seq = -1;
    if (lane < RUN && t < T) {
      k.seq = find_sequence(cu, N, t);
      if (k.seq >= 0) {
        first = __ldg(cu + k.seq);
        end = __ldg(cu + k.seq + 1);
        if (end > T) end = T;
      }
    }
    k.start = __ballot_sync(0xffffffffu, k.seq >= 0 && first == t);
    k.last = __ballot_sync(0xffffffffu, k.seq >= 0 && end == t + 1);
    k.valid = __ballot_sync(0xffffffffu, k.seq >= 0);
    n = __shfl_sync(0xffffffffu, k.seq, SIDE);
    from = __shfl_sync(0xffffffffu, first, SIDE);
    to = __shfl_sync(0xffffffffu, end, SIDE);
    return k;
  }
};

// Empty sequences hand their state (its gradient) through.
template <RowMode MODE>
__device__ __forceinline__ void pass_empty(const ScanParams& p, const float* from, float* to, const Pair<MODE>& ch, int base) {
  const int lane = threadIdx.x & 31;
  for (int n0 = (int)threadIdx.x - lane; n0 < p.B; n0 += blockDim.x) {
    const int n = n0 + lane;
    unsigned empty = __ballot_sync(0xffffffffu, n < p.B && is_empty(p.cu, n, p.T));
    while (empty) {
      const int64_t at = (int64_t)(n0 + __ffs(empty) - 1) * p.C + base;
      empty &= empty - 1;
      if (ch.on0) ch.store_state(to + at, from ? ch.load(from + at) : f2pk(0.f, 0.f));
    }
  }
}

// The state before segment `seg` (adjoint: after it): `c` through the maps of
// the segments before (after) it.
template <bool PACKED>
__device__ __forceinline__ f32x2 through_segments(const ScanParams& p, int64_t chain, int seg, int lane, f32x2 c) {
  const ulonglong2* m = p.maps + chain * p.segments * 32 + lane;
  const int* cut = p.map_cuts + chain * p.segments;
  #pragma unroll 8
  for (int s = 0; s < seg; ++s) {
    const ulonglong2 v = m[s * 32];
    c = PACKED && cut[s] ? v.y : through(v.x, c, v.y);
  }
  return c;
}
template <bool PACKED>
__device__ __forceinline__ void write_map(const ScanParams& p, int64_t chain, int seg, f32x2 A, f32x2 H, bool cut) {
  if (threadIdx.x < 32) p.maps[(chain * p.segments + seg) * 32 + threadIdx.x] = make_ulonglong2(A, H);
  if (PACKED && threadIdx.x == 0) p.map_cuts[chain * p.segments + seg] = cut;
}

// MAPS: only the segment's map, for the first of two launches.
template <typename TX, typename TG, RowMode MODE, int NW, bool COMP, bool PACKED, bool MAPS>
__global__ void __launch_bounds__(32 * NW, resident_blocks<TX, TG, MODE>(NW, false)) k_scan_fwd(const ScanParams p) {
  typedef Rows<TX, MODE> RX;
  typedef Rows<TG, MODE> RG;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ ScanMaps<NW> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seg = (int)(blockIdx.x % p.segments);
  const int64_t chain = blockIdx.x / p.segments;
  const int b = PACKED ? 0 : (int)(chain / p.sets);
  const int base = (int)(chain % p.sets) * SET;
  const Pair<MODE> ch(lane, p.C - base);
  const TX* x = static_cast<const TX*>(p.x.p) + b * p.x.s0 + base;
  const TG* g = static_cast<const TG*>(p.g.p) + b * p.g.s0 + base;
  TX* h = static_cast<TX*>(const_cast<void*>(p.h.p)) + b * p.h.s0 + base;
  const int runs = (p.T + RUN - 1) / RUN;

  if (PACKED && !MAPS && p.state_out && seg == 0) pass_empty(p, p.state_in, p.state_out, ch, base);
  if (!p.steps) return;
  f32x2 c = f2pk(0.f, 0.f), all = f2pk(1.f, 1.f);
  bool any_cut = false;
  if (!MAPS) {
    if (!PACKED && p.state_in) c = ch.load(p.state_in + (int64_t)b * p.C + base);
    if (p.maps) c = through_segments<PACKED>(p, chain, seg, lane, c);
  }

  constexpr int STAGE = RX::BYTES + RG::BYTES;
  auto stage = [&](int step) { return smem + ((step % STAGES) * NW + warp) * STAGE; };
  auto run_at = [&](int step) { return ((seg * p.steps + (MAPS ? p.steps - 1 - step : step)) * NW + warp) * RUN; };
  auto fetch = [&](int step) {
    if (step < p.steps) {
      RX{stage(step)}.fetch(x, p.x.s1, run_at(step), p.T, p.C - base, lane);
      RG{stage(step) + RX::BYTES}.fetch(g, p.g.s1, run_at(step), p.T, p.C - base, lane);
    }
    cp_async_commit();
  };
  SequenceCursor<MAPS ? 0 : RUN - 1> cursor;
  for (int step = 0; step < STAGES - 1; ++step) fetch(step);
  for (int step = 0; step < p.steps; ++step) {
    __syncwarp();
    fetch(step + STAGES - 1);
    const int t0 = run_at(step);
    RunMasks k{0, 0, ALL, 0};
    if (PACKED) k = cursor.masks(p.cu, p.B, p.T, t0, lane);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const auto xs = RX{stage(step)}.view(x, p.x.s1, t0, lane);
    const auto gs = RG{stage(step) + RX::BYTES}.view(g, p.g.s1, t0, lane);
    const unsigned cuts = PACKED ? (k.start | ~k.valid) & ALL : 0;
    TX* out = h + (int64_t)t0 * p.h.s1;
    float* carry = p.carry + (b * (int64_t)runs + t0 / RUN) * p.C + base;

    // a[i]: product of the decays up to token i, u[i]: the state there from a zero one before the run
    f32x2 a[RUN], u[RUN], A = f2pk(1.f, 1.f), H = f2pk(0.f, 0.f);
    f32x2 la[RUN], lu[RUN];  // the same token by token, where a decay is out of range
    bool cut = false;
    const bool plain = decays<COMP>(gs, a, u);
    if (plain && !cuts) {
      #pragma unroll
      for (int i = 0; i < RUN; ++i) {
        const f32x2 in = COMP ? f2mul(u[i], xs.get(i)) : xs.get(i);
        H = f2fma(a[i], H, in);
        A = f2mul(A, a[i]);
        a[i] = A;
        u[i] = H;
      }
    } else {
      auto token = [&](auto sure, int i, f32x2 g, f32x2 e, f32x2 r, f32x2& product, f32x2& state) {
        constexpr bool SURE = decltype(sure)::value;
        const f32x2 in = COMP ? grow<SURE>(r, g, xs.get(i)) : xs.get(i);
        if (PACKED && ((cuts >> i) & 1)) {
          const int n = k.sequence(i);
          cut = true;
          H = f2pk(0.f, 0.f);
          if ((k.start >> i) & 1) {
            if (p.state_in) H = ch.load(p.state_in + (int64_t)n * p.C + base);
            H = grow<SURE>(e, g, H, in);
          }
        } else {
          H = grow<SURE>(e, g, H, in);
          if (!cut) A = SURE ? f2mul(A, e) : chained(A, e);
        }
        product = A;
        state = H;
      };
      if (PACKED && plain) {
        #pragma unroll
        for (int i = 0; i < RUN; ++i) token(std::true_type(), i, a[i], a[i], u[i], a[i], u[i]);
      } else {
        #pragma unroll 1
        for (int i = 0; i < RUN; ++i) {
          f32x2 e, r;
          const f32x2 g = gs.get(i);
          decay_any<COMP>(g, e, r);
          token(std::false_type(), i, g, e, r, la[i], lu[i]);
        }
      }
    }
    f32x2 tile = f2pk(1.f, 1.f), before = f2pk(0.f, 0.f);
    bool wild;
    const f32x2 cin = join<NW, PACKED, MAPS>(sh, step & 1, warp, lane, A, H, cut, MAPS ? before : c, tile, any_cut, wild);
    if (MAPS) {  // this tile, then those behind it
      c = through(all, before, c);
      all = chained(sh, step & 1, lane, all, tile);
      if (PACKED && any_cut) break;
      continue;
    }
    if (p.carry && ch.on0 && t0 < p.T) ch.store_state(carry, cin);
    const int first_cut = cuts ? __ffs(cuts) - 1 : RUN;
    if (plain) {
      if (wild) {  // see through()
        float a0, a1, c0, c1;
        f2un(cin, c0, c1);
        #pragma unroll
        for (int i = 0; i < RUN; ++i) {
          f2un(a[i], a0, a1);
          a[i] = f2pk(c0 == 0.f ? 0.f : a0, c1 == 0.f ? 0.f : a1);
        }
      }
      if (!cuts) {
        #pragma unroll
        for (int i = 0; i < RUN; ++i) u[i] = f2fma(a[i], cin, u[i]);
      } else {
        #pragma unroll
        for (int i = 0; i < RUN; ++i)
          if (i < first_cut) u[i] = f2fma(a[i], cin, u[i]);
      }
      if (ch.on0) {
        if (t0 + RUN <= p.T) {
          #pragma unroll
          for (int i = 0; i < RUN; ++i, out += p.h.s1) ch.store(out, u[i]);
        } else {
          #pragma unroll
          for (int i = 0; i < RUN; ++i, out += p.h.s1)
            if (t0 + i < p.T) ch.store(out, u[i]);
        }
      }
      if (PACKED && p.state_out && k.last) {
        #pragma unroll
        for (int i = 0; i < RUN; ++i) {
          if (!((k.last >> i) & 1)) continue;
          const int n = k.sequence(i);
          if (ch.on0) ch.store_state(p.state_out + (int64_t)n * p.C + base, u[i]);
        }
      }
      continue;
    }
    #pragma unroll 1
    for (int i = 0; i < RUN && t0 + i < p.T; ++i, out += p.h.s1) {
      const f32x2 v = i < first_cut ? through(la[i], cin, lu[i]) : lu[i];
      const int n = k.sequence(i);
      if (!ch.on0) continue;
      ch.store(out, v);
      if (PACKED && p.state_out && ((k.last >> i) & 1)) ch.store_state(p.state_out + (int64_t)n * p.C + base, v);
    }
  }
  cp_async_wait<0>();
  if (MAPS) write_map<PACKED>(p, chain, seg, all, c, any_cut);
  else if (!PACKED && p.state_out && seg == p.segments - 1 && warp == 0 && ch.on0)
    ch.store_state(p.state_out + (int64_t)b * p.C + base, c);
}

// The adjoint, walked from the last tile to the first; warp 0 takes a step's
// latest run, segment 0 the latest segment.  States inside a run are rebuilt
// from the state that the forward kept before it.
template <typename TX, typename TG, RowMode MODE, int NW, bool COMP, bool PACKED, bool MAPS>
__global__ void __launch_bounds__(32 * NW, resident_blocks<TX, TG, MODE>(NW, true)) k_scan_bwd(const ScanParams p) {
  typedef Rows<TX, MODE> RX;
  typedef Rows<TG, MODE> RG;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ ScanMaps<NW> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seg = (int)(blockIdx.x % p.segments);
  const int64_t chain = blockIdx.x / p.segments;
  const int b = PACKED ? 0 : (int)(chain / p.sets);
  const int base = (int)(chain % p.sets) * SET;
  const Pair<MODE> ch(lane, p.C - base);
  const TX* x = static_cast<const TX*>(p.x.p) + b * p.x.s0 + base;
  const TG* g = static_cast<const TG*>(p.g.p) + b * p.g.s0 + base;
  const TX* dh = static_cast<const TX*>(p.h.p) + b * p.h.s0 + base;
  TX* dx = static_cast<TX*>(const_cast<void*>(p.dx.p)) + b * p.dx.s0 + base;
  TG* dg = static_cast<TG*>(const_cast<void*>(p.dg.p)) + b * p.dg.s0 + base;
  const int runs = (p.T + RUN - 1) / RUN;

  if (PACKED && !MAPS && p.d_state_in && seg == 0) pass_empty(p, p.d_state_out, p.d_state_in, ch, base);
  if (!p.steps) return;
  f32x2 c = f2pk(0.f, 0.f), all = f2pk(1.f, 1.f);
  bool any_cut = false;
  if (!MAPS) {
    if (!PACKED && p.d_state_out) c = ch.load(p.d_state_out + (int64_t)b * p.C + base);
    if (p.maps) c = through_segments<PACKED>(p, chain, seg, lane, c);
  }

  constexpr int STAGE = 2 * RX::BYTES + RG::BYTES;
  auto stage = [&](int step) { return smem + ((step % STAGES) * NW + warp) * STAGE; };
  auto run_at = [&](int step) {
    return ((p.segments * p.steps - 1 - (seg * p.steps + (MAPS ? p.steps - 1 - step : step))) * NW + NW - 1 - warp) * RUN;
  };
  f32x2 next_state = f2pk(0.f, 0.f);  // state before the next step's run
  auto fetch = [&](int step) {
    if (step < p.steps) {
      const int t0 = run_at(step);
      RX{stage(step)}.fetch(dh, p.h.s1, t0, p.T, p.C - base, lane);
      RG{stage(step) + RX::BYTES}.fetch(g, p.g.s1, t0, p.T, p.C - base, lane);
      if (!MAPS) RX{stage(step) + RX::BYTES + RG::BYTES}.fetch(x, p.x.s1, t0, p.T, p.C - base, lane);
      if (!MAPS && t0 < p.T) next_state = ch.load(p.carry + (b * (int64_t)runs + t0 / RUN) * p.C + base);
    }
    cp_async_commit();
  };
  static_assert(STAGES == 2, "next_state is one step ahead");
  SequenceCursor<MAPS ? RUN - 1 : 0> cursor;
  fetch(0);
  for (int step = 0; step < p.steps; ++step) {
    __syncwarp();
    f32x2 hp = next_state;
    fetch(step + 1);
    const int t0 = run_at(step);
    RunMasks k{0, 0, ALL, 0};
    if (PACKED) k = cursor.masks(p.cu, p.B, p.T, t0, lane);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const auto ds = RX{stage(step)}.view(dh, p.h.s1, t0, lane);
    const auto gs = RG{stage(step) + RX::BYTES}.view(g, p.g.s1, t0, lane);
    const auto xs = RX{stage(step) + RX::BYTES + RG::BYTES}.view(x, p.x.s1, t0, lane);
    const unsigned cuts = PACKED ? (k.last | ~k.valid) & ALL : 0;
    const int n0 = PACKED ? k.sequence(0) : 0;
    TX* ox = dx + (int64_t)(t0 + RUN - 1) * p.dx.s1;
    TG* og = dg + (int64_t)(t0 + RUN - 1) * p.dg.s1;

    // a[i]: decay of token i; w[i]: what dg multiplies, h_{i-1} or h_{i-1} - x_i
    f32x2 a[RUN], m[RUN], w[RUN], A = f2pk(1.f, 1.f), M = f2pk(0.f, 0.f);
    f32x2 la[RUN], lm[RUN], lw[RUN];  // the same token by token, where a decay is out of range
    bool cut = false;
    const bool plain = decays<COMP && !MAPS>(gs, a, m);
    // state after token i, from the one before it; its weight in dg
    auto forward = [&](auto sure, int i, f32x2 g, f32x2 e, f32x2 r) {
      constexpr bool SURE = decltype(sure)::value;
      const f32x2 xf = xs.get(i);
      if (PACKED && ((k.start >> i) & 1)) {
        const int n = k.sequence(i);
        hp = p.state_in ? ch.load(p.state_in + (int64_t)n * p.C + base) : f2pk(0.f, 0.f);
      }
      const f32x2 weight = COMP ? f2fma(xf, f2pk(-1.f, -1.f), hp) : hp;
      hp = grow<SURE>(e, g, hp, COMP ? grow<SURE>(r, g, xf) : xf);
      return weight;
    };
    // the run's map, extended to the front by token i
    auto adjoint = [&](auto sure, int i, f32x2 g, f32x2 e) {
      constexpr bool SURE = decltype(sure)::value;
      if (PACKED && ((cuts >> i) & 1)) {
        const int n = k.sequence(i);
        cut = true;
        M = f2pk(0.f, 0.f);
        if ((k.last >> i) & 1) {
          if (p.d_state_out) M = ch.load(p.d_state_out + (int64_t)n * p.C + base);
          M = grow<SURE>(e, g, f2add(ds.get(i), M));
        }
      } else {
        M = grow<SURE>(e, g, f2add(ds.get(i), M));
        if (!cut) A = SURE ? f2mul(A, e) : chained(A, e);
      }
    };
    if (plain && !cuts) {
      if (!MAPS) {
        if (PACKED && k.start)  // at the run's first token, if anywhere
          hp = p.state_in ? ch.load(p.state_in + (int64_t)n0 * p.C + base) : f2pk(0.f, 0.f);
        #pragma unroll
        for (int i = 0; i < RUN; ++i) {
          const f32x2 xf = xs.get(i);
          w[i] = COMP ? f2fma(xf, f2pk(-1.f, -1.f), hp) : hp;
          hp = f2fma(a[i], hp, COMP ? f2mul(m[i], xf) : xf);
        }
      }
      // the run's map from the adjoint after it to the adjoint before it
      #pragma unroll
      for (int i = RUN - 1; i >= 0; --i) {
        M = f2mul(a[i], f2add(ds.get(i), M));
        A = f2mul(A, a[i]);
      }
    } else if (PACKED && plain) {
      #pragma unroll
      for (int i = 0; i < RUN; ++i)
        if (!MAPS) w[i] = forward(std::true_type(), i, a[i], a[i], m[i]);
      #pragma unroll
      for (int i = RUN - 1; i >= 0; --i) adjoint(std::true_type(), i, a[i], a[i]);
    } else {
      #pragma unroll 1
      for (int i = 0; i < RUN; ++i) {
        decay_any<COMP && !MAPS>(gs.get(i), la[i], lm[i]);
        if (!MAPS) lw[i] = forward(std::false_type(), i, gs.get(i), la[i], lm[i]);
      }
      #pragma unroll 1
      for (int i = RUN - 1; i >= 0; --i) adjoint(std::false_type(), i, gs.get(i), la[i]);
    }
    f32x2 tile = f2pk(1.f, 1.f), behind = f2pk(0.f, 0.f);
    bool wild;
    f32x2 mu = join<NW, PACKED, MAPS>(sh, step & 1, warp, lane, A, M, cut, MAPS ? behind : c, tile, any_cut, wild);
    if (MAPS) {  // this tile, then those before it
      c = through(all, behind, c);
      all = chained(sh, step & 1, lane, all, tile);
      if (PACKED && any_cut) break;
      continue;
    }
    if (plain && !cuts && t0 + RUN <= p.T) {
      if (!ch.on0) continue;
      #pragma unroll
      for (int i = RUN - 1; i >= 0; --i, ox -= p.dx.s1, og -= p.dg.s1) {
        const f32x2 l = f2add(ds.get(i), mu);
        ch.store(ox, COMP ? f2mul(m[i], l) : l);
        mu = f2mul(a[i], l);
        ch.store(og, f2mul(mu, w[i]));
      }
      if (PACKED && p.d_state_in && k.start) ch.store_state(p.d_state_in + (int64_t)n0 * p.C + base, mu);
      continue;
    }
    auto write = [&](auto sure, int i, f32x2 g, f32x2 e, f32x2 r, f32x2 weight) {
      constexpr bool SURE = decltype(sure)::value;
      const int n = PACKED ? k.sequence(i) : 0;
      if (PACKED && ((k.last >> i) & 1))
        mu = p.d_state_out ? ch.load(p.d_state_out + (int64_t)n * p.C + base) : f2pk(0.f, 0.f);
      const f32x2 l = f2add(ds.get(i), mu);
      f32x2 vx = COMP ? grow<SURE>(r, g, l) : l;
      mu = grow<SURE>(e, g, l);
      f32x2 vg = f2mul(mu, weight);
      if (PACKED && !((k.valid >> i) & 1)) vx = vg = mu = f2pk(0.f, 0.f);
      if (ch.on0 && t0 + i < p.T) {
        ch.store(ox, vx);
        ch.store(og, vg);
        if (PACKED && p.d_state_in && ((k.start >> i) & 1)) ch.store_state(p.d_state_in + (int64_t)n * p.C + base, mu);
      }
      ox -= p.dx.s1;
      og -= p.dg.s1;
    };
    if (plain) {
      if (!PACKED && t0 >= p.T) continue;  // nothing to write
      #pragma unroll
      for (int i = RUN - 1; i >= 0; --i) write(std::true_type(), i, a[i], a[i], m[i], w[i]);
    } else {
      #pragma unroll 1
      for (int i = RUN - 1; i >= 0; --i) write(std::false_type(), i, gs.get(i), la[i], lm[i], lw[i]);
    }
  }
  cp_async_wait<0>();
  if (MAPS) write_map<PACKED>(p, chain, seg, all, c, any_cut);
  else if (!PACKED && p.d_state_in && seg == p.segments - 1 && warp == 0 && ch.on0)
    ch.store_state(p.d_state_in + (int64_t)b * p.C + base, c);
}

// One token per sequence, the decode step: elementwise, state read and
// written once.  One thread per VEC channels of a sequence.
template <typename TX, typename TG, int VEC, bool COMP>
__global__ void __launch_bounds__(256) k_scan_step(const ScanParams p) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = p.C / VEC;
  if (e >= (int64_t)p.B * per) return;
  const int64_t b = e / per;
  const int c0 = (int)(e % per) * VEC;
  float g[VEC], x[VEC], s[VEC] = {};
  Vec<TG, VEC>::unpack(Vec<TG, VEC>::load(static_cast<const TG*>(p.g.p) + b * p.g.s0 + c0), g);
  Vec<TX, VEC>::unpack(Vec<TX, VEC>::load(static_cast<const TX*>(p.x.p) + b * p.x.s0 + c0), x);
  if (p.state_in) load_f32<VEC>(p.state_in + b * p.C + c0, s);
  #pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const bool grown = g[v] <= FLT_MAX;  // see grow()
    const float in = !COMP ? x[v] : x[v] == 0.f && grown ? 0.f : -expm1f(g[v]) * x[v];
    s[v] = s[v] == 0.f && grown ? in : fmaf(expf(g[v]), s[v], in);
  }
  if (p.state_out) store_f32<VEC>(p.state_out + b * p.C + c0, s);
  Vec<TX, VEC>::store(static_cast<TX*>(const_cast<void*>(p.h.p)) + b * p.h.s0 + c0, s);
}

// ---- host: the kernels of one pair of types (one source file each, compiled side by side) ----

// How a call is cut up: how rows are held, warps (runs) of a block, segments of the time axis.
struct ScanPlan {
  RowMode mode;
  int warps, sets, steps, segments;
  int64_t chains;
};

template <typename K>
static int launch(K kernel, const ScanParams& p, const ScanPlan& n, int stage, cudaStream_t st, const char* fn) {
  const int64_t grid = n.chains * n.segments;
  if (grid > 0x7fffffffll) return set_error(GDN2_EUNSUPPORTED, "%s: %lld blocks", fn, (long long)grid);
  const int smem = STAGES * n.warps * stage;
  int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), fn);
  if (rc) return rc;
  kernel<<<(unsigned)grid, 32 * n.warps, smem, st>>>(p);
  return check_cuda(cudaGetLastError(), fn);
}

template <typename TX, typename TG, RowMode MODE, bool COMP, bool PACKED>
static int run_scan(const ScanParams& p, const ScanPlan& n, bool bwd, cudaStream_t st, const char* fn) {
  const int stage = stage_bytes<TX, TG, MODE>(bwd);
  if (n.warps == 8)
    return bwd ? launch(k_scan_bwd<TX, TG, MODE, 8, COMP, PACKED, false>, p, n, stage, st, fn)
               : launch(k_scan_fwd<TX, TG, MODE, 8, COMP, PACKED, false>, p, n, stage, st, fn);
  if (n.segments > 1) {
    int rc = bwd ? launch(k_scan_bwd<TX, TG, MODE, 4, COMP, PACKED, true>, p, n, stage, st, fn)
                 : launch(k_scan_fwd<TX, TG, MODE, 4, COMP, PACKED, true>, p, n, stage, st, fn);
    if (rc) return rc;
  }
  return bwd ? launch(k_scan_bwd<TX, TG, MODE, 4, COMP, PACKED, false>, p, n, stage, st, fn)
             : launch(k_scan_fwd<TX, TG, MODE, 4, COMP, PACKED, false>, p, n, stage, st, fn);
}

template <typename TX, typename TG, bool COMP>
static int run_step(const ScanParams& p, bool pairs, cudaStream_t st, const char* fn) {
  const int64_t count = ((int64_t)p.B * (p.C / (pairs ? 2 : 1)) + 255) / 256;
  if (count > 0x7fffffffll) return set_error(GDN2_EUNSUPPORTED, "%s: too many channels", fn);
  if (pairs) k_scan_step<TX, TG, 2, COMP><<<(unsigned)count, 256, 0, st>>>(p);
  else k_scan_step<TX, TG, 1, COMP><<<(unsigned)count, 256, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), fn);
}

template <typename TX, typename TG, bool COMP>
static int run_mode(const ScanParams& p, const ScanPlan& n, bool bwd, cudaStream_t st, const char* fn) {
  if (p.T == 1 && !p.cu && !p.carry && !bwd)
    return run_step<TX, TG, COMP>(p, n.mode == ROWS16 || n.mode == ROWS_PAIR, st, fn);
  if (p.cu)
    return n.mode == ROWS16      ? run_scan<TX, TG, ROWS16, COMP, true>(p, n, bwd, st, fn)
           : n.mode == ROWS_PAIR ? run_scan<TX, TG, ROWS_PAIR, COMP, true>(p, n, bwd, st, fn)
           : n.mode == ROWS_ODD  ? run_scan<TX, TG, ROWS_ODD, COMP, true>(p, n, bwd, st, fn)
                                 : run_scan<TX, TG, ROWS_ANY, COMP, true>(p, n, bwd, st, fn);
  return n.mode == ROWS16      ? run_scan<TX, TG, ROWS16, COMP, false>(p, n, bwd, st, fn)
         : n.mode == ROWS_PAIR ? run_scan<TX, TG, ROWS_PAIR, COMP, false>(p, n, bwd, st, fn)
         : n.mode == ROWS_ODD  ? run_scan<TX, TG, ROWS_ODD, COMP, false>(p, n, bwd, st, fn)
                               : run_scan<TX, TG, ROWS_ANY, COMP, false>(p, n, bwd, st, fn);
}

// The scan (its adjoint with bwd) of x in TX and g in TG.
template <typename TX, typename TG>
int run_types(const ScanParams& p, const ScanPlan& n, bool comp, bool bwd, cudaStream_t st, const char* fn) {
  return comp ? run_mode<TX, TG, true>(p, n, bwd, st, fn) : run_mode<TX, TG, false>(p, n, bwd, st, fn);
}
extern template int run_types<float, float>(const ScanParams&, const ScanPlan&, bool, bool, cudaStream_t, const char*);
extern template int run_types<__nv_bfloat16, float>(const ScanParams&, const ScanPlan&, bool, bool, cudaStream_t, const char*);
extern template int run_types<__nv_bfloat16, __nv_bfloat16>(const ScanParams&, const ScanPlan&, bool, bool, cudaStream_t,
                                                            const char*);

}  // namespace gdn2

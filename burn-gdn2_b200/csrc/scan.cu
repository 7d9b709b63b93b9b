// Gated scan: the diagonal gated linear recurrence
//
//   h_t = e^{g_t} h_{t-1} + s_t x_t        s_t = 1, or 1 - e^{g_t} (complement)
//
// per channel of [B][T][C] (or of packed sequences), and its adjoint
//
//   l_t = dh_t + e^{g_{t+1}} l_{t+1},  dx_t = s_t l_t,
//   dg_t = e^{g_t} (h_{t-1} [- x_t]) l_t,  dstate = e^{g_0} l_0.
//
// Both are bound by HBM: a forward reads x and g and writes h once, a
// backward reads x, g and dh and writes dx and dg, some ten flops per byte.
// So each value is read once into registers and every step of the scan
// happens there: a warp holds RUN tokens of 32 * VEC neighbouring channels (all
// its loads in flight at once), reduces them to the affine map
// c -> A c + H of the run, and the maps of a tile's runs are joined through
// shared memory and those of the cluster's tiles through distributed shared
// memory.  A cluster walks its channels' whole time axis, CL tiles a step,
// so one pass over the data suffices and the carry never leaves the chip.
// The cluster is wider the fewer chains there are.  The joining order is
// fixed: results do not depend on timing.
#include "scan.cuh"

namespace gdn2 {

constexpr int RUN = 16;  // tokens of a warp's run; also the spacing of the states a backward starts from
constexpr int MAX_CL = 8;

struct ScanParams {
  int B, T, C;     // dense: B sequences of T; packed: N sequences in T rows
  int tiles, steps;
  int sets;        // sets of 32 * VEC channels
  const int* cu;
  DView x, g, h;   // forward: h out.  backward: h = dh
  DView dx, dg;
  const float* state_in;
  float* state_out;
  const float* d_state_out;
  float* d_state_in;
  float* carry;    // [B or 1][ceil(T / RUN)][C]: state before every RUN-th token
};

// A product of decays that a sequence start cuts is the negative zero: no
// decay is negative, so the sign marks "take nothing from before", also
// where what is before holds an infinity or NaN of another sequence.
__device__ __forceinline__ bool is_cut(float A) { return __float_as_uint(A) == 0x80000000u; }

template <bool PACKED>
__device__ __forceinline__ float carry_on(float A, float H, float c) {
  return PACKED && is_cut(A) ? H : fmaf(A, c, H);
}
// The product of the decays A, then a; a cut stays one, whatever follows.
template <bool PACKED>
__device__ __forceinline__ float chain(float A, float a) {
  if (PACKED && is_cut(A)) return A;
  return PACKED && is_cut(a) ? a : A * a;
}

// The maps of a step, [run][channel] of this tile and [tile][channel] of the cluster, twice for alternating steps.
template <int NW, int CH>
struct ScanShared {
  float2 run[2][NW][CH];
  float2 tile[2][MAX_CL][CH];
};

// Joins the runs' maps: from the state `c` before the step's first token (or
// after its last, in the reverse direction), the state before this warp's
// run; c becomes the state after the step.  Run and tile order is the
// direction of the scan.
template <int NW, int VEC, bool PACKED>
__device__ __forceinline__ void join(ScanShared<NW, 32 * VEC>& sh, int buf, int CL, int rank, int warp, int lane,
                                     const float (&A)[VEC], const float (&H)[VEC], float (&c)[VEC],
                                     float (&cin)[VEC]) {
  constexpr int CH = 32 * VEC;
  const int ch = lane * VEC;
  #pragma unroll
  for (int v = 0; v < VEC; ++v) sh.run[buf][warp][ch + v] = make_float2(A[v], H[v]);
  __syncthreads();
  if (CL == 1) {
    #pragma unroll
    for (int w = 0; w < NW; ++w) {
      #pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if (w == warp) cin[v] = c[v];
        const float2 m = sh.run[buf][w][ch + v];
        c[v] = carry_on<PACKED>(m.x, m.y, c[v]);
      }
    }
    return;
  }
  for (int e = threadIdx.x; e < CH; e += 32 * NW) {
    float2 t = sh.run[buf][0][e];
    #pragma unroll
    for (int w = 1; w < NW; ++w) {
      const float2 m = sh.run[buf][w][e];
      t.y = carry_on<PACKED>(m.x, m.y, t.y);
      t.x = chain<PACKED>(t.x, m.x);
    }
    for (int r = 0; r < CL; ++r) {
      const uint32_t at = cluster_addr(&sh.tile[buf][rank][e], r);
      st_cluster_f32(at, t.x);
      st_cluster_f32(at + 4, t.y);
    }
  }
  cluster_sync_all();
  #pragma unroll
  for (int v = 0; v < VEC; ++v) {
    float s = c[v];
    for (int r = 0; r < CL; ++r) {
      if (r == rank) cin[v] = s;
      const float2 m = sh.tile[buf][r][ch + v];
      s = carry_on<PACKED>(m.x, m.y, s);
    }
    c[v] = s;
    for (int w = 0; w < warp; ++w) {
      const float2 m = sh.run[buf][w][ch + v];
      cin[v] = carry_on<PACKED>(m.x, m.y, cin[v]);
    }
  }
}

// Decays of a run: raw g to a = e^g and m = e^g - 1.
template <typename TG, int VEC>
__device__ __forceinline__ void decays(const typename Vec<TG, VEC>::Raw (&gr)[RUN], float (&a)[RUN][VEC],
                                       float (&m)[RUN][VEC]) {
  float g[RUN][VEC];
  float far = 0.f;
  #pragma unroll
  for (int i = 0; i < RUN; ++i) {
    Vec<TG, VEC>::unpack(gr[i], g[i]);
    #pragma unroll
    for (int v = 0; v < VEC; ++v) far = fmaxf(far, fabsf(g[i][v]));
  }
  if constexpr (VEC == 1) {
    #pragma unroll
    for (int i = 0; i < RUN; i += 2) exp_pair(g[i][0], g[i + 1][0], a[i][0], a[i + 1][0], m[i][0], m[i + 1][0]);
  } else {
    #pragma unroll
    for (int i = 0; i < RUN; ++i)
      #pragma unroll
      for (int v = 0; v < VEC; v += 2) exp_pair(g[i][v], g[i][v + 1], a[i][v], a[i][v + 1], m[i][v], m[i][v + 1]);
  }
  if (far > kExpRange) {  // a reset (-inf), a decay below every f32, or growth
    #pragma unroll
    for (int i = 0; i < RUN; ++i)
      #pragma unroll
      for (int v = 0; v < VEC; ++v)
        if (fabsf(g[i][v]) > kExpRange) {
          a[i][v] = expf(g[i][v]);
          m[i][v] = expm1f(g[i][v]);
        }
  }
}

// Whether packed sequence n has no row.  Offsets beyond the T rows count as T.
__device__ __forceinline__ bool is_empty(const int* __restrict__ cu, int n, int T) {
  const int from = __ldg(cu + n);
  return __ldg(cu + n + 1) <= from || from >= T;
}

// Which of a run's tokens open or close a sequence or lie in one, one bit a
// token; seq: the sequence of token `lane`.
struct RunMasks {
  unsigned start, last, valid;
  int seq;
};
__device__ __forceinline__ RunMasks run_masks(const int* __restrict__ cu, int N, int T, int t0, int lane) {
  RunMasks k;
  const int t = t0 + lane;
  k.seq = -1;
  bool s = false, l = false;
  if (lane < RUN && t < T) {
    k.seq = find_sequence(cu, N, t);
    if (k.seq >= 0) {
      s = __ldg(cu + k.seq) == t;
      l = t + 1 == T || __ldg(cu + k.seq + 1) == t + 1;
    }
  }
  k.start = __ballot_sync(0xffffffffu, s);
  k.last = __ballot_sync(0xffffffffu, l);
  k.valid = __ballot_sync(0xffffffffu, k.seq >= 0);
  return k;
}

template <typename TX, typename TG, int VEC, int NW, bool COMP, bool PACKED>
__global__ void __launch_bounds__(32 * NW) k_scan_fwd(ScanParams p, int CL) {
  constexpr int CH = 32 * VEC;
  __shared__ ScanShared<NW, CH> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = CL == 1 ? 0 : (int)(blockIdx.x % CL);
  const int64_t chain = blockIdx.x / CL;
  const int b = (int)(chain / p.sets);
  const int c0 = (int)(chain % p.sets) * CH + lane * VEC;
  const bool on = c0 < p.C;
  const TX* x = static_cast<const TX*>(p.x.p) + (PACKED ? 0 : (int64_t)b * p.x.s0) + c0;
  const TG* g = static_cast<const TG*>(p.g.p) + (PACKED ? 0 : (int64_t)b * p.g.s0) + c0;
  TX* h = static_cast<TX*>(const_cast<void*>(p.h.p)) + (PACKED ? 0 : (int64_t)b * p.h.s0) + c0;

  if (PACKED && p.state_out && rank == 0) {  // empty sequences keep their state
    for (int n0 = warp * 32; n0 < p.B; n0 += 32 * NW) {
      const int n = n0 + lane;
      unsigned empty = __ballot_sync(0xffffffffu, n < p.B && is_empty(p.cu, n, p.T));
      while (empty) {
        const int j = n0 + __ffs(empty) - 1;
        empty &= empty - 1;
        if (on) {
          float s[VEC] = {};
          if (p.state_in) load_f32<VEC>(p.state_in + (int64_t)j * p.C + c0, s);
          store_f32<VEC>(p.state_out + (int64_t)j * p.C + c0, s);
        }
      }
    }
  }

  if (CL > 1) cluster_sync_all();  // every CTA of the cluster runs before its memory is written

  float c[VEC] = {};
  if (!PACKED && p.state_in && on) load_f32<VEC>(p.state_in + (int64_t)b * p.C + c0, c);

  for (int step = 0; step < p.steps; ++step) {
    const int t0 = ((step * CL + rank) * NW + warp) * RUN;
    typename Vec<TX, VEC>::Raw xr[RUN];
    typename Vec<TG, VEC>::Raw gr[RUN];
    #pragma unroll
    for (int i = 0; i < RUN; ++i) {
      const bool in = on && t0 + i < p.T;
      xr[i] = typename Vec<TX, VEC>::Raw{};
      gr[i] = typename Vec<TG, VEC>::Raw{};
      if (in) {
        xr[i] = Vec<TX, VEC>::load(x + (int64_t)(t0 + i) * p.x.s1);
        gr[i] = Vec<TG, VEC>::load(g + (int64_t)(t0 + i) * p.g.s1);
      }
    }
    RunMasks k;
    if (PACKED) k = run_masks(p.cu, p.B, p.T, t0, lane);

    // a[i]: product of the decays up to token i, u[i]: the state there from a zero one before the run
    float a[RUN][VEC], u[RUN][VEC], A[VEC], H[VEC];
    decays<TG, VEC>(gr, a, u);
    #pragma unroll
    for (int v = 0; v < VEC; ++v) { A[v] = 1.f; H[v] = 0.f; }
    #pragma unroll
    for (int i = 0; i < RUN; ++i) {
      float xf[VEC];
      Vec<TX, VEC>::unpack(xr[i], xf);
      float st[VEC] = {};
      bool opens = false, out = false;
      if (PACKED) {
        opens = (k.start >> i) & 1;
        out = !((k.valid >> i) & 1);
        const int n = __shfl_sync(0xffffffffu, k.seq, i);
        if (opens && p.state_in && on) load_f32<VEC>(p.state_in + (int64_t)n * p.C + c0, st);
      }
      #pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float in = COMP ? -u[i][v] * xf[v] : xf[v];
        if (PACKED && (opens || out)) {
          H[v] = out ? 0.f : fmaf(a[i][v], st[v], in);
          A[v] = -0.f;
        } else {
          H[v] = fmaf(a[i][v], H[v], in);
          A[v] = PACKED && is_cut(A[v]) ? A[v] : A[v] * a[i][v];
        }
        a[i][v] = A[v];
        u[i][v] = H[v];
      }
    }
    float cin[VEC];
    join<NW, VEC, PACKED>(sh, step & 1, CL, rank, warp, lane, A, H, c, cin);

    if (on && t0 < p.T) {
      if (p.carry)
        store_f32<VEC>(p.carry + ((PACKED ? 0 : (int64_t)b * ((p.T + RUN - 1) / RUN)) + t0 / RUN) * p.C + c0, cin);
      #pragma unroll
      for (int i = 0; i < RUN; ++i) {
        #pragma unroll
        for (int v = 0; v < VEC; ++v) u[i][v] = carry_on<PACKED>(a[i][v], u[i][v], cin[v]);
        if (t0 + i < p.T) Vec<TX, VEC>::store(h + (int64_t)(t0 + i) * p.h.s1, u[i]);
      }
    }
    if (PACKED && p.state_out && k.last) {
      #pragma unroll
      for (int i = 0; i < RUN; ++i) {
        if (!((k.last >> i) & 1)) continue;
        const int n = __shfl_sync(0xffffffffu, k.seq, i);
        if (on) store_f32<VEC>(p.state_out + (int64_t)n * p.C + c0, u[i]);
      }
    }
  }
  if (!PACKED && p.state_out && rank == 0 && warp == 0 && on) store_f32<VEC>(p.state_out + (int64_t)b * p.C + c0, c);
}

// The adjoint, walked from the last tile to the first; warp 0 of rank 0 takes
// a step's latest run.  States inside a run are rebuilt from the state that
// the forward kept before it.
template <typename TX, typename TG, int VEC, int NW, bool COMP, bool PACKED>
__global__ void __launch_bounds__(32 * NW) k_scan_bwd(ScanParams p, int CL) {
  constexpr int CH = 32 * VEC;
  __shared__ ScanShared<NW, CH> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = CL == 1 ? 0 : (int)(blockIdx.x % CL);
  const int64_t chain = blockIdx.x / CL;
  const int b = (int)(chain / p.sets);
  const int c0 = (int)(chain % p.sets) * CH + lane * VEC;
  const bool on = c0 < p.C;
  const TX* x = static_cast<const TX*>(p.x.p) + (PACKED ? 0 : (int64_t)b * p.x.s0) + c0;
  const TG* g = static_cast<const TG*>(p.g.p) + (PACKED ? 0 : (int64_t)b * p.g.s0) + c0;
  const TX* dh = static_cast<const TX*>(p.h.p) + (PACKED ? 0 : (int64_t)b * p.h.s0) + c0;
  TX* dx = static_cast<TX*>(const_cast<void*>(p.dx.p)) + (PACKED ? 0 : (int64_t)b * p.dx.s0) + c0;
  TG* dg = static_cast<TG*>(const_cast<void*>(p.dg.p)) + (PACKED ? 0 : (int64_t)b * p.dg.s0) + c0;

  if (PACKED && p.d_state_in && rank == 0) {  // an empty sequence hands its state's gradient through
    for (int n0 = warp * 32; n0 < p.B; n0 += 32 * NW) {
      const int n = n0 + lane;
      unsigned empty = __ballot_sync(0xffffffffu, n < p.B && is_empty(p.cu, n, p.T));
      while (empty) {
        const int j = n0 + __ffs(empty) - 1;
        empty &= empty - 1;
        if (on) {
          float s[VEC] = {};
          if (p.d_state_out) load_f32<VEC>(p.d_state_out + (int64_t)j * p.C + c0, s);
          store_f32<VEC>(p.d_state_in + (int64_t)j * p.C + c0, s);
        }
      }
    }
  }

  if (CL > 1) cluster_sync_all();

  float c[VEC] = {};
  if (!PACKED && p.d_state_out && on) load_f32<VEC>(p.d_state_out + (int64_t)b * p.C + c0, c);

  for (int step = 0; step < p.steps; ++step) {
    const int t0 = (p.steps * CL * NW - 1 - ((step * CL + rank) * NW + warp)) * RUN;
    typename Vec<TX, VEC>::Raw xr[RUN], dr[RUN];
    typename Vec<TG, VEC>::Raw gr[RUN];
    #pragma unroll
    for (int i = 0; i < RUN; ++i) {
      const bool in = on && t0 + i < p.T;
      xr[i] = dr[i] = typename Vec<TX, VEC>::Raw{};
      gr[i] = typename Vec<TG, VEC>::Raw{};
      if (in) {
        xr[i] = Vec<TX, VEC>::load(x + (int64_t)(t0 + i) * p.x.s1);
        gr[i] = Vec<TG, VEC>::load(g + (int64_t)(t0 + i) * p.g.s1);
        dr[i] = Vec<TX, VEC>::load(dh + (int64_t)(t0 + i) * p.h.s1);
      }
    }
    float hp[VEC] = {};  // state before the run
    if (on && t0 < p.T)
      load_f32<VEC>(p.carry + ((PACKED ? 0 : (int64_t)b * ((p.T + RUN - 1) / RUN)) + t0 / RUN) * p.C + c0, hp);
    RunMasks k;
    if (PACKED) k = run_masks(p.cu, p.B, p.T, t0, lane);

    // a[i]: decay of token i; w[i]: what dg multiplies, h_{i-1} or h_{i-1} - x_i
    float a[RUN][VEC], m[RUN][VEC], w[RUN][VEC];
    decays<TG, VEC>(gr, a, m);
    #pragma unroll
    for (int i = 0; i < RUN; ++i) {
      float xf[VEC];
      Vec<TX, VEC>::unpack(xr[i], xf);
      if (PACKED && ((k.start >> i) & 1)) {
        const int n = __shfl_sync(0xffffffffu, k.seq, i);
        #pragma unroll
        for (int v = 0; v < VEC; ++v) hp[v] = 0.f;
        if (p.state_in && on) load_f32<VEC>(p.state_in + (int64_t)n * p.C + c0, hp);
      }
      #pragma unroll
      for (int v = 0; v < VEC; ++v) {
        w[i][v] = COMP ? hp[v] - xf[v] : hp[v];
        hp[v] = fmaf(a[i][v], hp[v], COMP ? -m[i][v] * xf[v] : xf[v]);
      }
    }
    // the run's map from the adjoint after it to the adjoint before it
    float A[VEC], M[VEC];
    #pragma unroll
    for (int v = 0; v < VEC; ++v) { A[v] = 1.f; M[v] = 0.f; }
    #pragma unroll
    for (int i = RUN - 1; i >= 0; --i) {
      float df[VEC];
      Vec<TX, VEC>::unpack(dr[i], df);
      bool closes = false, out = false;
      float st[VEC] = {};
      if (PACKED) {
        closes = (k.last >> i) & 1;
        out = !((k.valid >> i) & 1);
        const int n = __shfl_sync(0xffffffffu, k.seq, i);
        if (closes && p.d_state_out && on) load_f32<VEC>(p.d_state_out + (int64_t)n * p.C + c0, st);
      }
      #pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if (PACKED && (closes || out)) {
          M[v] = out ? 0.f : a[i][v] * (df[v] + st[v]);
          A[v] = -0.f;
        } else {
          M[v] = a[i][v] * (df[v] + M[v]);
          A[v] = PACKED && is_cut(A[v]) ? A[v] : A[v] * a[i][v];
        }
      }
    }
    float mu[VEC];
    join<NW, VEC, PACKED>(sh, step & 1, CL, rank, warp, lane, A, M, c, mu);

    #pragma unroll
    for (int i = RUN - 1; i >= 0; --i) {
      float df[VEC], ox[VEC], og[VEC];
      Vec<TX, VEC>::unpack(dr[i], df);
      bool out = false;
      if (PACKED) {
        out = !((k.valid >> i) & 1);
        if ((k.last >> i) & 1) {
          const int n = __shfl_sync(0xffffffffu, k.seq, i);
          #pragma unroll
          for (int v = 0; v < VEC; ++v) mu[v] = 0.f;
          if (p.d_state_out && on) load_f32<VEC>(p.d_state_out + (int64_t)n * p.C + c0, mu);
        }
      }
      #pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float l = df[v] + mu[v];
        ox[v] = COMP ? -m[i][v] * l : l;
        mu[v] = a[i][v] * l;
        og[v] = mu[v] * w[i][v];
        if (PACKED && out) ox[v] = og[v] = mu[v] = 0.f;
      }
      if (on && t0 + i < p.T) {
        Vec<TX, VEC>::store(dx + (int64_t)(t0 + i) * p.dx.s1, ox);
        Vec<TG, VEC>::store(dg + (int64_t)(t0 + i) * p.dg.s1, og);
      }
      if (PACKED && p.d_state_in && ((k.start >> i) & 1)) {
        const int n = __shfl_sync(0xffffffffu, k.seq, i);
        if (on) store_f32<VEC>(p.d_state_in + (int64_t)n * p.C + c0, mu);
      }
    }
  }
  if (!PACKED && p.d_state_in && rank == 0 && warp == 0 && on)
    store_f32<VEC>(p.d_state_in + (int64_t)b * p.C + c0, c);
}

// One token per sequence, the decode step: elementwise, state read and
// written once.  One thread per VEC channels of a sequence.
template <typename TX, typename TG, int VEC, bool COMP>
__global__ void __launch_bounds__(256) k_scan_step(ScanParams p) {
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
  for (int v = 0; v < VEC; ++v) s[v] = fmaf(expf(g[v]), s[v], COMP ? -expm1f(g[v]) * x[v] : x[v]);
  if (p.state_out) store_f32<VEC>(p.state_out + b * p.C + c0, s);
  Vec<TX, VEC>::store(static_cast<TX*>(const_cast<void*>(p.h.p)) + b * p.h.s0 + c0, s);
}

// ---- host ----

static bool rows_ok(const gdn2_view& v, int vec, int elem) {
  return (uintptr_t)v.data % (vec * elem) == 0 && v.stride0 % vec == 0 && v.stride1 % vec == 0;
}

static int elem_bytes(int dtype) { return dtype == GDN2_DTYPE_BF16 ? 2 : 4; }

// Tiles per step (the cluster): enough CTAs to hold the memory system's
// latency in flight, no more than the time axis has.
static int cluster_size(int64_t chains, int tiles) {
  int cl = 1;
  while (cl < MAX_CL && chains * cl < 2 * 148 && 2 * cl <= tiles) cl *= 2;
  return cl;
}

template <typename K>
static int launch(K kernel, ScanParams& p, int64_t chains, int nw, cudaStream_t st, const char* fn) {
  p.tiles = (p.T + nw * RUN - 1) / (nw * RUN);
  const int cl = cluster_size(chains, p.tiles);
  p.steps = (p.tiles + cl - 1) / cl;
  if (chains * cl > 0x7fffffffll) return set_error(GDN2_EUNSUPPORTED, "%s: %lld channel sets", fn, (long long)chains);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(chains * cl));
  cfg.blockDim = dim3(32 * nw);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cl;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, p, cl), fn);
}

template <typename TX, typename TG, int VEC, bool COMP>
static int run_fwd(ScanParams& p, cudaStream_t st, const char* fn) {
  p.sets = (p.C + 32 * VEC - 1) / (32 * VEC);
  if (p.cu) return launch(k_scan_fwd<TX, TG, VEC, 4, COMP, true>, p, p.sets, 4, st, fn);
  const int64_t chains = (int64_t)p.B * p.sets;
  if (p.T == 1 && !p.carry) {
    const int64_t n = (int64_t)p.B * (p.C / VEC);
    if ((n + 255) / 256 > 0x7fffffffll) return set_error(GDN2_EUNSUPPORTED, "%s: too many channels", fn);
    k_scan_step<TX, TG, VEC, COMP><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(p);
    return check_cuda(cudaGetLastError(), fn);
  }
  if (p.T <= RUN) return launch(k_scan_fwd<TX, TG, VEC, 1, COMP, false>, p, chains, 1, st, fn);
  return launch(k_scan_fwd<TX, TG, VEC, 4, COMP, false>, p, chains, 4, st, fn);
}

template <typename TX, typename TG, int VEC, bool COMP>
static int run_bwd(ScanParams& p, cudaStream_t st, const char* fn) {
  p.sets = (p.C + 32 * VEC - 1) / (32 * VEC);
  if (p.cu) return launch(k_scan_bwd<TX, TG, VEC, 4, COMP, true>, p, p.sets, 4, st, fn);
  const int64_t chains = (int64_t)p.B * p.sets;
  if (p.T <= RUN) return launch(k_scan_bwd<TX, TG, VEC, 1, COMP, false>, p, chains, 1, st, fn);
  return launch(k_scan_bwd<TX, TG, VEC, 4, COMP, false>, p, chains, 4, st, fn);
}

template <typename TX, typename TG, int VEC>
static int run_comp(ScanParams& p, bool comp, bool bwd, cudaStream_t st, const char* fn) {
  if (bwd) return comp ? run_bwd<TX, TG, VEC, true>(p, st, fn) : run_bwd<TX, TG, VEC, false>(p, st, fn);
  return comp ? run_fwd<TX, TG, VEC, true>(p, st, fn) : run_fwd<TX, TG, VEC, false>(p, st, fn);
}

template <typename TX, typename TG>
static int run_vec(ScanParams& p, bool pairs, bool comp, bool bwd, cudaStream_t st, const char* fn) {
  return pairs ? run_comp<TX, TG, 2>(p, comp, bwd, st, fn) : run_comp<TX, TG, 1>(p, comp, bwd, st, fn);
}

static int dispatch(ScanParams& p, const gdn2_scan_args* a, bool pairs, bool bwd, cudaStream_t st, const char* fn) {
  const bool comp = a->complement != 0;
  if (a->dtype == GDN2_DTYPE_F32) return run_vec<float, float>(p, pairs, comp, bwd, st, fn);
  if (a->g_dtype == GDN2_DTYPE_F32) return run_vec<__nv_bfloat16, float>(p, pairs, comp, bwd, st, fn);
  return run_vec<__nv_bfloat16, __nv_bfloat16>(p, pairs, comp, bwd, st, fn);
}

static int check_scan(const gdn2_scan_args* a, const char* fn) {
  if (!a) return set_error(GDN2_EINVAL, "%s: null args", fn);
  if (a->batch <= 0 || a->seq_len < 0 || a->channels <= 0 || (a->seq_len == 0 && !a->cu_seqlens))
    return set_error(GDN2_EINVAL, "%s: sizes must be > 0 (batch=%d seq_len=%d channels=%d)", fn, a->batch, a->seq_len,
                     a->channels);
  if (a->seq_len > (1 << 30)) return set_error(GDN2_EUNSUPPORTED, "%s: seq_len=%d above 2^30", fn, a->seq_len);
  if ((a->dtype != GDN2_DTYPE_F32 && a->dtype != GDN2_DTYPE_BF16) ||
      (a->g_dtype != GDN2_DTYPE_F32 && a->g_dtype != GDN2_DTYPE_BF16))
    return set_error(GDN2_EINVAL, "%s: unknown dtype %d / %d", fn, a->dtype, a->g_dtype);
  if (a->dtype == GDN2_DTYPE_F32 && a->g_dtype != GDN2_DTYPE_F32)
    return set_error(GDN2_EUNSUPPORTED, "%s: f32 x with bf16 g", fn);
  if (a->seq_len && (!a->x.data || !a->g.data)) return set_error(GDN2_EINVAL, "%s: null tensor pointer", fn);
  return GDN2_OK;
}

static void fill(ScanParams& p, const gdn2_scan_args* a) {
  p = ScanParams{};
  p.B = a->batch; p.T = a->seq_len; p.C = a->channels;
  p.cu = a->cu_seqlens;
  p.x = make_dview(a->x); p.g = make_dview(a->g);
  p.state_in = a->state_in;
  p.carry = a->carry;
}

int launch_scan_fwd(const gdn2_scan_args* a, const gdn2_view& h, float* state_out, cudaStream_t st) {
  const char* fn = "gdn2_gated_scan";
  int rc = check_scan(a, fn);
  if (rc) return rc;
  if (a->seq_len && !h.data) return set_error(GDN2_EINVAL, "%s: null tensor pointer", fn);
  ScanParams p;
  fill(p, a);
  p.h = make_dview(h);
  p.state_out = state_out;
  const int ex = elem_bytes(a->dtype), eg = elem_bytes(a->g_dtype);
  const bool pairs = a->channels % 2 == 0 && rows_ok(a->x, 2, ex) && rows_ok(a->g, 2, eg) && rows_ok(h, 2, ex);
  return dispatch(p, a, pairs, false, st, fn);
}

int launch_scan_bwd(const gdn2_scan_bwd_args* q, cudaStream_t st) {
  const char* fn = "gdn2_gated_scan_bwd";
  if (!q) return set_error(GDN2_EINVAL, "%s: null args", fn);
  const gdn2_scan_args* a = &q->fwd;
  int rc = check_scan(a, fn);
  if (rc) return rc;
  if (a->seq_len && (!q->d_h.data || !q->dx.data || !q->dg.data || !a->carry))
    return set_error(GDN2_EINVAL, "%s: null tensor pointer", fn);
  ScanParams p;
  fill(p, a);
  p.h = make_dview(q->d_h);
  p.dx = make_dview(q->dx); p.dg = make_dview(q->dg);
  p.d_state_out = q->d_state_out;
  p.d_state_in = q->d_state_in;
  const int ex = elem_bytes(a->dtype), eg = elem_bytes(a->g_dtype);
  const bool pairs = a->channels % 2 == 0 && rows_ok(a->x, 2, ex) && rows_ok(a->g, 2, eg) && rows_ok(q->d_h, 2, ex) &&
                     rows_ok(q->dx, 2, ex) && rows_ok(q->dg, 2, eg);
  return dispatch(p, a, pairs, true, st, fn);
}

}  // namespace gdn2

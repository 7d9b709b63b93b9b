// Causal depthwise convolution of four taps with SiLU over dense or packed
// sequences, and its adjoint:
//
//   pre_t = sum_j w[c][j] x_{t-3+j},  y_t = silu(pre_t)
//   dpre_t = dy_t silu'(pre_t),  dx_t = sum_k w[c][3-k] dpre_{t+k},  dw[c][j] = sum_t dpre_t x_{t-3+j}
//
// The three tokens before a sequence are its cache, or copies of its first
// token (src/short_conv.rs:42-54).  Bound by HBM: x in and y out, or x and dy
// in and dx out.  A warp walks a span of tokens of 64 channels in runs
// that are copied to shared memory a run ahead; the three values before a
// token stay in registers, so a span reads nothing twice but the three rows
// in front of it.  In the adjoint the dx of the last three tokens stay in
// registers as well until the tokens behind have added their parts, and a span
// ends with the three tokens behind it (13 own tokens and those make its last
// run).  Runs inside a sequence take a short path; those where one begins or
// ends sort out caches and copies token by token.  Each lane sums dw over its
// spans, the block adds its warps' sums and a second kernel the blocks', in a
// fixed order.
//
// 8 x 4096 x 2048 bf16: 57 us forward and 94 us backward, 72 % and 65 % of what a
// copy of as many bytes reaches, at some 36 (56) instructions for each token of
// 64 channels and 60 % of the issue slots: no one pipe is full.  One token of 256
// sequences of 2048 bf16 channels with a cache: 8.1 us, where its bytes take 2.3:
// it goes through a staged run and the token-by-token path like any other.
#include "sequence.cuh"

namespace gdn2 {

constexpr int HALO = 3;  // taps before a token
constexpr int CONV_WARPS = 4;

struct ConvParams {
  int B, T, C;
  int sets;   // sets of 64 channels
  int span;   // tokens of a warp's span
  int spans;  // spans of a sequence (of the packed buffer)
  const int* cu;
  DView x, y;  // y: out, or dy
  DView dx;
  const float* w;
  const float* cache_in;
  float* cache_out;
  const float* d_cache_out;
  float* d_cache_in;
  float* part;  // [gridDim.y][C][4]
};

// Where a warp is: a run of one of its spans.  `end`: one past the rows that
// the span walks (the adjoint three more than its own), `s1` past its own.
struct ConvWalk {
  int64_t unit;
  int b, s0, s1, end, t0;
  bool ok;
};
template <bool PACKED>
__device__ __forceinline__ ConvWalk conv_span(const ConvParams& p, int64_t unit, int behind) {
  ConvWalk w;
  w.unit = unit;
  w.ok = unit < (int64_t)p.spans * (PACKED ? 1 : p.B);
  w.b = PACKED ? 0 : (int)(unit / p.spans);
  w.s0 = w.t0 = (int)(PACKED ? unit : unit % p.spans) * p.span;
  w.s1 = w.s0 + p.span < p.T ? w.s0 + p.span : p.T;
  w.end = w.s1 + behind;
  return w;
}
template <bool PACKED>
__device__ __forceinline__ ConvWalk next_run(const ConvParams& p, ConvWalk w, int behind) {
  w.t0 += RUN;
  return w.t0 < w.end ? w : conv_span<PACKED>(p, w.unit + (int64_t)gridDim.y * CONV_WARPS, behind);
}

// What a run's tokens are: one bit a token; lane i holds the sequence and
// the first row of token i.
struct ConvRun {
  unsigned start, last, valid;
  int seq, first;
  __device__ __forceinline__ bool inside() const { return !start && !last && valid == (1u << RUN) - 1; }
};
template <bool PACKED>
__device__ __forceinline__ ConvRun conv_run(const ConvParams& p, int b, int t0, int lane) {
  const int t = t0 + lane;
  ConvRun k{0, 0, 0, -1, 0};
  bool l = false;
  if (lane < RUN && t < p.T) {
    if (PACKED) {
      k.seq = find_sequence(p.cu, p.B, t);
      if (k.seq >= 0) {
        k.first = max(__ldg(p.cu + k.seq), 0);  // rows before the buffer's are nobody's
        l = t + 1 == p.T || __ldg(p.cu + k.seq + 1) == t + 1;
      }
    } else {
      k.seq = b;
      l = t + 1 == p.T;
    }
  }
  k.valid = __ballot_sync(0xffffffffu, k.seq >= 0);
  k.start = __ballot_sync(0xffffffffu, k.seq >= 0 && k.first == t);
  k.last = __ballot_sync(0xffffffffu, l);
  return k;
}

// Row `slot` of a sequence's cache.
__device__ __forceinline__ int64_t cache_at(const ConvParams& p, int seq, int slot, int base) {
  return ((int64_t)seq * HALO + slot) * p.C + base;
}

// Empty sequences: the cache (its gradient) goes through; without one a new
// cache is zero.
template <RowMode MODE>
__device__ __forceinline__ void pass_empty(const ConvParams& p, const float* from, float* to, const Pair<MODE>& ch, int base) {
  const int lane = threadIdx.x & 31;
  for (int n0 = (int)threadIdx.x - lane; n0 < p.B; n0 += blockDim.x) {
    const int n = n0 + lane;
    unsigned empty = __ballot_sync(0xffffffffu, n < p.B && is_empty(p.cu, n, p.T));
    while (empty) {
      const int j = n0 + __ffs(empty) - 1;
      empty &= empty - 1;
      if (!ch.on0) continue;
      #pragma unroll
      for (int s = 0; s < HALO; ++s)
        ch.store_state(to + cache_at(p, j, s, base), from ? ch.load(from + cache_at(p, j, s, base)) : f2pk(0.f, 0.f));
    }
  }
}

// The three values before row t of sequence seq that begins at row first, oldest first; x at the set's first channel.
template <typename T, RowMode MODE>
__device__ __forceinline__ void window_before(const ConvParams& p, const T* x, int seq, int first, int t, int base,
                                              const Pair<MODE>& ch, f32x2 (&win)[HALO]) {
  #pragma unroll
  for (int i = 0; i < HALO; ++i) {
    const int row = t - HALO + i;
    if (row >= first) win[i] = ch.load(x + (int64_t)row * p.x.s1);
    else if (p.cache_in) win[i] = ch.load(p.cache_in + cache_at(p, seq, row - first + HALO, base));
    else win[i] = ch.load(x + (int64_t)first * p.x.s1);
  }
}

__device__ __forceinline__ f32x2 taps(const f32x2 (&win)[HALO], f32x2 x, const f32x2 (&w)[HALO + 1]) {
  return f2fma(x, w[3], f2fma(win[2], w[2], f2fma(win[1], w[1], f2mul(win[0], w[0]))));
}
__device__ __forceinline__ void slide(f32x2 (&win)[HALO], f32x2 x) {
  win[0] = win[1];
  win[1] = win[2];
  win[2] = x;
}
template <RowMode MODE>
__device__ __forceinline__ void load_taps(const ConvParams& p, int base, const Pair<MODE>& ch, f32x2 (&w)[HALO + 1]) {
  #pragma unroll
  for (int j = 0; j <= HALO; ++j)
    w[j] = f2pk(ch.on0 ? __ldg(p.w + (int64_t)(base + ch.c0) * (HALO + 1) + j) : 0.f,
                ch.on1 ? __ldg(p.w + (int64_t)(base + ch.c1) * (HALO + 1) + j) : 0.f);
}

template <typename T, RowMode MODE, bool PACKED>
__global__ void __launch_bounds__(32 * CONV_WARPS, 8) k_conv_fwd(const ConvParams p) {
  typedef Rows<T, MODE> R;
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int base = (int)blockIdx.x * SET;
  const Pair<MODE> ch(lane, p.C - base);
  if (PACKED && p.cache_out && blockIdx.y == 0) pass_empty(p, p.cache_in, p.cache_out, ch, base);
  f32x2 w[HALO + 1];
  load_taps(p, base, ch, w);

  auto rows = [&](int n) { return R{smem + ((n % STAGES) * CONV_WARPS + warp) * R::BYTES}; };
  auto x_of = [&](const ConvWalk& w) { return static_cast<const T*>(p.x.p) + w.b * p.x.s0 + base; };
  auto fetch = [&](const ConvWalk& w, int n) {
    if (w.ok) rows(n).fetch(x_of(w), p.x.s1, w.t0, p.T, p.C - base, lane);
    cp_async_commit();
  };
  ConvWalk at = conv_span<PACKED>(p, (int64_t)blockIdx.y * CONV_WARPS + warp, 0);
  fetch(at, 0);
  f32x2 win[HALO];
  for (int turn = 0; at.ok; ++turn) {
    const ConvWalk next = next_run<PACKED>(p, at, 0);
    __syncwarp();
    fetch(next, turn + 1);
    const int t0 = at.t0, s1 = at.s1;
    const T* x = x_of(at);
    const ConvRun k = conv_run<PACKED>(p, at.b, t0, lane);
    if (t0 == at.s0) {  // the tokens in front, of a span that begins inside a sequence
      #pragma unroll
      for (int i = 0; i < HALO; ++i) win[i] = f2pk(0.f, 0.f);
      const int seq = __shfl_sync(0xffffffffu, k.seq, 0), first = __shfl_sync(0xffffffffu, k.first, 0);
      if ((k.valid & 1) && !(k.start & 1)) window_before(p, x, seq, first, t0, base, ch, win);
    }
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const auto xs = rows(turn).view(x, p.x.s1, t0, lane);
    T* out = static_cast<T*>(const_cast<void*>(p.y.p)) + at.b * p.y.s0 + base + (int64_t)t0 * p.y.s1;
    at = next;
    if (k.inside() && t0 + RUN <= s1) {
      #pragma unroll
      for (int i = 0; i < RUN; ++i) {
        const f32x2 xf = xs.get(i), pre = taps(win, xf, w);
        if (ch.on0) ch.store(out, f2mul(pre, sigmoid2(pre)));
        out += p.y.s1;
        slide(win, xf);
      }
      continue;
    }
    #pragma unroll 1
    for (int i = 0; i < RUN && t0 + i < s1; ++i) {
      const int seq = __shfl_sync(0xffffffffu, k.seq, i);
      const f32x2 xf = xs.get(i);
      if ((k.start >> i) & 1) window_before(p, x, seq, t0 + i, t0 + i, base, ch, win);
      const f32x2 pre = taps(win, xf, w);
      if (ch.on0) ch.store(out, (k.valid >> i) & 1 ? f2mul(pre, sigmoid2(pre)) : f2pk(0.f, 0.f));
      out += p.y.s1;
      slide(win, xf);
      if (((k.last >> i) & 1) && p.cache_out && ch.on0)
        #pragma unroll
        for (int s = 0; s < HALO; ++s) ch.store_state(p.cache_out + cache_at(p, seq, s, base), win[s]);
    }
  }
}

// Adjoint.  Token s adds w[3-k] dpre_s to dx of token s - k, and to the
// gradient of the three values before its sequence where s - k lies there;
// the span that holds the sequence's first token collects those.
template <typename T, RowMode MODE, bool PACKED>
__global__ void __launch_bounds__(32 * CONV_WARPS, 4) k_conv_bwd(const ConvParams p) {
  typedef Rows<T, MODE> R;
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int base = (int)blockIdx.x * SET;
  const Pair<MODE> ch(lane, p.C - base);
  const f32x2 zero = f2pk(0.f, 0.f), one = f2pk(1.f, 1.f), minus = f2pk(-1.f, -1.f);
  if (PACKED && p.d_cache_in && blockIdx.y == 0) pass_empty(p, p.d_cache_out, p.d_cache_in, ch, base);
  f32x2 w[HALO + 1], dw[HALO + 1];
  load_taps(p, base, ch, w);
  #pragma unroll
  for (int j = 0; j <= HALO; ++j) dw[j] = zero;

  auto rows = [&](int n, int which) { return R{smem + (((n % STAGES) * CONV_WARPS + warp) * 2 + which) * R::BYTES}; };
  auto x_of = [&](const ConvWalk& w) { return static_cast<const T*>(p.x.p) + w.b * p.x.s0 + base; };
  auto dy_of = [&](const ConvWalk& w) { return static_cast<const T*>(p.y.p) + w.b * p.y.s0 + base; };
  auto fetch = [&](const ConvWalk& w, int n) {
    if (w.ok) {
      rows(n, 0).fetch(x_of(w), p.x.s1, w.t0, p.T, p.C - base, lane);
      rows(n, 1).fetch(dy_of(w), p.y.s1, w.t0, p.T, p.C - base, lane);
    }
    cp_async_commit();
  };
  ConvWalk at = conv_span<PACKED>(p, (int64_t)blockIdx.y * CONV_WARPS + warp, HALO);
  fetch(at, 0);
  f32x2 win[HALO], pend[HALO], before[HALO];
  int pos = HALO;      // place of the next token in its sequence, as far as the first three count
  bool owned = false;  // the sequence begins in this span
  for (int turn = 0; at.ok; ++turn) {
    const ConvWalk next = next_run<PACKED>(p, at, HALO);
    __syncwarp();
    fetch(next, turn + 1);
    const int t0 = at.t0, s0 = at.s0, s1 = at.s1, end = at.end;
    const T *x = x_of(at), *dy = dy_of(at);
    const ConvRun k = conv_run<PACKED>(p, at.b, t0, lane);
    if (t0 == s0) {
      #pragma unroll
      for (int i = 0; i < HALO; ++i) win[i] = pend[i] = before[i] = zero;
      pos = HALO;
      owned = false;
      const int seq = __shfl_sync(0xffffffffu, k.seq, 0), first = __shfl_sync(0xffffffffu, k.first, 0);
      if ((k.valid & 1) && !(k.start & 1)) {
        window_before(p, x, seq, first, t0, base, ch, win);
        pos = t0 - first;
      }
    }
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const auto xs = rows(turn, 0).view(x, p.x.s1, t0, lane);
    const auto ds = rows(turn, 1).view(dy, p.y.s1, t0, lane);
    T* out = static_cast<T*>(const_cast<void*>(p.dx.p)) + at.b * p.dx.s0 + base + (int64_t)(t0 - HALO) * p.dx.s1;
    at = next;
    // dpre of a token, and its part of dw where the token is the span's own
    auto adjoint = [&](f32x2 xf, f32x2 df, bool own) {
      const f32x2 pre = taps(win, xf, w), sig = sigmoid2(pre);
      const f32x2 dp = f2mul(df, f2mul(sig, f2fma(pre, f2fma(sig, minus, one), one)));
      if (own) {
        #pragma unroll
        for (int j = 0; j < HALO; ++j) dw[j] = f2fma(dp, win[j], dw[j]);
        dw[HALO] = f2fma(dp, xf, dw[HALO]);
      }
      return dp;
    };
    if (k.inside() && pos >= HALO) {
      #pragma unroll
      for (int i = 0; i < RUN; ++i) {
        const f32x2 xf = xs.get(i);
        const f32x2 dp = adjoint(xf, ds.get(i), i < RUN - HALO || t0 + i < s1);
        const f32x2 done = f2fma(w[0], dp, pend[2]);
        if (ch.on0 && (i >= HALO || t0 > s0)) ch.store(out, done);
        out += p.dx.s1;
        pend[2] = f2fma(w[1], dp, pend[1]);
        pend[1] = f2fma(w[2], dp, pend[0]);
        pend[0] = f2mul(w[3], dp);
        slide(win, xf);
      }
      continue;
    }
    #pragma unroll 1
    for (int i = 0; i < RUN && t0 + i < end; ++i) {
      const int seq = __shfl_sync(0xffffffffu, k.seq, i);
      const bool opens = (k.start >> i) & 1, closes = (k.last >> i) & 1, in = (k.valid >> i) & 1;
      const f32x2 xf = xs.get(i);
      if (opens) {
        pos = 0;
        owned = t0 + i < s1;
        window_before(p, x, seq, t0 + i, t0 + i, base, ch, win);
        before[0] = before[1] = before[2] = zero;
      }
      const f32x2 dp = in ? adjoint(xf, ds.get(i), t0 + i < s1) : zero;
      f32x2 part[HALO + 1] = {zero, pend[0], pend[1], pend[2]};  // dx of this token and the three before it
      auto give = [&](int j, f32x2 v) {  // to token s - j, or to what lies before the sequence
        if (pos >= j) part[j] = f2add(part[j], v);
        #pragma unroll
        for (int s = 0; s < HALO; ++s)
          if (pos < j && pos - j + HALO == s) before[s] = f2add(before[s], v);
      };
      if (in) {
        #pragma unroll
        for (int j = 0; j <= HALO; ++j) give(j, f2mul(w[HALO - j], dp));
        if (closes && p.d_cache_out) {  // the new cache holds the last three values
          #pragma unroll
          for (int j = 0; j < HALO; ++j)
            give(j, ch.load(p.d_cache_out + cache_at(p, seq, HALO - 1 - j, base)));
        }
        // no later token reaches before the sequence: hand on what does
        if (owned && (pos == HALO - 1 || (closes && pos < HALO - 1))) {
          if (p.d_cache_in) {
            if (ch.on0)
              #pragma unroll
              for (int s = 0; s < HALO; ++s) ch.store_state(p.d_cache_in + cache_at(p, seq, s, base), before[s]);
          } else if (!p.cache_in) {  // copies of the first token
            #pragma unroll
            for (int j = 0; j < HALO; ++j)
              if (pos == j) part[j] = f2add(part[j], f2add(before[0], f2add(before[1], before[2])));
          }
        }
      }
      const int row = t0 + i - HALO;
      if (ch.on0 && row >= s0 && row < s1) ch.store(out, part[HALO]);
      out += p.dx.s1;
      pend[0] = part[0];
      pend[1] = part[1];
      pend[2] = part[2];
      slide(win, xf);
      pos = pos < HALO ? pos + 1 : pos;
    }
  }
  if (!p.part) return;
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);  // [warp][channel][tap]
  #pragma unroll
  for (int j = 0; j <= HALO; ++j) {
    float d0, d1;
    f2un(dw[j], d0, d1);
    red[(warp * SET + ch.c0) * (HALO + 1) + j] = d0;
    red[(warp * SET + ch.c1) * (HALO + 1) + j] = d1;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < SET * (HALO + 1); e += 32 * CONV_WARPS) {
    if (base + e / (HALO + 1) >= p.C) continue;
    float s = 0.f;
    #pragma unroll
    for (int k = 0; k < CONV_WARPS; ++k) s += red[k * SET * (HALO + 1) + e];
    p.part[((int64_t)blockIdx.y * p.C + base) * (HALO + 1) + e] = s;
  }
}

// ---- host ----

static int check_conv(const gdn2_conv_args* a, const char* fn) {
  if (!a) return set_error(GDN2_EINVAL, "%s: null args", fn);
  if (a->batch <= 0 || a->seq_len < 0 || a->channels <= 0 || (a->seq_len == 0 && !a->cu_seqlens))
    return set_error(GDN2_EINVAL, "%s: sizes must be > 0 (batch=%d seq_len=%d channels=%d)", fn, a->batch, a->seq_len,
                     a->channels);
  if (a->seq_len > (1 << 30)) return set_error(GDN2_EUNSUPPORTED, "%s: seq_len=%d above 2^30", fn, a->seq_len);
  if (a->dtype != GDN2_DTYPE_F32 && a->dtype != GDN2_DTYPE_BF16)
    return set_error(GDN2_EINVAL, "%s: unknown dtype %d", fn, a->dtype);
  if ((a->seq_len && !a->x.data) || !a->weight) return set_error(GDN2_EINVAL, "%s: null tensor pointer", fn);
  return GDN2_OK;
}

// Blocks that an SM holds: by shared memory, and by registers 32 warps of a
// forward (64 a thread) and 16 of a backward (128).
constexpr int conv_resident(int bytes, bool bwd) {
  const int smem = STAGES * CONV_WARPS * bytes * (bwd ? 2 : 1) + 1024, by_smem = 227 * 1024 / smem;
  const int by_regs = (bwd ? 16 : 32) / CONV_WARPS;
  return by_smem < by_regs ? by_smem : by_regs;
}
static int conv_resident(RowMode mode, int e, bool bwd) {
  const bool shifted = mode == ROWS_PAIR || mode == ROWS_ODD;
  return conv_resident(RUN * (SET * e + (shifted ? 16 : 0)), bwd);
}

// How a call is cut up: how rows are held, spans of tokens and blocks along them.
struct ConvPlan {
  RowMode mode;
  int sets, span, spans, blocks;
};

// Spans of whole runs less `less` tokens.  Blocks (along the spans) as many as
// are resident, so that none waits for a second wave; span and blocks such that
// the warps with most to do have least: a span costs its runs and about half
// a run for its beginning.
static ConvPlan plan_conv(const gdn2_conv_args* a, RowMode mode, int less, int resident) {
  ConvPlan n;
  n.mode = mode;
  n.sets = (a->channels + SET - 1) / SET;
  const int rows = a->cu_seqlens ? 1 : a->batch;
  const int64_t most = 148 * (int64_t)resident / n.sets;
  int64_t best = -1;
  for (int runs = 16; runs >= 1; --runs) {
    const int span = runs * RUN - less;
    const int64_t spans = (a->seq_len + span - 1) / span, units = spans * rows;
    int64_t blocks = (units + CONV_WARPS - 1) / CONV_WARPS;
    if (blocks > most) blocks = most;
    if (blocks < 1) blocks = 1;
    if (blocks > 65535) blocks = 65535;
    const int64_t rounds = (units + blocks * CONV_WARPS - 1) / (blocks * CONV_WARPS), cost = rounds * (2 * runs + 1);
    if (best >= 0 && cost >= best) continue;
    best = cost;
    n.span = span;
    n.spans = (int)spans;
    n.blocks = (int)blocks;
  }
  return n;
}

static void fill_conv(ConvParams& p, const gdn2_conv_args* a, const ConvPlan& n) {
  p = ConvParams{};
  p.B = a->batch; p.T = a->seq_len; p.C = a->channels;
  p.sets = n.sets; p.span = n.span; p.spans = n.spans;
  p.cu = a->cu_seqlens;
  p.x = make_dview(a->x);
  p.w = a->weight;
  p.cache_in = a->cache_in;
}

template <typename K>
static int launch_conv(K kernel, const ConvParams& p, const ConvPlan& n, int stage, cudaStream_t st, const char* fn) {
  const int smem = STAGES * CONV_WARPS * stage;
  int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), fn);
  if (rc) return rc;
  kernel<<<dim3(n.sets, n.blocks), 32 * CONV_WARPS, smem, st>>>(p);
  return check_cuda(cudaGetLastError(), fn);
}

template <typename T, RowMode MODE>
static int run_conv(const ConvParams& p, const ConvPlan& n, bool bwd, cudaStream_t st, const char* fn) {
  const int bytes = Rows<T, MODE>::BYTES;
  if (bwd)
    return p.cu ? launch_conv(k_conv_bwd<T, MODE, true>, p, n, 2 * bytes, st, fn)
                : launch_conv(k_conv_bwd<T, MODE, false>, p, n, 2 * bytes, st, fn);
  return p.cu ? launch_conv(k_conv_fwd<T, MODE, true>, p, n, bytes, st, fn)
              : launch_conv(k_conv_fwd<T, MODE, false>, p, n, bytes, st, fn);
}

template <typename T>
static int dispatch_conv(const ConvParams& p, const ConvPlan& n, bool bwd, cudaStream_t st, const char* fn) {
  return n.mode == ROWS16      ? run_conv<T, ROWS16>(p, n, bwd, st, fn)
         : n.mode == ROWS_PAIR ? run_conv<T, ROWS_PAIR>(p, n, bwd, st, fn)
         : n.mode == ROWS_ODD  ? run_conv<T, ROWS_ODD>(p, n, bwd, st, fn)
                               : run_conv<T, ROWS_ANY>(p, n, bwd, st, fn);
}

int launch_conv_fwd(const gdn2_conv_args* a, const gdn2_view& y, float* cache_out, cudaStream_t st) {
  const char* fn = "gdn2_causal_conv";
  int rc = check_conv(a, fn);
  if (rc) return rc;
  if (a->seq_len && !y.data) return set_error(GDN2_EINVAL, "%s: null tensor pointer", fn);
  const int e = elem_bytes(a->dtype);
  const RowTensor t[] = {{&a->x, e, true}, {&y, e, false}};
  const RowMode mode = row_mode(a->channels, t, 2);
  const ConvPlan n = plan_conv(a, mode, 0, conv_resident(mode, e, false));
  ConvParams p;
  fill_conv(p, a, n);
  p.y = make_dview(y);
  p.cache_out = cache_out;
  return a->dtype == GDN2_DTYPE_F32 ? dispatch_conv<float>(p, n, false, st, fn)
                                    : dispatch_conv<__nv_bfloat16>(p, n, false, st, fn);
}

static ConvPlan plan_conv_bwd(const gdn2_conv_bwd_args* q) {
  const gdn2_conv_args* a = &q->fwd;
  const int e = elem_bytes(a->dtype);
  const RowTensor t[] = {{&a->x, e, true}, {&q->d_y, e, true}, {&q->dx, e, false}};
  const RowMode mode = row_mode(a->channels, t, 3);
  return plan_conv(a, mode, HALO, conv_resident(mode, e, true));
}

size_t conv_bwd_workspace_bytes(const gdn2_conv_bwd_args* q) {
  if (!q || check_conv(&q->fwd, "gdn2_causal_conv_bwd_workspace_bytes") || !q->d_weight) return 0;
  return (size_t)plan_conv_bwd(q).blocks * q->fwd.channels * (HALO + 1) * sizeof(float);
}

int launch_column_sums(const float* part, int64_t rows, int cols, int arrays, float* out0, float* out1,
                       cudaStream_t st, const char* fn);

int launch_conv_bwd(const gdn2_conv_bwd_args* q, void* ws, size_t ws_bytes, cudaStream_t st) {
  const char* fn = "gdn2_causal_conv_bwd";
  if (!q) return set_error(GDN2_EINVAL, "%s: null args", fn);
  const gdn2_conv_args* a = &q->fwd;
  int rc = check_conv(a, fn);
  if (rc) return rc;
  if (a->seq_len && (!q->d_y.data || !q->dx.data)) return set_error(GDN2_EINVAL, "%s: null tensor pointer", fn);
  if (q->d_cache_in && !a->cache_in)
    return set_error(GDN2_EINVAL, "%s: the gradient of a cache that is not there", fn);
  if (a->channels > 0x7fffffff / (HALO + 1)) return set_error(GDN2_EUNSUPPORTED, "%s: %d channels", fn, a->channels);
  const size_t need = conv_bwd_workspace_bytes(q);
  if (need && (!ws || ws_bytes < need))
    return set_error(GDN2_EWORKSPACE, "%s: workspace %zu bytes < required %zu", fn, ws ? ws_bytes : 0, need);
  const ConvPlan n = plan_conv_bwd(q);
  ConvParams p;
  fill_conv(p, a, n);
  p.y = make_dview(q->d_y);
  p.dx = make_dview(q->dx);
  p.d_cache_out = q->d_cache_out;
  p.d_cache_in = q->d_cache_in;
  p.part = need ? static_cast<float*>(ws) : nullptr;
  rc = a->dtype == GDN2_DTYPE_F32 ? dispatch_conv<float>(p, n, true, st, fn)
                                  : dispatch_conv<__nv_bfloat16>(p, n, true, st, fn);
  if (rc || !need) return rc;
  return launch_column_sums(p.part, n.blocks, p.C * (HALO + 1), 1, q->d_weight, nullptr, st, fn);
}

}  // namespace gdn2

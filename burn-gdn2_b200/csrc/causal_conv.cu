// Causal depthwise convolution of four taps with SiLU over dense or packed
// sequences, and its adjoint:
//
//   pre_t = sum_j w[c][j] x_{t-3+j},  y_t = silu(pre_t)
//   dpre_t = dy_t silu'(pre_t),  dx_t = sum_k w[c][3-k] dpre_{t+k},  dw[c][j] = sum_t dpre_t x_{t-3+j}
//
// The three tokens before a sequence are its cache, or copies of its first
// token (src/short_conv.rs:42-54).  Bound by HBM: x in and y out, or x and dy
// in and dx out.  A warp takes RUN tokens of 32 * VEC channels with all their
// rows in flight, and the three rows in front (behind too, in the adjoint)
// once more, which neighbouring warps have just read.  The adjoint forms pre
// again from x; each lane sums dw over the runs that its block walks, the
// block adds its warps' sums and a second kernel the blocks', in a fixed
// order.
#include "scan.cuh"

namespace gdn2 {

constexpr int HALO = 3;  // taps before a token
constexpr int CONV_RUN = 16, CONV_WARPS = 4;

struct ConvParams {
  int B, T, C;
  int runs, sets;
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

// Where a token lies in its sequence: number and first row (dense: its batch row and 0).
struct Place {
  int seq, first, end;
};
template <bool PACKED>
__device__ __forceinline__ Place place_of(const ConvParams& p, int b, int t) {
  if (!PACKED) return Place{t < p.T ? b : -1, 0, p.T};
  Place q{-1, 0, 0};
  if (t < p.T) {
    q.seq = find_sequence(p.cu, p.B, t);
    if (q.seq >= 0) {
      q.first = __ldg(p.cu + q.seq);
      q.end = __ldg(p.cu + q.seq + 1);
      if (q.end > p.T) q.end = p.T;
    }
  }
  return q;
}

template <int VEC>
__device__ __forceinline__ const float* cache_row(const float* cache, int seq, int slot, int C, int c0) {
  return cache + ((int64_t)seq * HALO + slot) * C + c0;
}

// Empty sequences: the cache (its gradient) goes through; without one a new
// cache is zero.
template <int VEC>
__device__ __forceinline__ void pass_empty(const ConvParams& p, const float* from, float* to, int c0, bool on,
                                           int warp, int lane) {
  for (int n0 = warp * 32; n0 < p.B; n0 += 32 * CONV_WARPS) {
    const int n = n0 + lane;
    bool e = false;
    if (n < p.B) {
      const int a = __ldg(p.cu + n);
      e = __ldg(p.cu + n + 1) <= a || a >= p.T;
    }
    unsigned empty = __ballot_sync(0xffffffffu, e);
    while (empty) {
      const int j = n0 + __ffs(empty) - 1;
      empty &= empty - 1;
      if (!on) continue;
      #pragma unroll
      for (int s = 0; s < HALO; ++s) {
        float v[VEC] = {};
        if (from) load_f32<VEC>(cache_row<VEC>(from, j, s, p.C, c0), v);
        store_f32<VEC>(to + ((int64_t)j * HALO + s) * p.C + c0, v);
      }
    }
  }
}

// The three values before row t of a sequence, oldest first.
template <typename T, int VEC>
__device__ __forceinline__ void window_before(const ConvParams& p, const T* x, const Place& q, int t, int c0,
                                              float (&win)[HALO][VEC]) {
  #pragma unroll
  for (int i = 0; i < HALO; ++i) {
    const int row = t - HALO + i;
    if (row >= q.first)
      Vec<T, VEC>::unpack(Vec<T, VEC>::load(x + (int64_t)row * p.x.s1), win[i]);
    else if (p.cache_in)
      load_f32<VEC>(cache_row<VEC>(p.cache_in, q.seq, row - q.first + HALO, p.C, c0), win[i]);
    else
      Vec<T, VEC>::unpack(Vec<T, VEC>::load(x + (int64_t)q.first * p.x.s1), win[i]);
  }
}

template <typename T, int VEC, bool PACKED>
__global__ void __launch_bounds__(32 * CONV_WARPS) k_conv_fwd(ConvParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t chain = blockIdx.x;
  const int b = (int)(chain / p.sets);
  const int c0 = (int)(chain % p.sets) * 32 * VEC + lane * VEC;
  const bool on = c0 < p.C;
  const T* x = static_cast<const T*>(p.x.p) + (PACKED ? 0 : (int64_t)b * p.x.s0) + c0;
  T* y = static_cast<T*>(const_cast<void*>(p.y.p)) + (PACKED ? 0 : (int64_t)b * p.y.s0) + c0;
  if (PACKED && p.cache_out && blockIdx.y == 0) pass_empty<VEC>(p, p.cache_in, p.cache_out, c0, on, warp, lane);

  float w[VEC][HALO + 1];
  #pragma unroll
  for (int v = 0; v < VEC; ++v)
    #pragma unroll
    for (int j = 0; j <= HALO; ++j) w[v][j] = on ? __ldg(p.w + (int64_t)(c0 + v) * (HALO + 1) + j) : 0.f;

  for (int run = blockIdx.y * CONV_WARPS + warp; run < p.runs; run += gridDim.y * CONV_WARPS) {
    const int t0 = run * CONV_RUN;
    typename Vec<T, VEC>::Raw xr[CONV_RUN];
    #pragma unroll
    for (int i = 0; i < CONV_RUN; ++i) {
      xr[i] = typename Vec<T, VEC>::Raw{};
      if (on && t0 + i < p.T) xr[i] = Vec<T, VEC>::load(x + (int64_t)(t0 + i) * p.x.s1);
    }
    // lane i: the place of token i
    const Place mine = place_of<PACKED>(p, b, lane < CONV_RUN ? t0 + lane : p.T);
    const unsigned valid = __ballot_sync(0xffffffffu, mine.seq >= 0);
    const unsigned start = __ballot_sync(0xffffffffu, mine.seq >= 0 && mine.first == t0 + lane);
    const unsigned last = __ballot_sync(0xffffffffu, mine.seq >= 0 && mine.end == t0 + lane + 1);
    float win[HALO][VEC] = {};
    if (valid & 1) {
      const Place q{__shfl_sync(0xffffffffu, mine.seq, 0), __shfl_sync(0xffffffffu, mine.first, 0), 0};
      if (on) window_before<T, VEC>(p, x, q, t0, c0, win);
    }
    #pragma unroll
    for (int i = 0; i < CONV_RUN; ++i) {
      float xf[VEC], out[VEC];
      Vec<T, VEC>::unpack(xr[i], xf);
      if (PACKED && i && ((start >> i) & 1)) {
        const Place q{__shfl_sync(0xffffffffu, mine.seq, i), t0 + i, 0};
        if (on) window_before<T, VEC>(p, x, q, t0 + i, c0, win);
      }
      #pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float s = win[0][v] * w[v][0];
        s = fmaf(win[1][v], w[v][1], s);
        s = fmaf(win[2][v], w[v][2], s);
        s = fmaf(xf[v], w[v][3], s);
        out[v] = !PACKED || ((valid >> i) & 1) ? silu_f(s) : 0.f;
        win[0][v] = win[1][v];
        win[1][v] = win[2][v];
        win[2][v] = xf[v];
      }
      if (on && t0 + i < p.T) Vec<T, VEC>::store(y + (int64_t)(t0 + i) * p.y.s1, out);
      if (((last >> i) & 1) && p.cache_out) {
        const int n = __shfl_sync(0xffffffffu, mine.seq, i);
        if (on)
          #pragma unroll
          for (int s = 0; s < HALO; ++s)
            store_f32<VEC>(p.cache_out + ((int64_t)n * HALO + s) * p.C + c0, win[s]);
      }
    }
  }
}

// Adjoint.  A run's tokens are walked with the three behind it; token s adds
// w[3-k] dpre_s to dx of token s - k, and to the cache's (or the first
// token's) gradient where s - k lies before its sequence, which the run that
// holds the sequence's first token collects.
template <typename T, int VEC, bool PACKED>
__global__ void __launch_bounds__(32 * CONV_WARPS) k_conv_bwd(ConvParams p) {
  __shared__ float red[CONV_WARPS][32 * VEC][HALO + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t chain = blockIdx.x;  // set of channels (all sequences of a dense batch are walked by one grid column)
  const int c0 = (int)chain * 32 * VEC + lane * VEC;
  const bool on = c0 < p.C;
  if (PACKED && p.d_cache_in && blockIdx.y == 0) pass_empty<VEC>(p, p.d_cache_out, p.d_cache_in, c0, on, warp, lane);

  float w[VEC][HALO + 1], dw[VEC][HALO + 1];
  #pragma unroll
  for (int v = 0; v < VEC; ++v)
    #pragma unroll
    for (int j = 0; j <= HALO; ++j) {
      w[v][j] = on ? __ldg(p.w + (int64_t)(c0 + v) * (HALO + 1) + j) : 0.f;
      dw[v][j] = 0.f;
    }

  const int64_t all = PACKED ? p.runs : (int64_t)p.runs * p.B;
  for (int64_t unit = (int64_t)blockIdx.y * CONV_WARPS + warp; unit < all; unit += (int64_t)gridDim.y * CONV_WARPS) {
    const int b = PACKED ? 0 : (int)(unit / p.runs);
    const int t0 = (int)(PACKED ? unit : unit % p.runs) * CONV_RUN;
    const T* x = static_cast<const T*>(p.x.p) + (PACKED ? 0 : (int64_t)b * p.x.s0) + c0;
    const T* dy = static_cast<const T*>(p.y.p) + (PACKED ? 0 : (int64_t)b * p.y.s0) + c0;
    T* dx = static_cast<T*>(const_cast<void*>(p.dx.p)) + (PACKED ? 0 : (int64_t)b * p.dx.s0) + c0;
    constexpr int N = CONV_RUN + HALO;
    typename Vec<T, VEC>::Raw xr[N], dr[N];
    #pragma unroll
    for (int i = 0; i < N; ++i) {
      xr[i] = dr[i] = typename Vec<T, VEC>::Raw{};
      if (on && t0 + i < p.T) {
        xr[i] = Vec<T, VEC>::load(x + (int64_t)(t0 + i) * p.x.s1);
        dr[i] = Vec<T, VEC>::load(dy + (int64_t)(t0 + i) * p.y.s1);
      }
    }
    const Place mine = place_of<PACKED>(p, b, lane < N ? t0 + lane : p.T);
    const unsigned valid = __ballot_sync(0xffffffffu, mine.seq >= 0);
    const unsigned start = __ballot_sync(0xffffffffu, mine.seq >= 0 && mine.first == t0 + lane);
    const unsigned last = __ballot_sync(0xffffffffu, mine.seq >= 0 && mine.end == t0 + lane + 1);
    float win[HALO][VEC] = {};
    if (valid & 1) {
      const Place q{__shfl_sync(0xffffffffu, mine.seq, 0), __shfl_sync(0xffffffffu, mine.first, 0), 0};
      if (on) window_before<T, VEC>(p, x, q, t0, c0, win);
    }
    int pos = HALO;  // place of the token in its sequence, as far as the first three count
    if (valid & 1) pos = t0 - __shfl_sync(0xffffffffu, mine.first, 0);
    bool owned = false;  // the sequence began in this run
    float pend[HALO + 1][VEC] = {};  // dx of tokens s, s - 1, s - 2, s - 3 as far as it is summed
    float before[HALO][VEC] = {};    // gradient of the three values before the sequence
    #pragma unroll
    for (int i = 0; i < N; ++i) {
      float xf[VEC], df[VEC];
      Vec<T, VEC>::unpack(xr[i], xf);
      Vec<T, VEC>::unpack(dr[i], df);
      const bool opens = (start >> i) & 1, closes = (last >> i) & 1, in = (valid >> i) & 1;
      if (opens) {
        pos = 0;
        owned = i < CONV_RUN;
        if (i) {
          const Place q{__shfl_sync(0xffffffffu, mine.seq, i), t0 + i, 0};
          if (on) window_before<T, VEC>(p, x, q, t0 + i, c0, win);
        }
        #pragma unroll
        for (int s = 0; s < HALO; ++s)
          #pragma unroll
          for (int v = 0; v < VEC; ++v) before[s][v] = 0.f;
      }
      #pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float pre = win[0][v] * w[v][0];
        pre = fmaf(win[1][v], w[v][1], pre);
        pre = fmaf(win[2][v], w[v][2], pre);
        pre = fmaf(xf[v], w[v][3], pre);
        const float sig = __fdividef(1.f, 1.f + __expf(-pre));
        const float dp = in ? df[v] * (sig * fmaf(pre, 1.f - sig, 1.f)) : 0.f;
        if (i < CONV_RUN && in) {
          dw[v][0] = fmaf(dp, win[0][v], dw[v][0]);
          dw[v][1] = fmaf(dp, win[1][v], dw[v][1]);
          dw[v][2] = fmaf(dp, win[2][v], dw[v][2]);
          dw[v][3] = fmaf(dp, xf[v], dw[v][3]);
        }
        win[0][v] = win[1][v];
        win[1][v] = win[2][v];
        win[2][v] = xf[v];
        pend[3][v] = pend[2][v];
        pend[2][v] = pend[1][v];
        pend[1][v] = pend[0][v];
        pend[0][v] = 0.f;
        #pragma unroll
        for (int k = 0; k <= HALO; ++k) {
          const float add = w[v][HALO - k] * dp;
          if (pos >= k) pend[k][v] += add;
          else
            #pragma unroll
            for (int s = 0; s < HALO; ++s)  // value s of the three before: pos - k = s - 3
              if (pos - k + HALO == s) before[s][v] += add;
        }
      }
      if (closes && p.d_cache_out) {  // the new cache holds the last three values
        const int n = __shfl_sync(0xffffffffu, mine.seq, i);
        if (on)
          #pragma unroll
          for (int k = 0; k < HALO; ++k) {
            float d[VEC];
            load_f32<VEC>(cache_row<VEC>(p.d_cache_out, n, HALO - 1 - k, p.C, c0), d);
            #pragma unroll
            for (int v = 0; v < VEC; ++v) {
              if (pos >= k) pend[k][v] += d[v];
              else
                #pragma unroll
                for (int s = 0; s < HALO; ++s)
                  if (pos - k + HALO == s) before[s][v] += d[v];
            }
          }
      }
      // the sequence's first tokens are past (no later token reaches before it): hand on what lies before it
      if (owned && in && (pos == HALO - 1 || (closes && pos < HALO - 1))) {
        const int n = __shfl_sync(0xffffffffu, mine.seq, i);
        if (p.d_cache_in) {
          if (on)
            #pragma unroll
            for (int s = 0; s < HALO; ++s)
              store_f32<VEC>(p.d_cache_in + ((int64_t)n * HALO + s) * p.C + c0, before[s]);
        } else if (!p.cache_in) {  // copies of the first token
          #pragma unroll
          for (int v = 0; v < VEC; ++v)
            #pragma unroll
            for (int k = 0; k < HALO; ++k)
              if (pos == k) pend[k][v] += before[0][v] + before[1][v] + before[2][v];
        }
      }
      if (i >= HALO && on && t0 + i - HALO < p.T) Vec<T, VEC>::store(dx + (int64_t)(t0 + i - HALO) * p.dx.s1, pend[HALO]);
      pos = pos < HALO ? pos + 1 : pos;
    }
  }
  if (!p.part) return;
  #pragma unroll
  for (int v = 0; v < VEC; ++v)
    #pragma unroll
    for (int j = 0; j <= HALO; ++j) red[warp][lane * VEC + v][j] = dw[v][j];
  __syncthreads();
  for (int e = threadIdx.x; e < 32 * VEC * (HALO + 1); e += 32 * CONV_WARPS) {
    const int c = e / (HALO + 1), j = e % (HALO + 1);
    const int at = (int)chain * 32 * VEC + c;
    if (at >= p.C) continue;
    float s = 0.f;
    #pragma unroll
    for (int k = 0; k < CONV_WARPS; ++k) s += red[k][c][j];
    p.part[((int64_t)blockIdx.y * p.C + at) * (HALO + 1) + j] = s;
  }
}

// ---- host ----

static bool conv_rows_ok(const gdn2_view& v, int vec, int elem) {
  return (uintptr_t)v.data % (vec * elem) == 0 && v.stride0 % vec == 0 && v.stride1 % vec == 0;
}

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

static void fill_conv(ConvParams& p, const gdn2_conv_args* a, int vec) {
  p = ConvParams{};
  p.B = a->batch; p.T = a->seq_len; p.C = a->channels;
  p.runs = (p.T + CONV_RUN - 1) / CONV_RUN;
  p.sets = (p.C + 32 * vec - 1) / (32 * vec);
  p.cu = a->cu_seqlens;
  p.x = make_dview(a->x);
  p.w = a->weight;
  p.cache_in = a->cache_in;
}

template <typename T, int VEC>
static int run_conv_fwd(const ConvParams& p, cudaStream_t st, const char* fn) {
  const int64_t chains = p.cu ? p.sets : (int64_t)p.B * p.sets;
  if (chains > 0x7fffffffll) return set_error(GDN2_EUNSUPPORTED, "%s: too many channels", fn);
  int gy = (p.runs + CONV_WARPS - 1) / CONV_WARPS;
  gy = gy < 1 ? 1 : gy > 65535 ? 65535 : gy;
  const dim3 grid((unsigned)chains, gy);
  if (p.cu) k_conv_fwd<T, VEC, true><<<grid, 32 * CONV_WARPS, 0, st>>>(p);
  else k_conv_fwd<T, VEC, false><<<grid, 32 * CONV_WARPS, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), fn);
}

int launch_conv_fwd(const gdn2_conv_args* a, const gdn2_view& y, float* cache_out, cudaStream_t st) {
  const char* fn = "gdn2_causal_conv";
  int rc = check_conv(a, fn);
  if (rc) return rc;
  if (a->seq_len && !y.data) return set_error(GDN2_EINVAL, "%s: null tensor pointer", fn);
  const int elem = a->dtype == GDN2_DTYPE_BF16 ? 2 : 4;
  const bool pairs = a->channels % 2 == 0 && conv_rows_ok(a->x, 2, elem) && conv_rows_ok(y, 2, elem);
  ConvParams p;
  fill_conv(p, a, pairs ? 2 : 1);
  p.y = make_dview(y);
  p.cache_out = cache_out;
  if (a->dtype == GDN2_DTYPE_F32)
    return pairs ? run_conv_fwd<float, 2>(p, st, fn) : run_conv_fwd<float, 1>(p, st, fn);
  return pairs ? run_conv_fwd<__nv_bfloat16, 2>(p, st, fn) : run_conv_fwd<__nv_bfloat16, 1>(p, st, fn);
}

// Blocks along the runs of a channel set in the adjoint: each leaves one partial row of dw.
static int conv_bwd_blocks(const gdn2_conv_args* a, int sets) {
  const int64_t runs = (int64_t)((a->seq_len + CONV_RUN - 1) / CONV_RUN) * (a->cu_seqlens ? 1 : a->batch);
  const int64_t most = (runs + CONV_WARPS - 1) / CONV_WARPS;
  int64_t want = (148 * 4 + sets - 1) / sets;
  want = want < most ? want : most;
  return (int)(want < 1 ? 1 : want);
}

static bool conv_bwd_pairs(const gdn2_conv_bwd_args* q) {
  const int elem = q->fwd.dtype == GDN2_DTYPE_BF16 ? 2 : 4;
  return q->fwd.channels % 2 == 0 && conv_rows_ok(q->fwd.x, 2, elem) && conv_rows_ok(q->d_y, 2, elem) &&
         conv_rows_ok(q->dx, 2, elem);
}

static int conv_sets(int C, bool pairs) { return pairs ? (C + 63) / 64 : (C + 31) / 32; }

size_t conv_bwd_workspace_bytes(const gdn2_conv_bwd_args* q) {
  if (!q || check_conv(&q->fwd, "gdn2_causal_conv_bwd_workspace_bytes")) return 0;
  if (!q->d_weight) return 0;
  const int sets = conv_sets(q->fwd.channels, conv_bwd_pairs(q));
  return (size_t)conv_bwd_blocks(&q->fwd, sets) * q->fwd.channels * (HALO + 1) * sizeof(float);
}

template <typename T, int VEC>
static int run_conv_bwd(const ConvParams& p, int gy, cudaStream_t st, const char* fn) {
  const dim3 grid((unsigned)p.sets, gy);
  if (p.cu) k_conv_bwd<T, VEC, true><<<grid, 32 * CONV_WARPS, 0, st>>>(p);
  else k_conv_bwd<T, VEC, false><<<grid, 32 * CONV_WARPS, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), fn);
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
  const bool pairs = conv_bwd_pairs(q);
  ConvParams p;
  fill_conv(p, a, pairs ? 2 : 1);
  p.y = make_dview(q->d_y);
  p.dx = make_dview(q->dx);
  p.d_cache_out = q->d_cache_out;
  p.d_cache_in = q->d_cache_in;
  p.part = need ? static_cast<float*>(ws) : nullptr;
  const int gy = conv_bwd_blocks(a, p.sets);
  if (a->dtype == GDN2_DTYPE_F32)
    rc = pairs ? run_conv_bwd<float, 2>(p, gy, st, fn) : run_conv_bwd<float, 1>(p, gy, st, fn);
  else
    rc = pairs ? run_conv_bwd<__nv_bfloat16, 2>(p, gy, st, fn) : run_conv_bwd<__nv_bfloat16, 1>(p, gy, st, fn);
  if (rc || !need) return rc;
  return launch_column_sums(p.part, gy, p.C * (HALO + 1), 1, q->d_weight, nullptr, st, fn);
}

}  // namespace gdn2

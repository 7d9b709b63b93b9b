// Group norm of each token's channels, channels last, with its affine map
// and a SiLU, and the adjoint.  For a row's group of `width` channels
//
//   n = (x - mean) rstd    rstd = 1 / sqrt(mean((x - mean)^2) + eps)   (mean = 0 without center)
//   z = n w + b,           y = z silu(gate),  or silu(z) without a gate
//
//   dz = dy silu(gate) (or dy silu'(z)),  dgate = dy z silu'(gate),  dw = sum dz n,  db = sum dz
//   dn = dz w,  dx = rstd (dn - mean(dn) - n mean(dn n))
//
// Bound by HBM: x and gate in, y out (dy in and dx, dgate out besides).  A
// group's values stay in the registers of L neighbouring lanes (or of the
// whole block for wide groups) from the load to the store, so everything is
// read once, statistics included: they are formed in two steps (mean, then
// squares of deviations) from registers, without the cancellation of
// E[x^2] - mean^2, and the backward forms them again rather than read them.
// A lane keeps its group for all its rows, so the affine weights and the sums
// of their gradients stay in registers too.  Those sums leave through one
// partial row per slot of lanes, added up by a second kernel in a fixed
// order: no atomics.
#include "scan.cuh"

namespace gdn2 {

constexpr int NORM_THREADS = 256;

struct NormParams {
  int64_t rows;
  int G, D, nv;          // groups, channels of each, vectors of each
  int L;                 // lanes of a group (the block in block mode)
  int slots;             // groups a block takes at a time
  int per_row, row_step; // of those, groups of one row; rows at a time
  int shared_w;          // weights [D] for all groups, else [G * D]
  int center;
  float eps;
  const void *x, *gate, *dy;
  void *y, *dx, *dgate;
  int64_t ldx, ldgate, lddy;
  const float *w, *b;
  float* part;           // [2][gridDim.y * row_step][G * D] partial dw, db
  int want_w, want_b;
};

// Sums of up to two values over a group's lanes (the block, in block mode).
template <bool BLOCK, int N>
__device__ __forceinline__ void group_sum(float (&s)[N], int L, float* red) {
  for (int o = BLOCK ? 16 : L >> 1; o > 0; o >>= 1)
    #pragma unroll
    for (int k = 0; k < N; ++k) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
  if (BLOCK) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
      #pragma unroll
      for (int k = 0; k < N; ++k) red[k * 8 + (threadIdx.x >> 5)] = s[k];
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < N; ++k) {
      s[k] = 0.f;
      #pragma unroll
      for (int i = 0; i < NORM_THREADS / 32; ++i) s[k] += red[k * 8 + i];
    }
  }
}

__device__ __forceinline__ float sigmoid_f(float t) { return __fdividef(1.f, 1.f + __expf(-t)); }

template <typename T, int VEC, int KV, bool BLOCK, bool GATE, bool BWD>
__global__ void __launch_bounds__(NORM_THREADS) k_group_norm(NormParams p) {
  __shared__ float red[16];
  const int slot = BLOCK ? 0 : threadIdx.x / p.L;
  const int lane = BLOCK ? threadIdx.x : threadIdx.x % p.L;
  const int group = blockIdx.x * p.per_row + slot % p.per_row;
  const int row0 = slot / p.per_row;
  const bool used = group < p.G && row0 < p.row_step;
  const int64_t col = (int64_t)group * p.D + lane * VEC;
  const int step = p.L * VEC;  // channels between a lane's vectors
  const float inv = 1.f / (float)p.D;

  float w[KV][VEC], b[KV][VEC], dw[KV][VEC], db[KV][VEC];
  #pragma unroll
  for (int k = 0; k < KV; ++k)
    #pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const bool in = used && k * p.L + lane < p.nv;
      const int64_t c = (p.shared_w ? 0 : (int64_t)group * p.D) + lane * VEC + k * step + v;
      w[k][v] = in && p.w ? __ldg(p.w + c) : 1.f;
      b[k][v] = in && p.b ? __ldg(p.b + c) : 0.f;
      dw[k][v] = db[k][v] = 0.f;
    }

  // every thread of a warp (of the block) takes part in the sums of each round
  const int64_t rounds = (p.rows + p.row_step - 1) / p.row_step;
  for (int64_t r = blockIdx.y; r < rounds; r += gridDim.y) {
    const int64_t row = r * p.row_step + row0;
    const bool on = used && row < p.rows;
    const T* xp = static_cast<const T*>(p.x) + row * p.ldx + col;
    const T* gp = GATE ? static_cast<const T*>(p.gate) + row * p.ldgate + col : nullptr;
    const T* dp = BWD ? static_cast<const T*>(p.dy) + row * p.lddy + col : nullptr;
    typename Vec<T, VEC>::Raw xr[KV], gr[KV], dr[KV];
    #pragma unroll
    for (int k = 0; k < KV; ++k) {
      xr[k] = gr[k] = dr[k] = typename Vec<T, VEC>::Raw{};
      if (on && k * p.L + lane < p.nv) {
        xr[k] = Vec<T, VEC>::load(xp + k * step);
        if (GATE) gr[k] = Vec<T, VEC>::load(gp + k * step);
        if (BWD) dr[k] = Vec<T, VEC>::load(dp + k * step);
      }
    }
    float x[KV][VEC];
    float s[1] = {0.f};
    #pragma unroll
    for (int k = 0; k < KV; ++k) {
      Vec<T, VEC>::unpack(xr[k], x[k]);
      #pragma unroll
      for (int v = 0; v < VEC; ++v) s[0] += x[k][v];
    }
    float mean = 0.f;
    if (p.center) {
      group_sum<BLOCK, 1>(s, p.L, red);
      mean = s[0] * inv;
    }
    s[0] = 0.f;
    #pragma unroll
    for (int k = 0; k < KV; ++k)
      #pragma unroll
      for (int v = 0; v < VEC; ++v) {
        x[k][v] = k * p.L + lane < p.nv ? x[k][v] - mean : 0.f;
        s[0] = fmaf(x[k][v], x[k][v], s[0]);
      }
    group_sum<BLOCK, 1>(s, p.L, red);
    const float rstd = rsqrtf(fmaf(s[0], inv, p.eps));

    if (!BWD) {
      T* yp = static_cast<T*>(p.y) + row * (int64_t)p.G * p.D + col;
      #pragma unroll
      for (int k = 0; k < KV; ++k) {
        float t[VEC], y[VEC];
        if (GATE) Vec<T, VEC>::unpack(gr[k], t);
        #pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float z = fmaf(x[k][v] * rstd, w[k][v], b[k][v]);
          if (!GATE) t[v] = z;
          const float act = t[v] * sigmoid_f(t[v]);
          y[v] = GATE ? z * act : act;
        }
        if (on && k * p.L + lane < p.nv) Vec<T, VEC>::store(yp + k * step, y);
      }
      continue;
    }
    float dn[KV][VEC];
    float q[2] = {0.f, 0.f};
    T* gout = static_cast<T*>(p.dgate) + row * (int64_t)p.G * p.D + col;
    #pragma unroll
    for (int k = 0; k < KV; ++k) {
      float t[VEC], d[VEC], dg[VEC];
      if (GATE) Vec<T, VEC>::unpack(gr[k], t);
      Vec<T, VEC>::unpack(dr[k], d);
      #pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float n = x[k][v] * rstd;
        const float z = fmaf(n, w[k][v], b[k][v]);
        if (!GATE) t[v] = z;
        const float sig = sigmoid_f(t[v]);
        const float slope = sig * fmaf(t[v], 1.f - sig, 1.f);
        const float dz = GATE ? d[v] * (t[v] * sig) : d[v] * slope;
        dg[v] = d[v] * z * slope;
        dw[k][v] = fmaf(dz, n, dw[k][v]);
        db[k][v] += dz;
        x[k][v] = n;
        dn[k][v] = dz * w[k][v];
        q[0] += dn[k][v];
        q[1] = fmaf(dn[k][v], n, q[1]);
      }
      if (GATE && p.dgate && on && k * p.L + lane < p.nv) Vec<T, VEC>::store(gout + k * step, dg);
    }
    group_sum<BLOCK, 2>(q, p.L, red);
    const float m0 = p.center ? q[0] * inv : 0.f, m1 = q[1] * inv;
    if (p.dx) {
      T* out = static_cast<T*>(p.dx) + row * (int64_t)p.G * p.D + col;
      #pragma unroll
      for (int k = 0; k < KV; ++k) {
        float o[VEC];
        #pragma unroll
        for (int v = 0; v < VEC; ++v) o[v] = rstd * (dn[k][v] - m0 - x[k][v] * m1);
        if (on && k * p.L + lane < p.nv) Vec<T, VEC>::store(out + k * step, o);
      }
    }
  }
  if (BWD && used && (p.want_w || p.want_b)) {
    const int64_t C = (int64_t)p.G * p.D, parts = (int64_t)gridDim.y * p.row_step;
    float* out = p.part + ((int64_t)blockIdx.y * p.row_step + row0) * C + col;
    #pragma unroll
    for (int k = 0; k < KV; ++k)
      if (k * p.L + lane < p.nv)
        #pragma unroll
        for (int v = 0; v < VEC; ++v) {
          if (p.want_w) out[k * step + v] = dw[k][v];
          if (p.want_b) out[(p.want_w ? parts * C : 0) + k * step + v] = db[k][v];
        }
  }
}

// Column sums of a [rows][cols] f32 array (blockIdx.y-th of several), rows in
// a fixed order: 32 columns a block, 32 partial sums of each.
__global__ void __launch_bounds__(1024) k_column_sums(const float* __restrict__ part, int64_t rows, int cols,
                                                     float* out0, float* out1) {
  __shared__ float sh[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const float* p = part + (int64_t)blockIdx.y * rows * cols;
  float s = 0.f;
  if (c < cols)
    #pragma unroll 8
    for (int64_t r = warp; r < rows; r += 32) s += __ldcs(p + r * cols + c);
  sh[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < cols) {
    s = 0.f;
    #pragma unroll
    for (int i = 0; i < 32; ++i) s += sh[i][lane];
    (blockIdx.y ? out1 : out0)[c] = s;
  }
}

int launch_column_sums(const float* part, int64_t rows, int cols, int arrays, float* out0, float* out1,
                       cudaStream_t st, const char* fn) {
  k_column_sums<<<dim3((unsigned)((cols + 31) / 32), arrays), 1024, 0, st>>>(part, rows, cols, out0, out1);
  return check_cuda(cudaGetLastError(), fn);
}

// ---- host ----

struct NormPlan {
  int vec, kv;
  bool block;
  unsigned gx, gy;
};

// Vector width, lanes and grid for these sizes; false where the group is too wide.
static bool plan_norm(NormParams& p, int dtype, int max_vec, int blocks_per_sm, NormPlan& n) {
  n.vec = dtype == GDN2_DTYPE_BF16 ? 8 : 4;
  while (n.vec > 1 && (p.D % n.vec || n.vec > max_vec)) n.vec /= 2;
  const int most_kv = n.vec == 8 ? 2 : 4;  // at most 16 values a lane: their sums of dw and db are registers too
  p.nv = p.D / n.vec;
  n.block = p.nv > 32 * most_kv;
  if (p.nv > NORM_THREADS * most_kv) return false;
  const int most = n.block ? NORM_THREADS : 32;
  p.L = n.block ? NORM_THREADS : 1;
  while (p.L < most && p.L < p.nv) p.L *= 2;
  const int need = (p.nv + p.L - 1) / p.L;
  n.kv = need <= 1 ? 1 : need <= 2 ? 2 : 4;
  p.slots = NORM_THREADS / p.L;
  p.per_row = p.G < p.slots ? p.G : p.slots;
  p.row_step = p.slots / p.per_row;
  n.gx = (unsigned)((p.G + p.per_row - 1) / p.per_row);
  const int64_t rounds = (p.rows + p.row_step - 1) / p.row_step;
  int64_t gy = ((int64_t)148 * blocks_per_sm + n.gx - 1) / n.gx;
  if (gy > rounds) gy = rounds;
  n.gy = (unsigned)(gy < 65535 ? gy : 65535);
  return true;
}

constexpr int NORM_FWD_BLOCKS = 8, NORM_BWD_BLOCKS = 4;

template <typename T, int VEC, int KV, bool BLOCK, bool BWD>
static int launch_norm_kernel(const NormParams& p, const NormPlan& n, cudaStream_t st, const char* fn) {
  if (p.gate)
    k_group_norm<T, VEC, KV, BLOCK, true, BWD><<<dim3(n.gx, n.gy), NORM_THREADS, 0, st>>>(p);
  else
    k_group_norm<T, VEC, KV, BLOCK, false, BWD><<<dim3(n.gx, n.gy), NORM_THREADS, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), fn);
}

template <typename T, int VEC, bool BWD>
static int launch_norm_vec(const NormParams& p, const NormPlan& n, cudaStream_t st, const char* fn) {
  constexpr int MORE = VEC == 8 ? 2 : 4;
  if (n.block)
    return n.kv == 1   ? launch_norm_kernel<T, VEC, 1, true, BWD>(p, n, st, fn)
           : n.kv == 2 ? launch_norm_kernel<T, VEC, 2, true, BWD>(p, n, st, fn)
                       : launch_norm_kernel<T, VEC, MORE, true, BWD>(p, n, st, fn);
  return n.kv == 1   ? launch_norm_kernel<T, VEC, 1, false, BWD>(p, n, st, fn)
         : n.kv == 2 ? launch_norm_kernel<T, VEC, 2, false, BWD>(p, n, st, fn)
                     : launch_norm_kernel<T, VEC, MORE, false, BWD>(p, n, st, fn);
}

template <bool BWD>
static int launch_norm(const NormParams& p, const NormPlan& n, int dtype, cudaStream_t st, const char* fn) {
  if (dtype == GDN2_DTYPE_F32) {
    if (n.vec == 4) return launch_norm_vec<float, 4, BWD>(p, n, st, fn);
    if (n.vec == 2) return launch_norm_vec<float, 2, BWD>(p, n, st, fn);
    return launch_norm_vec<float, 1, BWD>(p, n, st, fn);
  }
  typedef __nv_bfloat16 bf;
  if (n.vec == 8) return launch_norm_vec<bf, 8, BWD>(p, n, st, fn);
  if (n.vec == 4) return launch_norm_vec<bf, 4, BWD>(p, n, st, fn);
  if (n.vec == 2) return launch_norm_vec<bf, 2, BWD>(p, n, st, fn);
  return launch_norm_vec<bf, 1, BWD>(p, n, st, fn);
}

// Widest vector that this pointer and row pitch allow.
static int vec_of(const void* ptr, int64_t ld, int elem) {
  int v = 16 / elem;
  while (v > 1 && ((uintptr_t)ptr % (v * elem) || ld % v)) v /= 2;
  return v;
}
static int least(int a, int b) { return a < b ? a : b; }

static int prep_norm(const gdn2_group_norm_args* a, NormParams& p, int& vec, const char* fn) {
  if (!a) return set_error(GDN2_EINVAL, "%s: null args", fn);
  if (a->rows <= 0 || a->groups <= 0 || a->width <= 0)
    return set_error(GDN2_EINVAL, "%s: sizes must be > 0 (rows=%lld groups=%d width=%d)", fn, (long long)a->rows,
                     a->groups, a->width);
  if ((int64_t)a->groups * a->width > 0x7fffffffll)
    return set_error(GDN2_EUNSUPPORTED, "%s: %d groups of %d channels", fn, a->groups, a->width);
  if (a->dtype != GDN2_DTYPE_F32 && a->dtype != GDN2_DTYPE_BF16)
    return set_error(GDN2_EINVAL, "%s: unknown dtype %d", fn, a->dtype);
  if (!(a->eps > 0.f)) return set_error(GDN2_EINVAL, "%s: eps must be > 0, got %g", fn, (double)a->eps);
  if (!a->x) return set_error(GDN2_EINVAL, "%s: null tensor pointer", fn);
  const int elem = a->dtype == GDN2_DTYPE_BF16 ? 2 : 4;
  p = NormParams{};
  p.rows = a->rows; p.G = a->groups; p.D = a->width;
  p.shared_w = a->weight_shared; p.center = a->center; p.eps = a->eps;
  p.x = a->x; p.ldx = a->ld_x;
  p.gate = a->gate; p.ldgate = a->ld_gate;
  p.w = a->weight; p.b = a->bias;
  vec = vec_of(a->x, a->ld_x, elem);
  if (a->gate) vec = least(vec, vec_of(a->gate, a->ld_gate, elem));
  return GDN2_OK;
}

static int too_wide(const gdn2_group_norm_args* a, const char* fn) {
  return set_error(GDN2_EUNSUPPORTED, "%s: groups of %d channels are too wide for the rows' alignment", fn, a->width);
}

int launch_group_norm(const gdn2_group_norm_args* a, void* y, cudaStream_t st) {
  const char* fn = "gdn2_group_norm_gate";
  NormParams p;
  NormPlan n;
  int vec;
  int rc = prep_norm(a, p, vec, fn);
  if (rc) return rc;
  if (!y) return set_error(GDN2_EINVAL, "%s: null tensor pointer", fn);
  vec = least(vec, vec_of(y, (int64_t)p.G * p.D, a->dtype == GDN2_DTYPE_BF16 ? 2 : 4));
  if (!plan_norm(p, a->dtype, vec, NORM_FWD_BLOCKS, n)) return too_wide(a, fn);
  p.y = y;
  return launch_norm<false>(p, n, a->dtype, st, fn);
}

static int plan_norm_bwd(const gdn2_group_norm_bwd_args* q, NormParams& p, NormPlan& n, const char* fn) {
  if (!q) return set_error(GDN2_EINVAL, "%s: null args", fn);
  const gdn2_group_norm_args* a = &q->fwd;
  int vec;
  int rc = prep_norm(a, p, vec, fn);
  if (rc) return rc;
  if (!q->d_y) return set_error(GDN2_EINVAL, "%s: null tensor pointer", fn);
  if ((q->d_gate && !a->gate) || (q->d_weight && !a->weight) || (q->d_bias && !a->bias))
    return set_error(GDN2_EINVAL, "%s: the gradient of an input that is not there", fn);
  const int elem = a->dtype == GDN2_DTYPE_BF16 ? 2 : 4;
  vec = least(vec, vec_of(q->d_y, q->ld_dy, elem));
  if (q->dx) vec = least(vec, vec_of(q->dx, (int64_t)p.G * p.D, elem));
  if (q->d_gate) vec = least(vec, vec_of(q->d_gate, (int64_t)p.G * p.D, elem));
  if (!plan_norm(p, a->dtype, vec, NORM_BWD_BLOCKS, n)) return too_wide(a, fn);
  p.dy = q->d_y; p.lddy = q->ld_dy;
  p.dx = q->dx; p.dgate = q->d_gate;
  p.want_w = q->d_weight != nullptr;
  p.want_b = q->d_bias != nullptr;
  return GDN2_OK;
}

static int64_t norm_part_rows(const NormParams& p, const NormPlan& n) { return (int64_t)n.gy * p.row_step; }

size_t group_norm_bwd_workspace_bytes(const gdn2_group_norm_bwd_args* q) {
  NormParams p;
  NormPlan n;
  if (plan_norm_bwd(q, p, n, "gdn2_group_norm_gate_bwd_workspace_bytes")) return 0;
  return (size_t)norm_part_rows(p, n) * p.G * p.D * (p.want_w + p.want_b) * sizeof(float);
}

int launch_group_norm_bwd(const gdn2_group_norm_bwd_args* q, void* ws, size_t ws_bytes, cudaStream_t st) {
  const char* fn = "gdn2_group_norm_gate_bwd";
  NormParams p;
  NormPlan n;
  int rc = plan_norm_bwd(q, p, n, fn);
  if (rc) return rc;
  const int arrays = p.want_w + p.want_b;
  const size_t need = (size_t)norm_part_rows(p, n) * p.G * p.D * arrays * sizeof(float);
  if (need && (!ws || ws_bytes < need))
    return set_error(GDN2_EWORKSPACE, "%s: workspace %zu bytes < required %zu", fn, ws ? ws_bytes : 0, need);
  p.part = static_cast<float*>(ws);
  rc = launch_norm<true>(p, n, q->fwd.dtype, st, fn);
  if (rc || !arrays) return rc;
  float* first = p.want_w ? q->d_weight : q->d_bias;
  // weights shared by the groups: the groups' sums are rows too
  const int64_t rows = norm_part_rows(p, n) * (p.shared_w ? p.G : 1);
  return launch_column_sums(p.part, rows, p.shared_w ? p.D : p.G * p.D, arrays, first, q->d_bias, st, fn);
}

}  // namespace gdn2

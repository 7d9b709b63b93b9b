// Group norm of each token's channels, channels last, with its affine map
// and a SiLU, and the adjoint.  For a row's group of `width` channels
//
//   n = (x - mean) rstd    rstd = 1 / sqrt(mean((x - mean)^2) + eps)   (mean = 0 without center)
//   z = n w + b,           y = z silu(gate),  or silu(z) without a gate
//
//   dz = dy silu(gate) (or dy silu'(z)),  dgate = dy z silu'(gate),  dw = sum dz n,  db = sum dz
//   dn = dz w,  dx = rstd (dn - mean(dn) - n mean(dn n))
//
// Bound by HBM: x and gate in, y out (dy in and dx, dgate out besides); 8 x
// 4096 rows of 16 groups of 128 bf16: 72 us forward and 131 us backward, 86 %
// and 79 % of what a copy of as many bytes reaches.  A group's values stay in
// the registers of L neighbouring lanes (of the whole block where a group has
// more than 64 vectors of eight bf16, or 128 of fewer elements: above 512
// channels, or above 128 of an odd width) from the load to the store, so
// everything is read once,
// statistics included: they are formed in two steps (mean, then squares of
// deviations) from registers, without the cancellation of E[x^2] - mean^2, and
// the backward forms them again rather than read them.
// A lane keeps its group for all its rows, so the affine weights and the sums
// of their gradients stay in registers too.  Those sums leave through one
// partial row per slot of lanes, added up by a second kernel in a fixed
// order: no atomics.
#include "sequence.cuh"

namespace gdn2 {

constexpr int NORM_THREADS = 256;
constexpr int WIDE_THREADS = 512;  // of a block that walks a group beyond its registers
constexpr int WIDE_SMEM = 104 * 1024;  // most bytes of sums that such a block keeps: two blocks an SM

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
  float* part;           // partial rows of dw, then of db: [gridDim.y * row_step][G * D], or [blocks][D] shared
  int want_w, want_b;
  int wide_smem;         // a walked group's sums of dw and db stay in shared memory
};

// Sums of up to two values over a group's lanes (the block, in block mode).
template <bool BLOCK, int N, int THREADS = NORM_THREADS>
__device__ __forceinline__ void group_sum(float (&s)[N], int L, float* red) {
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (BLOCK || o < L)
      #pragma unroll
      for (int k = 0; k < N; ++k) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
  if (BLOCK) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
      #pragma unroll
      for (int k = 0; k < N; ++k) red[k * (THREADS / 32) + (threadIdx.x >> 5)] = s[k];
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < N; ++k) {
      s[k] = 0.f;
      #pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) s[k] += red[k * (THREADS / 32) + i];
    }
  }
}

// What a lane holds of a row: KV vectors of VEC channels, as NP pairs each
// (the second of a pair zero for VEC = 1).  Arithmetic runs on packed pairs:
// the kernel would be bound by its instructions otherwise.
template <typename T, int VEC, int KV, bool BLOCK, bool GATE, bool BWD>
__global__ void __launch_bounds__(NORM_THREADS, VEC * KV <= 8 ? (BWD ? 2 : 4) : 1) k_group_norm(const NormParams p) {
  constexpr int NP = VEC == 1 ? 1 : VEC / 2;
  typedef typename Vec<T, VEC>::Raw Raw;
  __shared__ float red[16];
  const int slot = BLOCK ? 0 : threadIdx.x / p.L;
  const int lane = BLOCK ? threadIdx.x : threadIdx.x % p.L;
  const int group = blockIdx.x * p.per_row + slot % p.per_row;
  const int row0 = slot / p.per_row;
  const bool used = group < p.G && row0 < p.row_step;
  const int64_t C = (int64_t)p.G * p.D, col = (int64_t)group * p.D + lane * VEC;
  const int step = p.L * VEC;  // channels between a lane's vectors
  const float inv = 1.f / (float)p.D;
  const f32x2 zero = f2pk(0.f, 0.f), one = f2pk(1.f, 1.f), minus = f2pk(-1.f, -1.f);
  auto has = [&](int k) { return k * p.L + lane < p.nv; };
  auto both = [&](float v) { return f2pk(v, VEC == 1 ? 0.f : v); };

  f32x2 w[KV][NP], b[KV][NP], dw[KV][NP], db[KV][NP];
  #pragma unroll
  for (int k = 0; k < KV; ++k)
    #pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int64_t c = (p.shared_w ? 0 : (int64_t)group * p.D) + lane * VEC + k * step + 2 * i;
      w[k][i] = used && has(k) && p.w ? f2pk(__ldg(p.w + c), VEC == 1 ? 0.f : __ldg(p.w + c + (VEC > 1))) : one;
      b[k][i] = used && has(k) && p.b ? f2pk(__ldg(p.b + c), VEC == 1 ? 0.f : __ldg(p.b + c + (VEC > 1))) : zero;
      dw[k][i] = db[k][i] = zero;
    }

  // every thread of a warp (of the block) takes part in the sums of each round; pointers walk the rows
  const int64_t first = (int64_t)blockIdx.y * p.row_step + row0, stride = (int64_t)gridDim.y * p.row_step;
  const T* xp = static_cast<const T*>(p.x) + first * p.ldx + col;
  const T* gp = static_cast<const T*>(p.gate) + first * p.ldgate + col;
  const T* dp = static_cast<const T*>(p.dy) + first * p.lddy + col;
  const int64_t out_at = first * C + col;
  T* yp = static_cast<T*>(p.y) + out_at;
  T* dxp = static_cast<T*>(p.dx) + out_at;
  T* dgp = static_cast<T*>(p.dgate) + out_at;
  const int64_t x_step = stride * p.ldx, g_step = stride * p.ldgate, d_step = stride * p.lddy, o_step = stride * C;
  // rounds of this lane's rows, and of the block
  int64_t left = used && first < p.rows ? (p.rows - first + stride - 1) / stride : 0;
  int64_t rounds = (p.rows - (int64_t)blockIdx.y * p.row_step + stride - 1) / stride;
  Raw xr[KV], gr[KV], dr[KV];
  auto fetch = [&](bool in) {
    #pragma unroll
    for (int k = 0; k < KV; ++k) {
      xr[k] = gr[k] = dr[k] = Raw{};
      if (in && has(k)) {
        xr[k] = Vec<T, VEC>::load(xp + k * step);
        if (GATE) gr[k] = Vec<T, VEC>::load(gp + k * step);
        if (BWD) dr[k] = Vec<T, VEC>::load(dp + k * step);
      }
    }
    xp += x_step;
    if (GATE) gp += g_step;
    if (BWD) dp += d_step;
  };
  fetch(left > 0);
  for (; rounds > 0; --rounds, --left, yp += o_step, dxp += o_step, dgp += o_step) {
    const bool on = left > 0;
    f32x2 x[KV][NP];
    Raw gc[KV], dc[KV];
    f32x2 acc = zero;
    #pragma unroll
    for (int k = 0; k < KV; ++k) {
      unpack_pairs<T, VEC>(xr[k], x[k]);
      gc[k] = gr[k];
      dc[k] = dr[k];
      #pragma unroll
      for (int i = 0; i < NP; ++i) acc = f2add(acc, x[k][i]);
    }
    fetch(left > 1);  // the next round's values while this one's are worked on
    float s[2], lo, hi;
    if (p.center) {
      f2un(acc, lo, hi);
      s[0] = lo + hi;
      group_sum<BLOCK, 1>(*reinterpret_cast<float (*)[1]>(s), p.L, red);
      const float mean = s[0] * inv;
      #pragma unroll
      for (int k = 0; k < KV; ++k) {
        const f32x2 m = both(has(k) ? -mean : 0.f);  // what a group does not have stays zero
        #pragma unroll
        for (int i = 0; i < NP; ++i) x[k][i] = f2add(x[k][i], m);
      }
    }
    acc = zero;
    #pragma unroll
    for (int k = 0; k < KV; ++k)
      #pragma unroll
      for (int i = 0; i < NP; ++i) acc = f2fma(x[k][i], x[k][i], acc);
    f2un(acc, lo, hi);
    s[0] = lo + hi;
    group_sum<BLOCK, 1>(*reinterpret_cast<float (*)[1]>(s), p.L, red);
    const float rstd = rsqrtf(fmaf(s[0], inv, p.eps));
    const f32x2 rstd2 = f2pk(rstd, rstd);

    if (!BWD) {
      #pragma unroll
      for (int k = 0; k < KV; ++k) {
        f32x2 t[NP], y[NP];
        if (GATE) unpack_pairs<T, VEC>(gc[k], t);
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
          const f32x2 z = f2fma(f2mul(x[k][i], rstd2), w[k][i], b[k][i]);
          if (!GATE) t[i] = z;
          y[i] = f2mul(t[i], sigmoid2(t[i]));
          if (GATE) y[i] = f2mul(z, y[i]);
        }
        if (on && has(k)) store_pairs<T, VEC>(yp + k * step, y);
      }
      continue;
    }
    f32x2 dn[KV][NP], q0 = zero, q1 = zero;
    #pragma unroll
    for (int k = 0; k < KV; ++k) {
      f32x2 t[NP], d[NP], dg[NP];
      if (GATE) unpack_pairs<T, VEC>(gc[k], t);
      unpack_pairs<T, VEC>(dc[k], d);
      #pragma unroll
      for (int i = 0; i < NP; ++i) {
        const f32x2 n = f2mul(x[k][i], rstd2);
        const f32x2 z = f2fma(n, w[k][i], b[k][i]);
        if (!GATE) t[i] = z;
        const f32x2 sig = sigmoid2(t[i]), act = f2mul(t[i], sig);
        const f32x2 slope = f2fma(act, f2fma(sig, minus, one), sig);
        const f32x2 dz = f2mul(d[i], GATE ? act : slope);
        if (GATE) dg[i] = f2mul(f2mul(d[i], z), slope);
        dw[k][i] = f2fma(dz, n, dw[k][i]);
        db[k][i] = f2add(db[k][i], dz);
        x[k][i] = n;
        dn[k][i] = f2mul(dz, w[k][i]);
        q0 = f2add(q0, dn[k][i]);
        q1 = f2fma(dn[k][i], n, q1);
      }
      if (GATE && p.dgate && on && has(k)) store_pairs<T, VEC>(dgp + k * step, dg);
    }
    f2un(q0, lo, hi);
    s[0] = lo + hi;
    f2un(q1, lo, hi);
    s[1] = lo + hi;
    group_sum<BLOCK, 2>(s, p.L, red);
    if (p.dx) {  // rstd (dn - mean(dn) - n mean(dn n))
      const float m0 = p.center ? -rstd * (s[0] * inv) : 0.f, m1 = -rstd * (s[1] * inv);
      const f32x2 m0p = f2pk(m0, m0), m1p = f2pk(m1, m1);
      #pragma unroll
      for (int k = 0; k < KV; ++k) {
        f32x2 o[NP];
        #pragma unroll
        for (int i = 0; i < NP; ++i) o[i] = f2fma(dn[k][i], rstd2, f2fma(x[k][i], m1p, m0p));
        if (on && has(k)) store_pairs<T, VEC>(dxp + k * step, o);
      }
    }
  }
  if (!BWD || !(p.want_w || p.want_b)) return;
  if (!p.shared_w) {
    const int64_t parts = (int64_t)gridDim.y * p.row_step;
    float* out = p.part + ((int64_t)blockIdx.y * p.row_step + row0) * C + col;
    #pragma unroll
    for (int k = 0; k < KV; ++k)
      if (used && has(k))
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
          if (p.want_w) put_f32<VEC == 1 ? 1 : 2>(out + k * step + 2 * i, dw[k][i]);
          if (p.want_b) put_f32<VEC == 1 ? 1 : 2>(out + (p.want_w ? parts * C : 0) + k * step + 2 * i, db[k][i]);
        }
    return;
  }
  // weights of all groups: the block's slots add up one after the other
  extern __shared__ float sums[];  // [2][D]
  for (int e = threadIdx.x; e < 2 * p.D; e += NORM_THREADS) sums[e] = 0.f;
  for (int turn = 0; turn < p.slots; ++turn) {
    __syncthreads();
    if (turn != slot || !used) continue;
    #pragma unroll
    for (int k = 0; k < KV; ++k)
      if (has(k))
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
          float* at = sums + lane * VEC + k * step + 2 * i;
          put_f32<VEC == 1 ? 1 : 2>(at, f2add(get_f32<VEC == 1 ? 1 : 2>(at), dw[k][i]));
          put_f32<VEC == 1 ? 1 : 2>(at + p.D, f2add(get_f32<VEC == 1 ? 1 : 2>(at + p.D), db[k][i]));
        }
  }
  __syncthreads();
  const int64_t parts = (int64_t)gridDim.y * gridDim.x, mine = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  for (int e = threadIdx.x; e < p.D; e += NORM_THREADS) {
    if (p.want_w) p.part[mine * p.D + e] = sums[e];
    if (p.want_b) p.part[((p.want_w ? parts : 0) + mine) * p.D + e] = sums[p.D + e];
  }
}

// Groups beyond what a block's registers hold: a block per group and row, walked
// again for each statistic and for the results (L1 and L2 hold it meanwhile).
// The sums of the weights' gradients are kept in shared memory, in the partial
// row itself where they do not fit; each place is one thread's.  8192 rows of
// 8192 bf16, one group, gated: 118 us forward and 338 us backward (410 with the
// sums of a lane's vector side by side, whose banks collide; 430 with all sums in
// the partial rows).
template <typename T, int VEC, bool GATE, bool BWD>
__global__ void __launch_bounds__(WIDE_THREADS, 2) k_group_norm_wide(const NormParams p) {
  constexpr int NP = VEC == 1 ? 1 : VEC / 2;
  typedef typename Vec<T, VEC>::Raw Raw;
  __shared__ float red[2 * WIDE_THREADS / 32];
  extern __shared__ float sums[];
  const int group = blockIdx.x;
  const int64_t C = (int64_t)p.G * p.D, col = (int64_t)group * p.D;
  const float inv = 1.f / (float)p.D;
  const f32x2 zero = f2pk(0.f, 0.f), one = f2pk(1.f, 1.f), minus = f2pk(-1.f, -1.f);
  const float* w = p.w ? p.w + (p.shared_w ? 0 : col) : nullptr;
  const float* b = p.b ? p.b + (p.shared_w ? 0 : col) : nullptr;
  const int64_t cols = p.shared_w ? p.D : C, parts = (p.shared_w ? (int64_t)gridDim.x : 1) * gridDim.y;
  float* part_w = p.part + (p.shared_w ? ((int64_t)blockIdx.y * gridDim.x + group) * p.D : (int64_t)blockIdx.y * C + col);
  float* part_b = part_w + (p.want_w ? parts * cols : 0);
  float* sum_w = p.wide_smem ? sums : part_w;
  float* sum_b = p.wide_smem ? sums + (p.want_w ? p.D : 0) : part_b;
  // where pair i of the vector at e is summed; in shared memory neighbouring lanes' pairs are neighbours
  auto place = [&](int64_t e, int i) { return VEC > 1 && p.wide_smem ? 2 * (i * (int64_t)p.nv + e / VEC) : e + 2 * i; };
  auto pair = [&](const float* q) { return f2pk(q[0], VEC == 1 ? 0.f : q[VEC > 1]); };
  auto values = [&](const void* base, int64_t row, int64_t ld, int64_t e, f32x2 (&v)[NP]) {
    unpack_pairs<T, VEC>(__ldg(reinterpret_cast<const Raw*>(static_cast<const T*>(base) + row * ld + col + e)), v);
  };
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    float s[2], lo, hi;
    f32x2 mean = zero, v[NP];
    if (p.center) {
      s[0] = 0.f;
      #pragma unroll 2
      for (int64_t e = threadIdx.x * VEC; e < p.D; e += WIDE_THREADS * VEC) {
        values(p.x, row, p.ldx, e, v);
        f32x2 acc = v[0];
        #pragma unroll
        for (int i = 1; i < NP; ++i) acc = f2add(acc, v[i]);
        f2un(acc, lo, hi);
        s[0] += lo + hi;
      }
      group_sum<true, 1, WIDE_THREADS>(*reinterpret_cast<float (*)[1]>(s), p.L, red);
      mean = f2pk(s[0] * inv, VEC == 1 ? 0.f : s[0] * inv);
    }
    s[0] = 0.f;
    #pragma unroll 2
    for (int64_t e = threadIdx.x * VEC; e < p.D; e += WIDE_THREADS * VEC) {
      values(p.x, row, p.ldx, e, v);
      f32x2 acc = zero;
      #pragma unroll
      for (int i = 0; i < NP; ++i) {
        const f32x2 d = f2fma(mean, minus, v[i]);
        acc = f2fma(d, d, acc);
      }
      f2un(acc, lo, hi);
      s[0] += lo + hi;
    }
    group_sum<true, 1, WIDE_THREADS>(*reinterpret_cast<float (*)[1]>(s), p.L, red);
    const float rstd = rsqrtf(fmaf(s[0], inv, p.eps));
    const f32x2 rstd2 = f2pk(rstd, rstd);
    if (!BWD) {
      for (int64_t e = threadIdx.x * VEC; e < p.D; e += WIDE_THREADS * VEC) {
        f32x2 t[NP];
        values(p.x, row, p.ldx, e, v);
        if (GATE) values(p.gate, row, p.ldgate, e, t);
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
          const f32x2 n = f2mul(f2fma(mean, minus, v[i]), rstd2);
          const f32x2 z = f2fma(n, w ? pair(w + e + 2 * i) : one, b ? pair(b + e + 2 * i) : zero);
          if (!GATE) t[i] = z;
          const f32x2 act = f2mul(t[i], sigmoid2(t[i]));
          v[i] = GATE ? f2mul(z, act) : act;
        }
        store_pairs<T, VEC>(static_cast<T*>(p.y) + row * C + col + e, v);
      }
      continue;
    }
    // n, dz and dgate of a vector
    auto adjoint = [&](int64_t e, f32x2 (&n)[NP], f32x2 (&dz)[NP], f32x2 (&dg)[NP]) {
      f32x2 t[NP];
      values(p.x, row, p.ldx, e, n);
      values(p.dy, row, p.lddy, e, dz);
      if (GATE) values(p.gate, row, p.ldgate, e, t);
      #pragma unroll
      for (int i = 0; i < NP; ++i) {
        n[i] = f2mul(f2fma(mean, minus, n[i]), rstd2);
        const f32x2 z = f2fma(n[i], w ? pair(w + e + 2 * i) : one, b ? pair(b + e + 2 * i) : zero);
        if (!GATE) t[i] = z;
        const f32x2 sig = sigmoid2(t[i]), act = f2mul(t[i], sig), slope = f2fma(act, f2fma(sig, minus, one), sig);
        if (GATE) dg[i] = f2mul(f2mul(dz[i], z), slope);
        dz[i] = f2mul(dz[i], GATE ? act : slope);
      }
    };
    f32x2 n[NP], dz[NP], dg[NP];
    s[0] = s[1] = 0.f;
    for (int64_t e = threadIdx.x * VEC; e < p.D; e += WIDE_THREADS * VEC) {
      adjoint(e, n, dz, dg);
      if (GATE && p.dgate) store_pairs<T, VEC>(static_cast<T*>(p.dgate) + row * C + col + e, dg);
      f32x2 q0 = zero, q1 = zero;
      #pragma unroll
      for (int i = 0; i < NP; ++i) {
        const f32x2 dn = w ? f2mul(dz[i], pair(w + e + 2 * i)) : dz[i];
        q0 = f2add(q0, dn);
        q1 = f2fma(dn, n[i], q1);
        float* at_w = sum_w + place(e, i);
        float* at_b = sum_b + place(e, i);
        const bool open = row == blockIdx.y;  // the block's first row
        if (p.want_w) put_f32<VEC == 1 ? 1 : 2>(at_w, f2fma(dz[i], n[i], open ? zero : pair(at_w)));
        if (p.want_b) put_f32<VEC == 1 ? 1 : 2>(at_b, f2add(dz[i], open ? zero : pair(at_b)));
      }
      f2un(q0, lo, hi);
      s[0] += lo + hi;
      f2un(q1, lo, hi);
      s[1] += lo + hi;
    }
    group_sum<true, 2, WIDE_THREADS>(s, p.L, red);
    if (!p.dx) continue;
    const float m0 = p.center ? -rstd * (s[0] * inv) : 0.f, m1 = -rstd * (s[1] * inv);
    const f32x2 m0p = f2pk(m0, m0), m1p = f2pk(m1, m1);
    for (int64_t e = threadIdx.x * VEC; e < p.D; e += WIDE_THREADS * VEC) {
      adjoint(e, n, dz, dg);
      #pragma unroll
      for (int i = 0; i < NP; ++i) {
        const f32x2 dn = w ? f2mul(dz[i], pair(w + e + 2 * i)) : dz[i];
        v[i] = f2fma(dn, rstd2, f2fma(n[i], m1p, m0p));
      }
      store_pairs<T, VEC>(static_cast<T*>(p.dx) + row * C + col + e, v);
    }
  }
  if (!BWD || !p.wide_smem) return;
  for (int64_t e = threadIdx.x * VEC; e < p.D; e += WIDE_THREADS * VEC)  // this thread's own places
    #pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (p.want_w) put_f32<VEC == 1 ? 1 : 2>(part_w + e + 2 * i, pair(sum_w + place(e, i)));
      if (p.want_b) put_f32<VEC == 1 ? 1 : 2>(part_b + e + 2 * i, pair(sum_b + place(e, i)));
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
  bool block, wide;
  unsigned gx, gy;
};

// Vector width, lanes and grid for these sizes.
static void plan_norm(NormParams& p, int dtype, int max_vec, int blocks_per_sm, NormPlan& n) {
  n.vec = dtype == GDN2_DTYPE_BF16 ? 8 : 4;
  while (n.vec > 1 && (p.D % n.vec || n.vec > max_vec)) n.vec /= 2;
  const int most_kv = n.vec == 8 ? 2 : 4;  // at most 16 values a lane: their sums of dw and db are registers too
  p.nv = p.D / n.vec;
  n.block = p.nv > 32 * most_kv;
  n.wide = p.nv > NORM_THREADS * most_kv;
  if (n.wide) {  // every value is fetched again anyway: whole vectors or single ones
    if (n.vec != (dtype == GDN2_DTYPE_BF16 ? 8 : 4)) n.vec = 1;
    n.block = true;
  }
  // lanes of a group and vectors of a lane: as few idle places as possible, then the fewer vectors
  p.L = NORM_THREADS;
  n.kv = (p.nv + p.L - 1) / p.L;
  if (!n.block) {
    int best = 1 << 30;
    for (int l = 32; l >= 1; l /= 2) {
      const int kv = (p.nv + l - 1) / l;
      if (kv > most_kv) break;
      if (l * kv < best) {
        best = l * kv;
        p.L = l;
        n.kv = kv;
      }
    }
  }
  p.slots = NORM_THREADS / p.L;
  p.per_row = p.G < p.slots ? p.G : p.slots;
  p.row_step = p.slots / p.per_row;
  n.gx = (unsigned)((p.G + p.per_row - 1) / p.per_row);
  const int64_t rounds = (p.rows + p.row_step - 1) / p.row_step;
  int64_t gy = ((int64_t)148 * blocks_per_sm + n.gx - 1) / n.gx;
  if (gy > rounds) gy = rounds;
  n.gy = (unsigned)(gy < 65535 ? gy : 65535);
}

// Blocks per SM: as many as are resident, so that each block's weights are
// read (and its partial sums written) once.  8 x 4096 rows of 16 groups of
// 128 bf16: 72 us forward with 4, 83 with 6; 131 us backward with 2, 139 with 8.
constexpr int NORM_FWD_BLOCKS = 4, NORM_BWD_BLOCKS = 2;

template <typename T, int VEC, int KV, bool BLOCK, bool BWD>
static int launch_norm_kernel(const NormParams& p, const NormPlan& n, cudaStream_t st, const char* fn) {
  const int smem = BWD && p.shared_w && (p.want_w || p.want_b) ? 2 * p.D * (int)sizeof(float) : 0;  // 32 KB at most
  if (p.gate)
    k_group_norm<T, VEC, KV, BLOCK, true, BWD><<<dim3(n.gx, n.gy), NORM_THREADS, smem, st>>>(p);
  else
    k_group_norm<T, VEC, KV, BLOCK, false, BWD><<<dim3(n.gx, n.gy), NORM_THREADS, smem, st>>>(p);
  return check_cuda(cudaGetLastError(), fn);
}

template <typename T, int VEC, bool BWD>
static int launch_norm_vec(const NormParams& p, const NormPlan& n, cudaStream_t st, const char* fn) {
  // three vectors only within a warp, where the choice is free; eight elements a vector: two at most
  constexpr int MORE = VEC == 8 ? 2 : 4, THREE = VEC == 8 ? 2 : 3;
  if (n.block)
    return n.kv == 1   ? launch_norm_kernel<T, VEC, 1, true, BWD>(p, n, st, fn)
           : n.kv == 2 ? launch_norm_kernel<T, VEC, 2, true, BWD>(p, n, st, fn)
                       : launch_norm_kernel<T, VEC, MORE, true, BWD>(p, n, st, fn);
  return n.kv == 1   ? launch_norm_kernel<T, VEC, 1, false, BWD>(p, n, st, fn)
         : n.kv == 2 ? launch_norm_kernel<T, VEC, 2, false, BWD>(p, n, st, fn)
         : n.kv == 3 ? launch_norm_kernel<T, VEC, THREE, false, BWD>(p, n, st, fn)
                     : launch_norm_kernel<T, VEC, MORE, false, BWD>(p, n, st, fn);
}

template <typename T, int VEC, bool BWD>
static int launch_norm_wide(const NormParams& p, const NormPlan& n, cudaStream_t st, const char* fn) {
  NormParams q = p;
  const int64_t bytes = BWD ? (int64_t)(p.want_w + p.want_b) * p.D * (int)sizeof(float) : 0;
  q.wide_smem = bytes > 0 && bytes <= WIDE_SMEM;
  const int smem = q.wide_smem ? (int)bytes : 0;
  auto run = [&](auto kernel) {
    // the limit is the function's, not the launch's: one value, so that calls of several threads cannot lower it for each other
    int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BWD ? WIDE_SMEM : 0), fn);
    if (rc) return rc;
    kernel<<<dim3(n.gx, n.gy), WIDE_THREADS, smem, st>>>(q);
    return check_cuda(cudaGetLastError(), fn);
  };
  return p.gate ? run(k_group_norm_wide<T, VEC, true, BWD>) : run(k_group_norm_wide<T, VEC, false, BWD>);
}

template <bool BWD>
static int launch_norm(const NormParams& p, const NormPlan& n, int dtype, cudaStream_t st, const char* fn) {
  if (n.wide) {
    if (dtype == GDN2_DTYPE_F32)
      return n.vec == 4 ? launch_norm_wide<float, 4, BWD>(p, n, st, fn) : launch_norm_wide<float, 1, BWD>(p, n, st, fn);
    return n.vec == 8 ? launch_norm_wide<__nv_bfloat16, 8, BWD>(p, n, st, fn)
                      : launch_norm_wide<__nv_bfloat16, 1, BWD>(p, n, st, fn);
  }
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

int launch_group_norm(const gdn2_group_norm_args* a, void* y, cudaStream_t st) {
  const char* fn = "gdn2_group_norm_gate";
  NormParams p;
  NormPlan n;
  int vec;
  int rc = prep_norm(a, p, vec, fn);
  if (rc) return rc;
  if (!y) return set_error(GDN2_EINVAL, "%s: null tensor pointer", fn);
  vec = least(vec, vec_of(y, (int64_t)p.G * p.D, a->dtype == GDN2_DTYPE_BF16 ? 2 : 4));
  plan_norm(p, a->dtype, vec, NORM_FWD_BLOCKS, n);
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
  plan_norm(p, a->dtype, vec, NORM_BWD_BLOCKS, n);
  p.dy = q->d_y; p.lddy = q->ld_dy;
  p.dx = q->dx; p.dgate = q->d_gate;
  p.want_w = q->d_weight != nullptr;
  p.want_b = q->d_bias != nullptr;
  return GDN2_OK;
}

// Partial rows of the weights' gradients and their columns.
static int64_t norm_part_rows(const NormParams& p, const NormPlan& n) {
  return p.shared_w ? (int64_t)n.gx * n.gy : (int64_t)n.gy * p.row_step;
}
static int norm_part_cols(const NormParams& p) { return p.shared_w ? p.D : p.G * p.D; }
static size_t norm_workspace(const NormParams& p, const NormPlan& n) {
  return (size_t)norm_part_rows(p, n) * norm_part_cols(p) * (p.want_w + p.want_b) * sizeof(float);
}

size_t group_norm_bwd_workspace_bytes(const gdn2_group_norm_bwd_args* q) {
  NormParams p;
  NormPlan n;
  if (plan_norm_bwd(q, p, n, "gdn2_group_norm_gate_bwd_workspace_bytes")) return 0;
  return norm_workspace(p, n);
}

int launch_group_norm_bwd(const gdn2_group_norm_bwd_args* q, void* ws, size_t ws_bytes, cudaStream_t st) {
  const char* fn = "gdn2_group_norm_gate_bwd";
  NormParams p;
  NormPlan n;
  int rc = plan_norm_bwd(q, p, n, fn);
  if (rc) return rc;
  const int arrays = p.want_w + p.want_b;
  const size_t need = norm_workspace(p, n);
  if (need && (!ws || ws_bytes < need))
    return set_error(GDN2_EWORKSPACE, "%s: workspace %zu bytes < required %zu", fn, ws ? ws_bytes : 0, need);
  p.part = static_cast<float*>(ws);
  rc = launch_norm<true>(p, n, q->fwd.dtype, st, fn);
  if (rc || !arrays) return rc;
  float* first = p.want_w ? q->d_weight : q->d_bias;
  return launch_column_sums(p.part, norm_part_rows(p, n), norm_part_cols(p), arrays, first, q->d_bias, st, fn);
}

}  // namespace gdn2

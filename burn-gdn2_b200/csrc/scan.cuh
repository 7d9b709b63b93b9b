// Pieces shared by the sequence operators (gated scan, causal convolution,
// group norm): vector access to rows of channels, staged rows, packed-sequence
// lookup and the decay's exponential.
#pragma once

#include "common.cuh"
#include "ptx.cuh"

namespace gdn2 {

// VEC consecutive elements of T as one memory access of sizeof(T) * VEC bytes.
template <int BYTES>
struct RawOf;
template <>
struct RawOf<2> { typedef unsigned short type; };
template <>
struct RawOf<4> { typedef unsigned type; };
template <>
struct RawOf<8> { typedef uint2 type; };
template <>
struct RawOf<16> { typedef uint4 type; };

template <typename T, int VEC>
struct Vec {
  typedef typename RawOf<(int)sizeof(T) * VEC>::type Raw;
  static __device__ __forceinline__ Raw load(const T* p) { return __ldcs(reinterpret_cast<const Raw*>(p)); }
  static __device__ __forceinline__ void unpack(Raw r, float (&f)[VEC]) {
    T e[VEC];
    memcpy(e, &r, sizeof(r));
    #pragma unroll
    for (int v = 0; v < VEC; ++v) f[v] = to_f32<T>(e[v]);
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[VEC]) {
    T e[VEC];
    #pragma unroll
    for (int v = 0; v < VEC; ++v) e[v] = from_f32<T>(f[v]);
    Raw r;
    memcpy(&r, e, sizeof(r));
    return r;
  }
  static __device__ __forceinline__ void store(T* p, const float (&f)[VEC]) {
    __stcs(reinterpret_cast<Raw*>(p), pack(f));
  }
};

// A vector as pairs of f32 (one pair with a zero for VEC = 1).
template <typename T, int VEC>
__device__ __forceinline__ void unpack_pairs(typename Vec<T, VEC>::Raw r, f32x2 (&f)[VEC == 1 ? 1 : VEC / 2]) {
  float v[VEC == 1 ? 2 : VEC];
  v[VEC == 1 ? 1 : 0] = 0.f;
  Vec<T, VEC>::unpack(r, *reinterpret_cast<float (*)[VEC]>(v));
  #pragma unroll
  for (int i = 0; i < (VEC == 1 ? 1 : VEC / 2); ++i) f[i] = f2pk(v[2 * i], v[2 * i + 1]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pairs(T* p, const f32x2 (&f)[VEC == 1 ? 1 : VEC / 2]) {
  float v[VEC == 1 ? 2 : VEC];
  #pragma unroll
  for (int i = 0; i < (VEC == 1 ? 1 : VEC / 2); ++i) f2un(f[i], v[2 * i], v[2 * i + 1]);
  Vec<T, VEC>::store(p, *reinterpret_cast<const float (*)[VEC]>(v));
}

// Sigmoid of a pair: 1 / (1 + 2^(-t log2 e)) by the approximate exponential
// and reciprocal (2 ulp and 1 ulp), far below the rounding of a bf16 result
// and near f32's own.
__device__ __forceinline__ f32x2 sigmoid2(f32x2 t) {
  float e0, e1;
  f2un(f2mul(t, f2pk(-1.44269504088896f, -1.44269504088896f)), e0, e1);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e0));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e1));
  f2un(f2add(f2pk(e0, e1), f2pk(1.f, 1.f)), e0, e1);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e0));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e1));
  return f2pk(e0, e1);
}

template <int VEC>
__device__ __forceinline__ void load_f32(const float* p, float (&f)[VEC]) {
  #pragma unroll
  for (int v = 0; v < VEC; ++v) f[v] = p[v];
}
template <int VEC>
__device__ __forceinline__ void store_f32(float* p, const float (&f)[VEC]) {
  #pragma unroll
  for (int v = 0; v < VEC; ++v) p[v] = f[v];
}

// Sequence of packed row t: the n with cu[n] <= t < cu[n + 1], or -1 for a
// row outside every sequence.  Reads cu[0..N] only, whatever it holds, and
// takes at most 32 halvings.
__device__ __forceinline__ int find_sequence(const int* __restrict__ cu, int N, int t) {
  int lo = 0, hi = N + 1;  // first index whose entry is above t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= t) lo = mid + 1;
    else hi = mid;
  }
  return lo >= 1 && lo <= N ? lo - 1 : -1;
}

// a = e^g and k = 1 - e^g of two log decays.  Argument reduction by powers of
// two (Cody and Waite): g = n ln 2 + r with |r| <= ln 2 / 2, p = e^r - 1 by its
// Taylor polynomial to r^7 (its first dropped term is below 2^-25 of p), then
// a = 2^n (1 + p), k = (1 - 2^n) - 2^n p.  For n = 0 (the slow channels, whose
// decay is applied thousands of times) a is 1 + p rounded once and k is -p
// itself, without the cancellation of 1 - a: an ulp of bias in a would grow
// by the length of the channel's memory.  Valid for |g| <= 87; NaN stays NaN.
template <bool WITH_K>
__device__ __forceinline__ void exp_pair(f32x2 g, f32x2& a, f32x2& k) {
  const f32x2 kLog2e = f2pk(1.44269504088896f, 1.44269504088896f);
  const f32x2 kMagic = f2pk(12582912.f, 12582912.f);  // 1.5 * 2^23: its sum rounds to a whole number
  const f32x2 kOne = f2pk(1.f, 1.f), kMinus = f2pk(-1.f, -1.f);
  const f32x2 t = f2fma(g, kLog2e, kMagic);
  const f32x2 n = f2fma(kMagic, kMinus, t);
  f32x2 r = f2fma(n, f2pk(-0.693145751953125f, -0.693145751953125f), g);
  r = f2fma(n, f2pk(-1.42860677e-6f, -1.42860677e-6f), r);
  f32x2 q = f2fma(r, f2pk(1.f / 5040, 1.f / 5040), f2pk(1.f / 720, 1.f / 720));
  q = f2fma(q, r, f2pk(1.f / 120, 1.f / 120));
  q = f2fma(q, r, f2pk(1.f / 24, 1.f / 24));
  q = f2fma(q, r, f2pk(1.f / 6, 1.f / 6));
  q = f2fma(q, r, f2pk(0.5f, 0.5f));
  const f32x2 p = f2fma(f2mul(r, r), q, r);
  float t0, t1;
  f2un(t, t0, t1);
  const f32x2 s = f2pk(__uint_as_float((__float_as_uint(t0) << 23) + 0x3f800000u),
                       __uint_as_float((__float_as_uint(t1) << 23) + 0x3f800000u));
  a = f2fma(s, p, s);
  if constexpr (WITH_K) k = f2fma(f2mul(s, kMinus), p, f2fma(s, kMinus, kOne));
}
constexpr float kExpRange = 87.f;

constexpr int RUN = 16;     // tokens of a warp's run
constexpr int STAGES = 2;   // runs in flight or in use

// One warp's staged rows, [RUN][32 * VEC] of T.  Copied 16 bytes a lane over
// several rows where rows allow it (COOP: few instructions; lanes read what
// others copied), else each lane its own values.
template <typename T, int VEC, bool COOP>
struct Rows {
  static constexpr int ROW = 32 * VEC * (int)sizeof(T), BYTES = RUN * ROW;
  unsigned char* base;
  // rows t0 .. of p (its lane 0 channel), those below T, channels below `left`
  __device__ __forceinline__ void fetch(const T* p, int64_t stride, int t0, int T_, int left, int lane) const {
    if constexpr (COOP) {
      constexpr int LANES = ROW / 16, AT_ONCE = 32 / LANES;  // lanes of a row, rows at once
      const int c = lane % LANES * (16 / (int)sizeof(T)), r = lane / LANES;
      const T* q = p + (int64_t)(t0 + r) * stride + c;
      #pragma unroll
      for (int i = 0; i < RUN; i += AT_ONCE) {
        const bool in = c < left && t0 + r + i < T_;
        cp_async_zfill<16>(base + (i + r) * ROW + lane % LANES * 16, in ? q : p, in);
        q += AT_ONCE * stride;
      }
    } else {
      typedef typename Vec<T, VEC>::Raw Raw;
      const T* q = p + (int64_t)t0 * stride + lane * VEC;
      #pragma unroll
      for (int i = 0; i < RUN; ++i) {
        const bool in = lane * VEC < left && t0 + i < T_;
        Raw* to = reinterpret_cast<Raw*>(base + i * ROW) + lane;
        if constexpr (sizeof(Raw) >= 4) cp_async_zfill<(int)sizeof(Raw)>(to, in ? q : p, in);
        else *to = in ? Vec<T, VEC>::load(q) : Raw{};
        q += stride;
      }
    }
  }
  // a lane's channels of row i as a pair (the second zero for VEC = 1)
  __device__ __forceinline__ f32x2 get(int i, int lane) const {
    float f[2] = {0.f, 0.f};
    const T* p = reinterpret_cast<const T*>(base + i * ROW) + lane * VEC;
    if constexpr (VEC == 2) Vec<T, 2>::unpack(*reinterpret_cast<const typename Vec<T, 2>::Raw*>(p), f);
    else f[0] = to_f32<T>(*p);
    return f2pk(f[0], f[1]);
  }
};

template <typename T, int VEC>
__device__ __forceinline__ void put(T* p, f32x2 v) {
  float f[2];
  f2un(v, f[0], f[1]);
  if constexpr (VEC == 2) Vec<T, 2>::store(p, f);
  else {
    float one[1] = {f[0]};
    Vec<T, 1>::store(p, one);
  }
}
template <int VEC>
__device__ __forceinline__ f32x2 get_f32(const float* p) {
  return f2pk(p[0], VEC == 2 ? p[VEC - 1] : 0.f);
}
template <int VEC>
__device__ __forceinline__ void put_f32(float* p, f32x2 v) {
  float f0, f1;
  f2un(v, f0, f1);
  p[0] = f0;
  if (VEC == 2) p[VEC - 1] = f1;
}

// Whether packed sequence n has no row.  Offsets beyond the T rows count as T.
__device__ __forceinline__ bool is_empty(const int* __restrict__ cu, int n, int T) {
  const int from = __ldg(cu + n);
  return __ldg(cu + n + 1) <= from || from >= T;
}

// Rows of v start on `bytes` boundaries.
inline bool rows_ok(const gdn2_view& v, int bytes, int elem) {
  return (uintptr_t)v.data % bytes == 0 && v.stride0 * elem % bytes == 0 && v.stride1 * elem % bytes == 0;
}

inline int elem_bytes(int dtype) { return dtype == GDN2_DTYPE_BF16 ? 2 : 4; }

}  // namespace gdn2

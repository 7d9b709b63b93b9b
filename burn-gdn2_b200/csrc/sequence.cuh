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
  // bf16 in pairs: a shift and a mask to f32, one conversion of both back
  static __device__ __forceinline__ void unpack(Raw r, float (&f)[VEC]) {
    if constexpr (sizeof(T) == 2 && VEC > 1) {
      unsigned w[VEC / 2];
      memcpy(w, &r, sizeof(r));
      #pragma unroll
      for (int v = 0; v < VEC / 2; ++v) {
        f[2 * v] = __uint_as_float(w[v] << 16);
        f[2 * v + 1] = __uint_as_float(w[v] & 0xffff0000u);
      }
    } else {
      T e[VEC];
      memcpy(e, &r, sizeof(r));
      #pragma unroll
      for (int v = 0; v < VEC; ++v) f[v] = to_f32<T>(e[v]);
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[VEC]) {
    Raw r;
    if constexpr (sizeof(T) == 2 && VEC > 1) {
      __nv_bfloat162 w[VEC / 2];
      #pragma unroll
      for (int v = 0; v < VEC / 2; ++v) w[v] = __floats2bfloat162_rn(f[2 * v], f[2 * v + 1]);
      memcpy(&r, w, sizeof(r));
    } else {
      T e[VEC];
      #pragma unroll
      for (int v = 0; v < VEC; ++v) e[v] = from_f32<T>(f[v]);
      memcpy(&r, e, sizeof(r));
    }
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
// and reciprocal (2 ulp and 1 ulp).  The rounded product t log2 e adds up to
// 2 |t| half-steps, relative, where the exponential counts (t < 0), so an f32
// silu is off by (16 + 2 |t|) 2^-24 of its value at most: below the rounding of
// a bf16 result, a few times expf's own error near t = 0 and more on the left.
// From about t = -87.3 down the reciprocal is below the smallest normal f32 and
// counts as zero (silu's true value there is 1e-36 and less).
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

// How a warp holds rows of 64 channels, a pair of channels a lane, in shared
// memory.  All but the last copy 16 aligned bytes a lane over several rows, few
// instructions, and lanes read what others copied:
//   ROWS16     rows start on 16 bytes; a lane's pair are neighbours
//   ROWS_PAIR  rows start on the pair's size: copied from the 16 bytes below
//              their start on, which the reader skips (pitch one vector more)
//   ROWS_ODD   the same for rows of any start; pairs are channels lane, lane + 32
//   ROWS_ANY   a tensor that itself starts off 16 bytes (the bytes below its
//              first row are not its own): each lane copies its own elements
enum RowMode { ROWS16, ROWS_PAIR, ROWS_ODD, ROWS_ANY };
constexpr int SET = 64;  // channels of a warp's rows

// The channels of a lane in a set of `left` channels; the first is one where
// the second is.  Stores are for lanes whose first is (on0).
template <RowMode MODE>
struct Pair {
  static constexpr bool NEXT = MODE == ROWS16 || MODE == ROWS_PAIR;  // neighbours
  int c0, c1;     // offsets in the set
  bool on0, on1;  // whether they are channels
  __device__ __forceinline__ Pair(int lane, int left)
      : c0(NEXT ? 2 * lane : lane), c1(NEXT ? 2 * lane + 1 : lane + 32), on0(c0 < left), on1(c1 < left) {}
  template <typename T>
  __device__ __forceinline__ f32x2 load(const T* p) const {  // p: the set's first channel
    float f[2] = {0.f, 0.f};
    if constexpr (NEXT && sizeof(T) == 2) {
      if (on0) Vec<T, 2>::unpack(Vec<T, 2>::load(p + c0), f);
    } else {  // f32 rows beside bf16 ones may start on 4 bytes
      if (on0) f[0] = to_f32<T>(p[c0]);
      if (on1) f[1] = to_f32<T>(p[c1]);
    }
    return f2pk(f[0], f[1]);
  }
  template <typename T>
  __device__ __forceinline__ void store(T* p, f32x2 v) const {
    float f[2];
    f2un(v, f[0], f[1]);
    if constexpr (NEXT) {
      Vec<T, 2>::store(p + c0, f);
    } else {
      __stcs(p + c0, from_f32<T>(f[0]));
      if (on1) __stcs(p + c1, from_f32<T>(f[1]));
    }
  }
  // a state, cache or carry, which may start on any f32
  __device__ __forceinline__ void store_state(float* p, f32x2 v) const {
    float f[2];
    f2un(v, f[0], f[1]);
    p[c0] = f[0];
    if (on1) p[c1] = f[1];
  }
};

// One warp's staged rows, [RUN][SET] of T.
template <typename T, RowMode MODE>
struct Rows {
  static constexpr int E = (int)sizeof(T), ROW = SET * E;
  static constexpr bool SHIFTED = MODE == ROWS_PAIR || MODE == ROWS_ODD;
  static constexpr int PITCH = ROW + (SHIFTED ? 16 : 0), BYTES = RUN * PITCH;
  unsigned char* base;
  // rows t0 .. of p (the set's first channel), those below `end`, channels below `left`
  __device__ __forceinline__ void fetch(const T* p, int64_t stride, int t0, int end, int left, int lane) const {
    if constexpr (MODE == ROWS16) {
      constexpr int LANES = ROW / 16, AT_ONCE = 32 / LANES;  // lanes of a row, rows at once
      const int c = lane % LANES * (16 / E), r = lane / LANES;
      const T* q = p + (int64_t)(t0 + r) * stride + c;
      #pragma unroll
      for (int i = 0; i < RUN; i += AT_ONCE) {
        const bool in = c < left && t0 + r + i < end;
        cp_async_zfill<16>(base + (i + r) * PITCH + lane % LANES * 16, in ? q : p, in ? 16 : 0);
        q += AT_ONCE * stride;
      }
    } else if constexpr (SHIFTED) {
      constexpr int CHUNKS = PITCH / 16;  // 16-byte pieces of a row
      const int bytes = (left < SET ? left : SET) * E;
      const char* q = reinterpret_cast<const char*>(p) + (int64_t)t0 * stride * E;
      #pragma unroll
      for (int i = 0; i < RUN * CHUNKS; i += 32) {
        const int n = i + lane, r = n / CHUNKS, c = n % CHUNKS * 16;
        if (n >= RUN * CHUNKS) break;
        const char* row = q + (int64_t)r * stride * E;
        const int skip = (int)((uintptr_t)row & 15);
        int size = bytes + skip - c;  // valid bytes from the piece on
        size = size > 16 ? 16 : size;
        const bool in = size > 0 && t0 + r < end;
        const char* from = in ? row - skip + c : reinterpret_cast<const char*>((uintptr_t)p & ~(uintptr_t)15);
        cp_async_zfill<16>(base + r * PITCH + c, from, in ? size : 0);
      }
    } else {
      const T* q = p + (int64_t)t0 * stride + lane;
      #pragma unroll
      for (int i = 0; i < RUN; ++i) {
        T* to = reinterpret_cast<T*>(base + i * PITCH) + lane;
        #pragma unroll
        for (int v = 0; v < SET; v += 32) {
          const bool in = lane + v < left && t0 + i < end;
          if constexpr (E >= 4) cp_async_zfill<4>(to + v, in ? q + v : p, in ? 4 : 0);
          else to[v] = in ? __ldcs(q + v) : T(0.f);
        }
        q += stride;
      }
    }
  }
  // where row i starts in a shifted copy: the low bits of its address
  struct View {
    const unsigned char* base;
    unsigned start, step;
    int lane;
    // a lane's pair of row i
    __device__ __forceinline__ f32x2 get(int i) const {
      const unsigned char* at = base + i * PITCH;
      if constexpr (SHIFTED) at += (start + i * step) & 15;
      const T* p = reinterpret_cast<const T*>(at);
      if constexpr (!Pair<MODE>::NEXT) return f2pk(to_f32<T>(p[lane]), to_f32<T>(p[lane + 32]));
      float f[2];
      Vec<T, 2>::unpack(*reinterpret_cast<const typename Vec<T, 2>::Raw*>(p + 2 * lane), f);
      return f2pk(f[0], f[1]);
    }
  };
  __device__ __forceinline__ View view(const T* p, int64_t stride, int t0, int lane) const {
    return View{base, SHIFTED ? (unsigned)(uintptr_t)(p + (int64_t)t0 * stride) : 0u, SHIFTED ? (unsigned)(stride * E) : 0u, lane};
  }
};

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

// How rows of these tensors (elements of e bytes, `staged` ones copied to
// shared memory) can be held.
struct RowTensor {
  const gdn2_view* v;
  int e;
  bool staged;
};
inline RowMode row_mode(int channels, const RowTensor* t, int count) {
  bool pairs = channels % 2 == 0, sixteen = true, based = true;
  for (int i = 0; i < count; ++i) {
    pairs = pairs && rows_ok(*t[i].v, 2 * t[i].e, t[i].e);
    if (!t[i].staged) continue;
    sixteen = sixteen && channels * t[i].e % 16 == 0 && rows_ok(*t[i].v, 16, t[i].e);
    based = based && (uintptr_t)t[i].v->data % 16 == 0;
  }
  return pairs && sixteen ? ROWS16 : !based ? ROWS_ANY : pairs ? ROWS_PAIR : ROWS_ODD;
}

}  // namespace gdn2

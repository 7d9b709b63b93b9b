// Moving the rows of state pools: for every tensor of a pool, row d becomes
// what row index[d] was, all rows at once (a parallel assignment, so that
// rows may be swapped, forked and moved down in the same call); -1 frees a
// row (zeros), a row's own number leaves it alone.
//
// Bound by HBM: every moved row is read and written once, no other row is
// touched.  A block owns a span of byte columns across all rows.  It packs
// the list of moved rows, reads that span of every source into shared memory
// and writes it only after the last of them has been read, so no row has to
// be staged elsewhere and no order of moves can go wrong.  The span is
// narrowed until all moved rows fit.
#include "scan.cuh"

namespace gdn2 {

constexpr int ROWS_THREADS = 256, ROWS_BLOCKS = 2;  // threads, blocks per SM
constexpr int ROWS_SMEM = 96 * 1024;                // list of moved rows, then the staged spans
constexpr int MAX_POOL = 16;                        // tensors a launch takes

struct RowsParams {
  int count, src_rows, dst_rows;
  bool inplace;
  const int* index;
  struct { const unsigned char* src; unsigned char* dst; int64_t bytes; int width; } t[MAX_POOL];
};

template <typename W>
__device__ __forceinline__ void move_spans(const unsigned char* src, unsigned char* dst, int64_t bytes,
                                           const int2* moves, int n, unsigned char* stage, int room) {
  W* buf = reinterpret_cast<W*>(stage);
  const int64_t words = bytes / (int64_t)sizeof(W);
  // words of a span: as many as leave room for every moved row, a power of two up to the block
  int span = ROWS_THREADS;
  while (span > 1 && (int64_t)span * n * (int)sizeof(W) > room) span >>= 1;
  const int col = threadIdx.x % span, row0 = threadIdx.x / span, rows = ROWS_THREADS / span;
  for (int64_t at = (int64_t)blockIdx.x * span; at < words; at += (int64_t)gridDim.x * span) {
    const int64_t w = at + col;
    if (w < words)
      #pragma unroll 8
      for (int i = row0; i < n; i += rows) {
        const int s = moves[i].y;
        buf[i * span + col] = s >= 0 ? __ldcs(reinterpret_cast<const W*>(src + (int64_t)s * bytes) + w) : W{};
      }
    __syncthreads();
    if (w < words)
      #pragma unroll 8
      for (int i = row0; i < n; i += rows)
        __stcs(reinterpret_cast<W*>(dst + (int64_t)moves[i].x * bytes) + w, buf[i * span + col]);
    __syncthreads();
  }
}

__global__ void __launch_bounds__(ROWS_THREADS) k_state_rows(RowsParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  int2* moves = reinterpret_cast<int2*>(smem);  // (row, source)
  __shared__ int counts[ROWS_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int n = 0;
  for (int d0 = 0; d0 < p.dst_rows; d0 += ROWS_THREADS) {
    const int d = d0 + threadIdx.x;
    int s = 0;
    bool moved = false;
    if (d < p.dst_rows) {
      s = __ldg(p.index + d);
      const bool bad = s < -1 || s >= p.src_rows;
      if (bad && blockIdx.x == 0) atomicOr(&g_device_errors, DEVERR_STATE_INDEX);
      moved = !p.inplace || (!bad && s != d);
      if (bad) s = -1;
    }
    const unsigned m = __ballot_sync(0xffffffffu, moved);
    if (lane == 0) counts[warp] = __popc(m);
    __syncthreads();
    int at = n;
    #pragma unroll
    for (int w = 0; w < ROWS_THREADS / 32; ++w) {
      if (w == warp && moved) moves[at + __popc(m & ((1u << lane) - 1))] = make_int2(d, s);
      at += counts[w];
    }
    n = at;
    __syncthreads();
  }
  if (!n) return;
  const int list = (n * (int)sizeof(int2) + 15) / 16 * 16;
  unsigned char* stage = smem + list;
  for (int k = 0; k < p.count; ++k) {
    if (p.t[k].width == 16)
      move_spans<uint4>(p.t[k].src, p.t[k].dst, p.t[k].bytes, moves, n, stage, ROWS_SMEM - list);
    else if (p.t[k].width == 4)
      move_spans<unsigned>(p.t[k].src, p.t[k].dst, p.t[k].bytes, moves, n, stage, ROWS_SMEM - list);
    else
      move_spans<unsigned char>(p.t[k].src, p.t[k].dst, p.t[k].bytes, moves, n, stage, ROWS_SMEM - list);
  }
}

GDN2_DEVICE_ERROR_READER(read_device_errors_state_rows)

int launch_state_rows(const gdn2_state_rows* t, int32_t count, const int32_t* index, int32_t src_rows,
                      int32_t dst_rows, cudaStream_t st) {
  const char* fn = "gdn2_move_state_rows";
  if (count < 0 || src_rows < 0 || dst_rows < 0)
    return set_error(GDN2_EINVAL, "%s: negative size (count=%d src_rows=%d dst_rows=%d)", fn, count, src_rows, dst_rows);
  if (!count || !dst_rows) return GDN2_OK;
  if (!t || !index) return set_error(GDN2_EINVAL, "%s: null pointer", fn);
  static_assert(GDN2_MAX_STATE_ROWS * (16 + sizeof(int2)) <= ROWS_SMEM, "a word of every row and the list of moves");
  if (dst_rows > GDN2_MAX_STATE_ROWS)
    return set_error(GDN2_EUNSUPPORTED, "%s: %d rows, at most %d", fn, dst_rows, GDN2_MAX_STATE_ROWS);
  bool inplace = false;
  for (int k = 0; k < count; ++k) {
    if ((!t[k].src && src_rows) || !t[k].dst || t[k].row_bytes <= 0)
      return set_error(GDN2_EINVAL, "%s: tensor %d: null pointer or no bytes", fn, k);
    const bool same = t[k].src == t[k].dst;
    if (k && same != inplace) return set_error(GDN2_EINVAL, "%s: tensors in place and not in one call", fn);
    inplace = same;
    const char* a = static_cast<const char*>(t[k].src);
    const char* b = static_cast<const char*>(t[k].dst);
    if (!same && a < b + (int64_t)dst_rows * t[k].row_bytes && b < a + (int64_t)src_rows * t[k].row_bytes)
      return set_error(GDN2_EINVAL, "%s: tensor %d: source and destination overlap", fn, k);
  }
  if (inplace && src_rows != dst_rows)
    return set_error(GDN2_EINVAL, "%s: in place with %d and %d rows", fn, src_rows, dst_rows);
  int rc = check_cuda(cudaFuncSetAttribute(k_state_rows, cudaFuncAttributeMaxDynamicSharedMemorySize, ROWS_SMEM), fn);
  for (int first = 0; !rc && first < count; first += MAX_POOL) {
    RowsParams p;
    p.count = count - first < MAX_POOL ? count - first : MAX_POOL;
    p.src_rows = src_rows; p.dst_rows = dst_rows;
    p.inplace = inplace;
    p.index = index;
    int64_t widest = 0;
    for (int k = 0; k < p.count; ++k) {
      const gdn2_state_rows& e = t[first + k];
      const uintptr_t all = (uintptr_t)e.src | (uintptr_t)e.dst | (uintptr_t)e.row_bytes;
      p.t[k] = {static_cast<const unsigned char*>(e.src), static_cast<unsigned char*>(e.dst), e.row_bytes,
                all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1};
      const int64_t spans = e.row_bytes / p.t[k].width;
      widest = spans > widest ? spans : widest;
    }
    const int64_t want = (widest + 3) / 4;  // a block has at least a few words of every row to do
    const int blocks = (int)(want < 148 * ROWS_BLOCKS ? want : 148 * ROWS_BLOCKS);
    k_state_rows<<<blocks, ROWS_THREADS, ROWS_SMEM, st>>>(p);
    rc = check_cuda(cudaGetLastError(), fn);
  }
  return rc;
}

}  // namespace gdn2

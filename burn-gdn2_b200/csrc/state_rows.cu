// Moving the rows of state pools: for every tensor of a pool, row d becomes
// what row index[d] was, all rows at once (a parallel assignment, so that
// rows may be swapped, forked and moved down in the same call); -1 frees a
// row (zeros), a row's own number leaves it alone.
//
// Bound by HBM: every moved row is read and written once, no other row is
// touched (43 of 256 rows of 1.1 MB: 18.8 us, 79 % of what a copy reaches).
// Each block packs the list of moved rows.  Where no move's source
// is overwritten by another one (a compaction, a fork, rows gathered into
// another pool) the blocks copy pieces of rows in no particular order (256 rows
// of 1 MB into another pool: 80 us, all of what a copy reaches).
// Otherwise a block owns a span of byte columns across all rows, reads that
// span of every source into shared memory and writes it only after the last
// of them has been read, so no order of moves can go wrong; the span is
// narrowed until all moved rows fit.
#include "sequence.cuh"

namespace gdn2 {

constexpr int ROWS_THREADS = 256;
constexpr int ROWS_SMEM_MIN = 16 * 1024, ROWS_SMEM_MAX = 96 * 1024;  // list of moved rows, then the staged spans
constexpr int MAX_POOL = 16;                                         // tensors a launch takes
constexpr int PIECE_WORDS = 4;                                       // words of a piece per thread

struct RowsParams {
  int count, src_rows, dst_rows, smem;
  bool inplace;
  const int* index;
  int64_t pieces;  // of one row, over all tensors
  struct {
    const unsigned char* src;
    unsigned char* dst;
    int64_t bytes, first_piece;
    int width;
  } t[MAX_POOL];
};

// Piece `at` of a row: PIECE_WORDS words a thread.
template <typename W>
__device__ __forceinline__ void copy_piece(const unsigned char* src, unsigned char* dst, int64_t bytes, int64_t at, int2 move) {
  const int64_t words = bytes / (int64_t)sizeof(W), w0 = at * (ROWS_THREADS * PIECE_WORDS) + threadIdx.x;
  const W* from = reinterpret_cast<const W*>(src + (int64_t)(move.y < 0 ? 0 : move.y) * bytes);
  W* to = reinterpret_cast<W*>(dst + (int64_t)move.x * bytes);
  W v[PIECE_WORDS];
  #pragma unroll
  for (int i = 0; i < PIECE_WORDS; ++i) {
    const int64_t w = w0 + i * ROWS_THREADS;
    v[i] = move.y >= 0 && w < words ? __ldcs(from + w) : W{};
  }
  #pragma unroll
  for (int i = 0; i < PIECE_WORDS; ++i) {
    const int64_t w = w0 + i * ROWS_THREADS;
    if (w < words) __stcs(to + w, v[i]);
  }
}

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
  int n = 0, entangled = 0;
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
      if (p.inplace && moved && s >= 0) {
        const int over = __ldg(p.index + s);  // is the source a moved row too?
        entangled |= over != s && over >= -1 && over < p.src_rows;
      }
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
  if (!__syncthreads_or(entangled)) {
    for (int64_t unit = blockIdx.x; unit < n * p.pieces; unit += gridDim.x) {
      const int64_t piece = unit % p.pieces;
      int k = 0;
      while (k + 1 < p.count && piece >= p.t[k + 1].first_piece) ++k;
      const int64_t at = piece - p.t[k].first_piece;
      const int2 move = moves[unit / p.pieces];
      if (p.t[k].width == 16) copy_piece<uint4>(p.t[k].src, p.t[k].dst, p.t[k].bytes, at, move);
      else if (p.t[k].width == 4) copy_piece<unsigned>(p.t[k].src, p.t[k].dst, p.t[k].bytes, at, move);
      else copy_piece<unsigned char>(p.t[k].src, p.t[k].dst, p.t[k].bytes, at, move);
    }
    return;
  }
  const int list = (n * (int)sizeof(int2) + 15) / 16 * 16;
  unsigned char* stage = smem + list;
  const int room = p.smem - list;
  for (int k = 0; k < p.count; ++k) {
    if (p.t[k].width == 16) move_spans<uint4>(p.t[k].src, p.t[k].dst, p.t[k].bytes, moves, n, stage, room);
    else if (p.t[k].width == 4) move_spans<unsigned>(p.t[k].src, p.t[k].dst, p.t[k].bytes, moves, n, stage, room);
    else move_spans<unsigned char>(p.t[k].src, p.t[k].dst, p.t[k].bytes, moves, n, stage, room);
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
  static_assert(GDN2_MAX_STATE_ROWS * (16 + sizeof(int2)) <= ROWS_SMEM_MAX, "a word of every row and the list of moves");
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
  // Room for 64 bytes of every row: narrow spans in many blocks on an SM hold more in flight than wide ones in few.
  // 256 rows of 1.1 MB, a turn of all rows: 163 us (187 with 128 bytes, 181 with 256); 43 of them moved into holes,
  // where nothing is staged: 18.7 us (20.3, 22.6).
  const int want = dst_rows * (int)(sizeof(int2) + 64) + 16;
  const int smem = want < ROWS_SMEM_MIN ? ROWS_SMEM_MIN : want > ROWS_SMEM_MAX ? ROWS_SMEM_MAX : want / 16 * 16;
  // the limit is the function's, not the launch's: one value, so that calls of several threads cannot lower it for each other
  int rc = check_cuda(cudaFuncSetAttribute(k_state_rows, cudaFuncAttributeMaxDynamicSharedMemorySize, ROWS_SMEM_MAX), fn);
  for (int first = 0; !rc && first < count; first += MAX_POOL) {
    RowsParams p;
    p.count = count - first < MAX_POOL ? count - first : MAX_POOL;
    p.src_rows = src_rows; p.dst_rows = dst_rows;
    p.smem = smem;
    p.inplace = inplace;
    p.index = index;
    p.pieces = 0;
    for (int k = 0; k < p.count; ++k) {
      const gdn2_state_rows& e = t[first + k];
      const uintptr_t all = (uintptr_t)e.src | (uintptr_t)e.dst | (uintptr_t)e.row_bytes;
      const int width = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
      p.t[k] = {static_cast<const unsigned char*>(e.src), static_cast<unsigned char*>(e.dst), e.row_bytes, p.pieces, width};
      const int64_t piece = (int64_t)width * ROWS_THREADS * PIECE_WORDS;
      p.pieces += (e.row_bytes + piece - 1) / piece;
    }
    // every SM filled, or a piece of every row at most
    const int64_t most = p.pieces * dst_rows, resident = 148 * (int64_t)(200 * 1024 / smem < 8 ? 200 * 1024 / smem : 8);
    const int blocks = (int)(most < resident ? most : resident);
    k_state_rows<<<blocks, ROWS_THREADS, smem, st>>>(p);
    rc = check_cuda(cudaGetLastError(), fn);
  }
  return rc;
}

}  // namespace gdn2

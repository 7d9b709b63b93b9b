// Gated scan, host side: argument checks, how a call is cut up, and its
// launches (kernels: scan.cuh).
#include "scan.cuh"

namespace gdn2 {

template <typename TX, typename TG>
static int resident(RowMode mode, bool bwd) {
  return mode == ROWS16      ? resident_blocks<TX, TG, ROWS16>(4, bwd)
         : mode == ROWS_PAIR ? resident_blocks<TX, TG, ROWS_PAIR>(4, bwd)
         : mode == ROWS_ODD  ? resident_blocks<TX, TG, ROWS_ODD>(4, bwd)
                             : resident_blocks<TX, TG, ROWS_ANY>(4, bwd);
}

static ScanPlan plan_scan(const gdn2_scan_args* a, RowMode mode, bool bwd) {
  ScanPlan n;
  n.mode = mode;
  n.sets = (a->channels + SET - 1) / SET;
  n.chains = (int64_t)n.sets * (a->cu_seqlens ? 1 : a->batch);
  const int runs = (a->seq_len + RUN - 1) / RUN;
  // 4096 tokens of 32 n chains, bf16 x and f32 g, forward: n = 2: segments 53 us, eight warps 62; n = 3: 71 and 63;
  // n = 8: eight warps 102, four 98.  Measured at this length alone.
  const bool cut = n.chains < 80;
  n.warps = cut || n.chains >= 220 ? 4 : 8;
  const int tiles = (runs + n.warps - 1) / n.warps;
  n.segments = 1;
  n.steps = tiles;
  if (cut) {
    // one wave of resident blocks: a second one would walk as long again
    typedef __nv_bfloat16 bf;
    const int per_sm = a->dtype == GDN2_DTYPE_F32     ? resident<float, float>(mode, bwd)
                       : a->g_dtype == GDN2_DTYPE_F32 ? resident<bf, float>(mode, bwd)
                                                      : resident<bf, bf>(mode, bwd);
    int64_t want = 148 * per_sm / n.chains;
    want = want < MAX_SEGMENTS ? want : MAX_SEGMENTS;
    want = want < tiles ? want : tiles;
    if (want > 1) {
      n.steps = (int)((tiles + want - 1) / want);
      n.segments = (tiles + n.steps - 1) / n.steps;
    }
  }
  return n;
}

// Workspace of a cut time axis: the maps, their cut flags, and a copy of the
// initial states for a call that writes the final ones over them.
struct ScanSpace {
  size_t cuts, states, bytes;
};
static ScanSpace scan_workspace(const ScanPlan& n, const gdn2_scan_args* a) {
  ScanSpace w{};
  if (n.segments == 1) return w;
  w.cuts = (size_t)n.chains * n.segments * 32 * sizeof(ulonglong2);
  w.states = w.cuts + ((size_t)n.chains * n.segments * sizeof(int) + 15) / 16 * 16;
  w.bytes = w.states + (a->state_in ? (size_t)a->batch * a->channels * sizeof(float) : 0);
  return w;
}

static int dispatch(ScanParams& p, const gdn2_scan_args* a, const ScanPlan& n, bool bwd, void* ws, size_t ws_bytes,
                    cudaStream_t st, const char* fn) {
  const ScanSpace w = scan_workspace(n, a);
  if (w.bytes && (!ws || ws_bytes < w.bytes))
    return set_error(GDN2_EWORKSPACE, "%s: workspace %zu bytes < required %zu", fn, ws ? ws_bytes : 0, w.bytes);
  if (w.bytes && (uintptr_t)ws % 16) return set_error(GDN2_EINVAL, "%s: workspace must be 16-byte aligned", fn);
  p.sets = n.sets; p.steps = n.steps; p.segments = n.segments;
  if (w.bytes) {
    char* at = static_cast<char*>(ws);
    p.maps = reinterpret_cast<ulonglong2*>(at);
    p.map_cuts = reinterpret_cast<int*>(at + w.cuts);
    if (!bwd && p.state_in && p.state_in == p.state_out) {
      int rc = check_cuda(cudaMemcpyAsync(at + w.states, p.state_in, (size_t)p.B * p.C * sizeof(float),
                                          cudaMemcpyDeviceToDevice, st), fn);
      if (rc) return rc;
      p.state_in = reinterpret_cast<const float*>(at + w.states);
    }
  }
  const bool comp = a->complement != 0;
  if (a->dtype == GDN2_DTYPE_F32) return run_types<float, float>(p, n, comp, bwd, st, fn);
  if (a->g_dtype == GDN2_DTYPE_F32) return run_types<__nv_bfloat16, float>(p, n, comp, bwd, st, fn);
  return run_types<__nv_bfloat16, __nv_bfloat16>(p, n, comp, bwd, st, fn);
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

static ScanPlan plan_fwd(const gdn2_scan_args* a, const gdn2_view& h) {
  const int ex = elem_bytes(a->dtype), eg = elem_bytes(a->g_dtype);
  const RowTensor t[] = {{&a->x, ex, true}, {&a->g, eg, true}, {&h, ex, false}};
  return plan_scan(a, row_mode(a->channels, t, 3), false);
}

static ScanPlan plan_bwd(const gdn2_scan_bwd_args* q) {
  const gdn2_scan_args* a = &q->fwd;
  const int ex = elem_bytes(a->dtype), eg = elem_bytes(a->g_dtype);
  const RowTensor t[] = {{&a->x, ex, true}, {&a->g, eg, true}, {&q->d_h, ex, true}, {&q->dx, ex, false}, {&q->dg, eg, false}};
  return plan_scan(a, row_mode(a->channels, t, 5), true);
}

size_t scan_workspace_bytes(const gdn2_scan_args* a, const gdn2_view& h) {
  return check_scan(a, "gdn2_gated_scan_workspace_bytes") ? 0 : scan_workspace(plan_fwd(a, h), a).bytes;
}
size_t scan_bwd_workspace_bytes(const gdn2_scan_bwd_args* q) {
  return !q || check_scan(&q->fwd, "gdn2_gated_scan_bwd_workspace_bytes") ? 0 : scan_workspace(plan_bwd(q), &q->fwd).bytes;
}

int launch_scan_fwd(const gdn2_scan_args* a, const gdn2_view& h, float* state_out, void* ws, size_t ws_bytes,
                    cudaStream_t st) {
  const char* fn = "gdn2_gated_scan";
  int rc = check_scan(a, fn);
  if (rc) return rc;
  if (a->seq_len && !h.data) return set_error(GDN2_EINVAL, "%s: null tensor pointer", fn);
  ScanParams p;
  fill(p, a);
  p.h = make_dview(h);
  p.state_out = state_out;
  return dispatch(p, a, plan_fwd(a, h), false, ws, ws_bytes, st, fn);
}

int launch_scan_bwd(const gdn2_scan_bwd_args* q, void* ws, size_t ws_bytes, cudaStream_t st) {
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
  return dispatch(p, a, plan_bwd(q), true, ws, ws_bytes, st, fn);
}

}  // namespace gdn2

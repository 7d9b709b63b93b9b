"""GPU: gated_scan and causal_conv_silu on launch paths that take a certain number of chains (sequences times sets of
64 channels), a certain length or tensors of a certain start: eight-warp blocks, segments of several tiles, tensors that
start off 16 bytes, with gradients.  Bounds as in test_gpu_scan.py and test_gpu_conv.py (sequence_ref)."""
import pytest
import torch

import sequence_ref as R
from test_gpu_scan import DT, TYPES, _check, _decay, _gen, _inputs, _run

pytestmark = pytest.mark.gpu


def _check_sequences(got, xs, gs, st, dh, ds, T, comp, which):
    for b in which:
        part, rows = slice(b * T, (b + 1) * T), xs.shape[0]
        want, bound = R.scan(xs[part], gs[part], st[b:b + 1], [T], comp, dh[part], ds[b:b + 1])
        _check({k: v[part] if v.shape[0] == rows else v[b:b + 1] for k, v in got.items()}, want, bound)


@pytest.mark.parametrize("x,g", TYPES)
@pytest.mark.parametrize("C", [64, 65, 66])
@pytest.mark.parametrize("T,comp", [(1, True), (127, False), (129, True), (300, False)])
def test_eight_warps(x, g, C, T, comp):
    """100 to 200 chains: blocks of eight warps, tiles of 128 tokens."""
    B = 100
    xs, gs, st, dh, ds = _inputs(B * T, C, B, x, g, True, T + C)
    got = _run(xs, gs, st, dh, ds, (B, T), None, comp, True)
    _check_sequences(got, xs, gs, st, dh, ds, T, comp, (0, 57, 99))
    h = _run(xs, gs, st, dh, ds, (B, T), None, comp, False)
    assert torch.equal(h["h"], got["h"]) or T == 1  # one token alone is another kernel


@pytest.mark.parametrize("x,g", TYPES)
@pytest.mark.parametrize("C", [5200, 5121])
def test_eight_warps_packed(x, g, C):
    lens, behind = [130, 0, 17, 200, 1], 11
    rows = sum(lens) + behind
    xs, gs, st, dh, ds = _inputs(rows, C, len(lens), x, g, True, C)
    for t in (xs, gs, dh):
        t[-behind:] = 0
    want, bound = R.scan(xs, gs, st, lens, True, dh, ds)
    xs[-behind:], gs[-behind:], dh[-behind:] = float("nan"), float("inf"), float("nan")
    cu = torch.tensor([0] + lens).cumsum(0).int()
    _check(_run(xs, gs, st, dh, ds, (1, rows), cu, True, True), want, bound)


@pytest.mark.parametrize("B,T,C,x,g", [(1, 24581, 12, "f32", "f32"), (1, 24581, 13, "bf16", "f32"), (79, 4000, 64, "f32", "f32"),
                                       (79, 4000, 64, "bf16", "bf16")])
def test_segments_of_several_tiles(B, T, C, x, g):
    """One chain of 385 tiles, 79 of 63: a segment is several tiles long in both directions."""
    xs, gs, st, dh, ds = _inputs(B * T, C, B, x, g, True, T)
    got = _run(xs, gs, st, dh, ds, (B, T), None, True, True)
    _check_sequences(got, xs, gs, st, dh, ds, T, True, sorted({0, B // 2, B - 1}))
    again = _run(xs, gs, st, dh, ds, (B, T), None, True, True)
    assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize("C,segment,x,g", [(20, 256, "f32", "f32"), (21, 256, "bf16", "f32"), (79 * 64, 832, "f32", "f32")])
def test_packed_boundaries_in_segments(C, segment, x, g):
    """Sequences that begin in the first, a middle and the last tile of a segment, at its start and its end, and that
    lie within one or span several."""
    rows = 24600 if C < 100 else 4000
    marks = [10, 3 * segment, segment + 100, segment // 2, 2 * segment - 6, 3 * segment + 64, 4 * segment - 1]
    if C < 100:
        marks += [11 * segment + 250, 20 * segment + 64, 40 * segment, 40 * segment + 130, 95 * segment + 200]
    marks = sorted(m for m in marks if m < rows - 40)
    lens = [b - a for a, b in zip([0] + marks, marks + [rows - 30])]
    lens.insert(3, 0)
    xs, gs, st, dh, ds = _inputs(rows, C, len(lens), x, g, True, C)
    cu = torch.tensor([0] + lens).cumsum(0).int()
    got = _run(xs, gs, st, dh, ds, (1, rows), cu, False, True)
    cols = torch.arange(C) if C < 100 else torch.cat((torch.arange(66), torch.arange(C - 6, C)))
    pick = lambda t: t[..., cols]
    for t in (xs, gs, dh):
        t[-30:] = 0
    want, bound = R.scan(pick(xs), pick(gs), pick(st), lens, False, pick(dh), pick(ds))
    _check({k: pick(v.cpu()) for k, v in got.items()}, want, bound)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,C,cut", [(70, 33, None), (70, 64, None), (700, 40, None), (150, 64, [40, 0, 100])])
@pytest.mark.parametrize("side", ["x", "g", "both"])
def test_scan_gradients_off_16_bytes(dtype, T, C, cut, side):
    """Training through column slices that start one element into a buffer."""
    import burn_gdn2 as bg

    lens = cut or [T]
    N = len(lens)
    xs, gs, st, dh, ds = _inputs(T, C, N, dtype, dtype, True, T + C)
    want, bound = R.scan(xs[:sum(lens)], gs[:sum(lens)], st, lens, False, dh[:sum(lens)], ds)

    def off(t, yes):
        if not yes:
            return (t[None].cuda().requires_grad_(True),) * 2
        wide = torch.zeros(1, T, C + 3, dtype=t.dtype, device="cuda")
        wide[:, :, 1:1 + C] = t
        wide.requires_grad_(True)
        part = wide[:, :, 1:1 + C]
        assert part.data_ptr() % 16
        return wide, part

    xw, xp = off(xs, side != "g")
    gw, gp = off(gs, side != "x")
    s = st.cuda().requires_grad_(True)
    cu = None if cut is None else torch.tensor([0] + lens).cumsum(0).int()
    h, last = bg.gated_scan(xp, gp, s, cu_seqlens=cu)
    dx, dg, dstate = torch.autograd.grad((h, last), (xw, gw, s), (dh[None].cuda(), ds.cuda()))
    inner = lambda t: (t if t.shape[-1] == C else t[:, :, 1:1 + C])[0, :sum(lens)]
    _check({"h": h.detach()[0, :sum(lens)], "state": last.detach(), "dx": inner(dx), "dg": inner(dg), "d_state": dstate}, want, bound)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,C,cut", [(70, 33, None), (70, 64, None), (400, 130, None), (150, 64, [40, 0, 3, 100])])
def test_conv_gradients_off_16_bytes(dtype, T, C, cut):
    import burn_gdn2 as bg

    lens = cut or [T]
    N, R0 = len(lens), sum(cut or [T])
    gen = _gen(T + C)
    xs, dy = torch.randn(T, C, generator=gen).to(DT[dtype]), torch.randn(T, C, generator=gen).to(DT[dtype])
    w, cache, dc = torch.randn(C, 4, generator=gen), torch.randn(N, 3, C, generator=gen), torch.randn(N, 3, C, generator=gen)
    want, bound = R.conv(xs[:R0], w, cache, lens, dy[:R0], dc)
    wide = torch.zeros(1, T, C + 3, dtype=DT[dtype], device="cuda")
    wide[:, :, 1:1 + C] = xs
    wide.requires_grad_(True)
    dwide = torch.zeros_like(wide.detach())
    dwide[:, :, 1:1 + C] = dy
    leaves = [wide, w.cuda().requires_grad_(True), cache.cuda().requires_grad_(True)]
    cu = None if cut is None else torch.tensor([0] + lens).cumsum(0).int()
    y, new = bg.causal_conv_silu(wide[:, :, 1:1 + C], *leaves[1:], cu_seqlens=cu)
    grads = torch.autograd.grad((y, new), leaves, (dwide[:, :, 1:1 + C], dc.cuda()))
    got = {"y": y.detach()[0, :R0], "cache": new.detach(), "dx": grads[0][0, :R0, 1:1 + C], "d_weight": grads[1], "d_cache": grads[2]}
    for k, v in got.items():
        R.check(v, want[k], bound[k], k)

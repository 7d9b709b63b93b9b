"""GPU: causal_conv_silu against its formula in float64, forward and every
gradient, dense and packed, at the elementwise bound of f32 arithmetic
(sequence_ref.conv) plus one rounding to the output's type."""
import pytest
import torch

import sequence_ref as R

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _inputs(rows, C, N, dtype, cache, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, C, generator=gen).mul(2).to(DT[dtype])
    w = torch.randn(C, 4, generator=gen)
    c = torch.randn(N, 3, C, generator=gen) if cache else None
    return x, w, c, torch.randn(rows, C, generator=gen).to(DT[dtype]), torch.randn(N, 3, C, generator=gen)


def _run(x, w, c, d, dc, shape, cu, train):
    import burn_gdn2 as bg

    C = x.shape[1]
    args = [x.reshape(*shape, C).cuda(), w.cuda(), None if c is None else c.cuda()]
    if not train:
        y, new = bg.causal_conv_silu(*args, cu_seqlens=cu)
        return {"y": y.reshape(-1, C), "cache": new}
    leaves = [t.requires_grad_(True) for t in args if t is not None]
    y, new = bg.causal_conv_silu(*args, cu_seqlens=cu)
    grads = torch.autograd.grad((y, new), leaves, (d.reshape(*shape, C).cuda(), dc.cuda()))
    got = {"y": y.detach().reshape(-1, C), "cache": new.detach(), "dx": grads[0].reshape(-1, C), "d_weight": grads[1]}
    return got if c is None else {**got, "d_cache": grads[2]}


def _check(got, want, bound):
    assert set(got) == set(want) or set(got) == {"y", "cache"}
    for k, v in got.items():
        R.check(v, want[k], bound[k], k)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cache", [False, True])
@pytest.mark.parametrize("B,T,C", [(1, 1, 1), (3, 1, 64), (2, 2, 66), (2, 3, 33), (4, 4, 64), (2, 15, 7), (2, 16, 64),
                                   (2, 17, 130), (1, 18, 64), (3, 19, 34), (2, 64, 64), (2, 257, 65), (1, 700, 40),
                                   (1, 40, 132), (2, 33, 260)])
def test_dense(dtype, cache, B, T, C):
    data = _inputs(B * T, C, B, dtype, cache, B * 1000 + T + C)
    want, bound = R.conv(*data[:3], [T] * B, *data[3:])
    _check(_run(*data, (B, T), None, True), want, bound)
    _check(_run(*data, (B, T), None, False), want, bound)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cache", [False, True])
@pytest.mark.parametrize("C", [33, 64])
@pytest.mark.parametrize("lens,behind", [([1], 0), ([0, 5, 0], 0), ([3, 0, 16, 1, 1, 64, 0], 9), ([130, 70, 333], 0),
                                         ([15, 1, 17, 2, 13, 3, 29, 4], 1), ([1] * 70, 3), ([2] * 40, 0), ([3] * 33, 2),
                                         ([0, 0], 4), ([16, 16, 32], 40)])
def test_packed(dtype, cache, C, lens, behind):
    rows = sum(lens) + behind
    x, w, c, d, dc = _inputs(rows, C, len(lens), dtype, cache, rows + C)
    clean = lambda t: torch.cat((t[:sum(lens)], torch.zeros(behind, C, dtype=t.dtype)))
    want, bound = R.conv(clean(x), w, c, lens, clean(d), dc)
    if behind:  # padding may hold anything
        x[-behind:], d[-behind:] = float("nan"), float("inf")
    cu = torch.tensor([0] + lens).cumsum(0).int()
    got = _run(x, w, c, d, dc, (1, rows), cu.cuda(), True)
    _check(got, want, bound)
    if behind:
        assert not got["y"][-behind:].any() and not got["dx"][-behind:].any()
    _check(_run(x, w, c, d, dc, (1, rows), cu, False), want, bound)


def test_equals_short_conv_1d():
    import burn_gdn2 as bg

    x, w, c, _, _ = (t.cuda() for t in _inputs(90, 24, 2, "f32", True, 1))
    x = x.reshape(2, 45, 24)
    for cache in (None, c):
        y, new = bg.causal_conv_silu(x, w, cache)
        y0, new0 = bg.short_conv_1d(x, w, cache)
        assert torch.equal(new, new0)
        assert torch.allclose(y, y0, rtol=1e-5, atol=1e-6)


def test_pieces_equal_a_whole_pass():
    """Through the cache in pieces of 1, 2, 3 and more tokens, forward and gradients, as one call."""
    import burn_gdn2 as bg

    B, T, C = 2, 40, 34
    x, w, c, d, dc = _inputs(B * T, C, B, "f32", True, 2)
    want, bound = R.conv(x, w, c, [T] * B, d, dc)
    leaves = [x.reshape(B, T, C).cuda().requires_grad_(True), w.cuda().requires_grad_(True), c.cuda().requires_grad_(True)]
    cache, ys, at = leaves[2], [], 0
    for n in (1, 2, 3, 1, 1, 17, 15):
        y, cache = bg.causal_conv_silu(leaves[0][:, at:at + n], leaves[1], cache)
        ys.append(y)
        at += n
    assert at == T
    grads = torch.autograd.grad((torch.cat(ys, 1), cache), leaves, (d.reshape(B, T, C).cuda(), dc.cuda()))
    got = {"y": torch.cat(ys, 1).detach().reshape(-1, C), "cache": cache.detach(), "dx": grads[0].reshape(-1, C),
           "d_weight": grads[1], "d_cache": grads[2]}
    # dx and dw come in up to seven parts, each of the bound: adding them rounds a few times more
    for k in ("dx", "d_weight", "d_cache"):
        bound[k] = bound[k] + 8 * R.EPS * want[k].abs() + bound[k]
    _check(got, want, bound)


def test_strided_inputs_and_partial_gradients():
    import burn_gdn2 as bg

    B, T, C = 2, 50, 40
    x, w, c, d, dc = _inputs(B * T, C, B, "bf16", True, 3)
    wide = torch.zeros(B, T, 2 * C + 1, dtype=torch.bfloat16, device="cuda")
    wide[..., 1:1 + C] = x.reshape(B, T, C).cuda()
    want, bound = R.conv(x, w, c, [T] * B, d, dc)
    y, new = bg.causal_conv_silu(wide[..., 1:1 + C], w.cuda(), c.cuda())
    _check({"y": y.reshape(-1, C), "cache": new}, want, bound)
    tb = x.reshape(B, T, C).transpose(0, 1).contiguous().cuda()
    y, new = bg.causal_conv_silu(tb.transpose(0, 1), w.cuda(), c.cuda())
    _check({"y": y.reshape(-1, C), "cache": new}, want, bound)
    for k, name in enumerate(("dx", "d_weight", "d_cache")):
        args = [x.reshape(B, T, C).cuda(), w.cuda(), c.cuda()]
        args[k].requires_grad_(True)
        twice = []
        for _ in range(2):
            y, new = bg.causal_conv_silu(*args)
            twice.append(torch.autograd.grad((y, new), args[k], (d.reshape(B, T, C).cuda(), dc.cuda()))[0])
        assert torch.equal(*twice)
        R.check(twice[0].reshape(want[name].shape), want[name], bound[name], name)
    # the new cache alone, and a plain sum (an expanded gradient)
    args = [t.requires_grad_(True) for t in (x.reshape(B, T, C).cuda(), w.cuda(), c.cuda())]
    y, new = bg.causal_conv_silu(*args)
    want, bound = R.conv(x, w, c, [T] * B, torch.zeros_like(d), dc)
    (g,) = torch.autograd.grad(new, args[0], dc.cuda(), retain_graph=True)
    R.check(g.reshape(-1, C), want["dx"], bound["dx"], "dx")
    want, bound = R.conv(x, w, c, [T] * B, torch.ones_like(d), None)
    (g,) = torch.autograd.grad(y.sum(), args[0])
    R.check(g.reshape(-1, C), want["dx"], bound["dx"], "dx")


def test_values_that_are_not_finite_stay_in_their_sequence():
    lens = [20, 30, 20]
    x, w, c, d, dc = _inputs(70, 33, 3, "f32", True, 4)
    want, bound = R.conv(x, w, c, lens, d, dc)
    x[20:50:4], d[22:50:5] = float("nan"), float("inf")
    c[1], dc[1] = float("inf"), float("nan")
    got = _run(x, w, c, d, dc, (1, 70), torch.tensor([0, 20, 50, 70], dtype=torch.int32), True)
    keep = torch.cat((torch.arange(20), torch.arange(50, 70)))
    for k in ("y", "dx"):
        R.check(got[k].cpu()[keep], want[k][keep], bound[k][keep], k)
    for k in ("cache", "d_cache"):
        R.check(got[k].cpu()[[0, 2]], want[k][[0, 2]], bound[k][[0, 2]], k)


def test_side_stream_and_graph():
    import burn_gdn2 as bg

    x, w, c, d, dc = _inputs(66, 32, 1, "f32", True, 5)
    lens = [10, 0, 56]
    c, dc = c.expand(3, 3, 32).contiguous(), dc.expand(3, 3, 32).contiguous()
    want, bound = R.conv(x, w, c, lens, d, dc)
    cu = torch.tensor([0, 10, 10, 66], dtype=torch.int32, device="cuda")
    static = [torch.zeros(t.shape, device="cuda", requires_grad=True) for t in (x[None], w, c)]
    grads = (d[None].cuda(), dc.cuda())

    def step(*args):
        y, new = bg.causal_conv_silu(*args, cu_seqlens=cu)
        return (y.detach(), new.detach()) + torch.autograd.grad((y, new), args, grads)

    graph = bg.GraphedCall(step, *static)
    with torch.no_grad():
        for s, t in zip(static, (x[None], w, c)):
            s.copy_(t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    got = dict(zip(("y", "cache", "dx", "d_weight", "d_cache"), out))
    got["y"], got["dx"] = got["y"][0], got["dx"][0]
    _check(got, want, bound)


def test_rows_beyond_32_bit_offsets():
    import burn_gdn2 as bg

    T, C, pitch = 3000, 32, 1 << 20
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GB of free device memory")
    big = torch.empty(T, pitch, dtype=torch.bfloat16, device="cuda")
    x, w, c, _, _ = _inputs(T, C, 1, "bf16", True, 6)
    big[:, 7:7 + C] = x.cuda()
    want, bound = R.conv(x, w, c, [T])
    y, new = bg.causal_conv_silu(big[None, :, 7:7 + C], w.cuda(), c.cuda())
    _check({"y": y.reshape(-1, C), "cache": new}, want, bound)


def test_refusals():
    import burn_gdn2 as bg

    x, w = torch.zeros(2, 5, 8, device="cuda"), torch.zeros(8, 4, device="cuda")
    for bad in ((x[0], w), (x, w[:, :3]), (x, w[:7]), (x, w, torch.zeros(1, 3, 8, device="cuda")), (x, w.cpu())):
        with pytest.raises(ValueError):
            bg.causal_conv_silu(*bad)
    for bad in ((x.half(), w), (x, w.bfloat16()), (x, w, torch.zeros(2, 3, 8, device="cuda").double())):
        with pytest.raises(TypeError):
            bg.causal_conv_silu(*bad)
    with pytest.raises(ValueError, match="one buffer"):
        bg.causal_conv_silu(x, w, cu_seqlens=torch.tensor([0, 5], dtype=torch.int32))
    y, new = bg.causal_conv_silu(x[:, :0], w)
    assert y.shape == (2, 0, 8) and not new.any()

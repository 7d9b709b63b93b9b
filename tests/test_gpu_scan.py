"""GPU: gated_scan against the token loop in float64, forward and adjoint, at
the elementwise bound of f32 arithmetic (sequence_ref.scan_one) plus one
rounding to the output's type."""
import pytest
import torch

import sequence_ref as R

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _decay(gen, *shape):
    """Log decays from the slowest (memory of a thousand tokens) to a reset a token."""
    return -torch.exp(torch.rand(*shape, generator=gen) * 9.0 - 7.0)


def _inputs(rows, C, N, x, g, state, seed):
    gen = _gen(seed)
    xs = torch.randn(rows, C, generator=gen).to(DT[x])
    gs = _decay(gen, rows, C).to(DT[g])
    st = torch.randn(N, C, generator=gen) if state else None
    return xs, gs, st, torch.randn(rows, C, generator=gen).to(DT[x]), torch.randn(N, C, generator=gen)


def _run(xs, gs, st, dh, ds, shape, cu, comp, train):
    import burn_gdn2 as bg

    C = xs.shape[1]
    x, g = xs.reshape(*shape, C).cuda(), gs.reshape(*shape, C).cuda()
    s = None if st is None else st.cuda()
    if not train:
        h, last = bg.gated_scan(x, g, s, cu_seqlens=cu, complement=comp)
        return {"h": h.reshape(-1, C), "state": last}
    leaves = [t.requires_grad_(True) for t in (x, g, s) if t is not None]
    h, last = bg.gated_scan(x, g, s, cu_seqlens=cu, complement=comp)
    grads = torch.autograd.grad((h, last), leaves, (dh.reshape(*shape, C).cuda(), ds.cuda()))
    got = {"h": h.detach().reshape(-1, C), "state": last.detach(), "dx": grads[0].reshape(-1, C), "dg": grads[1].reshape(-1, C)}
    if s is not None:
        got["d_state"] = grads[2]
    return got


def _check(got, want, bound):
    for k, v in got.items():
        assert v.dtype in (torch.float32, torch.bfloat16)
        R.check(v, want[k], bound[k], k)


TYPES = [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")]


@pytest.mark.parametrize("x,g", TYPES)
@pytest.mark.parametrize("B,T,C", [(1, 1, 1), (3, 1, 64), (2, 2, 66), (2, 15, 33), (2, 16, 64), (1, 17, 130), (3, 63, 7),
                                   (2, 64, 64), (1, 65, 96), (2, 257, 65), (1, 700, 40)])
@pytest.mark.parametrize("comp,state,train", [(False, True, True), (True, False, True), (True, True, False)])
def test_dense(x, g, B, T, C, comp, state, train):
    xs, gs, st, dh, ds = _inputs(B * T, C, B, x, g, state, B * 1000 + T + C)
    want, bound = R.scan(xs, gs, st, [T] * B, comp, dh if train else None, ds if train else None)
    _check(_run(xs, gs, st, dh, ds, (B, T), None, comp, train), want, bound)


@pytest.mark.parametrize("x,g", TYPES)
@pytest.mark.parametrize("lens,behind", [([1], 0), ([0, 5, 0], 0), ([3, 0, 16, 1, 1, 64, 0], 9), ([130, 70, 333], 0),
                                         ([16, 16, 32, 64, 128], 1), ([1] * 70, 3), ([0, 0], 4)])
@pytest.mark.parametrize("C,comp,state", [(33, True, True), (64, False, False), (64, False, True)])
def test_packed(x, g, lens, behind, C, comp, state):
    rows = sum(lens) + behind
    xs, gs, st, dh, ds = _inputs(rows, C, len(lens), x, g, state, rows + C)
    if behind:  # padding may hold anything
        xs[-behind:], gs[-behind:], dh[-behind:] = float("nan"), float("inf"), float("nan")
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).int()
    clean = lambda t: torch.cat((t[:sum(lens)], torch.zeros(behind, C, dtype=t.dtype)))
    want, bound = R.scan(clean(xs), clean(gs), st, lens, comp, clean(dh), ds)
    got = _run(xs, gs, st, dh, ds, (1, rows), cu.cuda(), comp, True)
    _check(got, want, bound)
    if behind:
        for k in ("h", "dx", "dg"):
            assert not got[k][-behind:].any(), k
    _check(_run(xs, gs, st, dh, ds, (1, rows), cu, comp, False), want, bound)


def test_few_long_chains_and_many_short():
    """The widest and the narrowest clusters: one chain set over 5000 tokens, 600 of them over 70."""
    for B, T, C in ((1, 5000, 12), (600, 70, 64)):
        xs, gs, st, dh, ds = _inputs(B * T, C, B, "f32", "f32", True, T)
        rows = [0, B // 2, B - 1]
        got = _run(xs, gs, st, dh, ds, (B, T), None, True, True)
        for b in rows:
            part = slice(b * T, (b + 1) * T)
            want, bound = R.scan(xs[part], gs[part], st[b:b + 1], [T], True, dh[part], ds[b:b + 1])
            seq = {k: (v[part] if v.shape[0] == B * T else v[b:b + 1]) for k, v in got.items()}
            _check(seq, want, bound)


def test_resets_growth_and_infinities():
    """g = -inf cuts off the past, g far below every f32 too, g > 0 grows; NaN in one sequence stays there."""
    gen = _gen(5)
    T, C = 100, 34
    xs, gs = torch.randn(T, C, generator=gen), _decay(gen, T, C)
    gs[10], gs[20], gs[30:33], gs[40] = -float("inf"), -1e30, 0.7, -100.0
    gs[50] = 0.0
    dh, ds, st = torch.randn(T, C, generator=gen), torch.randn(1, C, generator=gen), torch.randn(1, C, generator=gen)
    for comp in (False, True):
        want, bound = R.scan(xs, gs, st, [T], comp, dh, ds)
        _check(_run(xs, gs, st, dh, ds, (1, T), None, comp, True), want, bound)
    # a sequence whose values are not finite does not reach its neighbours, in either direction
    lens = [30, 40, 30]
    st, ds = torch.randn(3, C, generator=gen), torch.randn(3, C, generator=gen)
    want, bound = R.scan(xs, gs, st, lens, True, dh, ds)
    bad = [t.clone() for t in (xs, gs, dh, st, ds)]
    bad[0][30:70:3] = float("inf")
    bad[1][31:70:5] = float("nan")
    bad[2][35:70:7] = float("nan")
    bad[3][1] = float("nan")
    bad[4][1] = float("inf")
    got = _run(bad[0], bad[1], bad[3], bad[2], bad[4], (1, T), torch.tensor([0, 30, 70, 100], dtype=torch.int32), True, True)
    keep = torch.cat((torch.arange(30), torch.arange(70, 100)))
    for k, v in got.items():
        at = keep if v.shape[0] == T else torch.tensor([0, 2])
        R.check(v.cpu()[at], want[k][at], bound[k][at], k)


@pytest.mark.parametrize("rate,T,C", [(20.0, 90, 34), (90.0, 90, 34), (6.0, 40, 64), (0.4, 5000, 12), (3.0, 700, 600)])
@pytest.mark.parametrize("lens", [None, "packed"])
def test_growth_of_nothing(rate, T, C, lens):
    """A decay above one over tokens whose state (adjoint) is zero: its product over a run, a tile or a segment
    leaves f32's range, and zero times that stays zero."""
    gen = _gen(int(rate))
    xs, gs = torch.randn(T, C, generator=gen), _decay(gen, T, C)
    dh, ds = torch.randn(T, C, generator=gen), torch.zeros(1, C)
    late = T - 5
    gs[3:late, ::2] = rate   # every other channel, which neither x nor the gradient of h touches meanwhile
    xs[:late, ::2], dh[4:, ::2] = 0.0, 0.0
    cu = None if lens is None else torch.tensor([0, T, T], dtype=torch.int32)
    st, ds = (None, ds) if lens is None else (torch.zeros(2, C), torch.cat((ds, ds)))
    def both_ways(lengths, comp):
        want, bound = R.scan(xs, gs, st, lengths, comp, dh, ds)
        got = _run(xs, gs, st, dh, ds, (1, T), cu, comp, True)
        if rate > 88.8:  # e^90 dh[3] > 2^128 for dh[3] > 0.28: no f32 adjoint before token 3, and none in its dg (or 1 - e^90 times it)
            for k, rows in (("dx", 4 if comp else 3), ("dg", 4), ("d_state", 1)):
                if k in got:
                    got[k], want[k] = got[k].clone(), want[k].clone()
                    got[k][:rows, ::2] = want[k][:rows, ::2] = 0.0
        _check(got, want, bound)

    both_ways([T] if lens is None else [T, 0], False)
    if lens is None and T == 90:  # a leaky average of nothing, and token by token
        both_ways([T], True)
        want, bound = R.scan(xs, gs, None, [1] * T, True)
        _check(_run(xs, gs, torch.zeros(T, C), None, None, (T, 1), None, True, False), want, bound)


def test_strided_and_broadcast_inputs():
    """Column slices, a batch-transposed buffer, an odd offset, gradients of broadcast inputs."""
    import burn_gdn2 as bg

    B, T, C = 2, 70, 48
    gen = _gen(6)
    wide = torch.randn(B, T, 3 * C + 1, generator=gen).cuda()
    tb = torch.randn(T, B, C, generator=gen).cuda()
    x, g = wide[:, :, C + 1:2 * C + 1], -tb.transpose(0, 1).abs()
    want, bound = R.scan(x.cpu().reshape(-1, C), g.cpu().reshape(-1, C), None, [T] * B, False)
    h, last = bg.gated_scan(x, g)
    _check({"h": h.reshape(-1, C), "state": last}, want, bound)
    # one decay for all tokens and channels, one x for the batch
    rate = torch.tensor([-0.1], device="cuda", requires_grad=True)
    x1 = torch.randn(1, T, C, generator=gen).cuda().requires_grad_(True)
    h, last = bg.gated_scan(x1.expand(B, T, C), rate.expand(B, T, C))
    (h.sum() + last.sum()).backward()
    xc, gc = x1.detach().cpu().expand(B, T, C).reshape(-1, C), rate.detach().cpu().expand(B * T, C)
    want, bound = R.scan(xc, gc, None, [T] * B, False, torch.ones(B * T, C), torch.ones(B, C))
    # sums of B (x) and B T C (rate) gradients in torch: their own roundings come on top, n EPS of the sizes at most
    R.check(x1.grad.reshape(T, C), want["dx"].reshape(B, T, C).sum(0),
            bound["dx"].reshape(B, T, C).sum(0) + 2 * B * R.EPS * want["dx"].reshape(B, T, C).abs().sum(0), "dx")
    n = B * T * C
    R.check(rate.grad, want["dg"].sum().reshape(1), (bound["dg"].sum() + n * R.EPS * want["dg"].abs().sum()).reshape(1), "dg")


def test_gradient_against_differences():
    """Central differences of the kernel's own forward.  f is linear in x and state, so their differences are exact
    but for rounding; in g the cubic term is below step^2 of the third derivative."""
    import burn_gdn2 as bg

    T, C = 40, 6
    gen = _gen(7)
    x, st = torch.randn(1, T, C, generator=gen).cuda(), torch.randn(1, C, generator=gen).cuda()
    g = (-torch.rand(1, T, C, generator=gen)).cuda()
    r, rs = torch.randn(1, T, C, generator=gen).cuda().double(), torch.randn(1, C, generator=gen).cuda().double()

    def f(x, g, st):
        h, last = bg.gated_scan(x, g, st, complement=True)
        return float((h.double() * r).sum() + (last.double() * rs).sum())

    leaves = [t.clone().requires_grad_(True) for t in (x, g, st)]
    h, last = bg.gated_scan(*leaves, complement=True)
    grads = torch.autograd.grad((h, last), leaves, (r.float(), rs.float()))
    step = 2.0 ** -6
    for k, t in enumerate((x, g, st)):
        way = torch.randn(t.shape, generator=gen).cuda()
        args = lambda s: [v + s * way if i == k else v for i, v in enumerate((x, g, st))]
        diff = (f(*args(step)) - f(*args(-step))) / (2 * step)
        dot = float((grads[k].double() * way.double()).sum())
        # rounding: some 300 values of size 1 to 3, each off by at most 1e-5 (the bound above), over 2 steps; the
        # cubic term: step^2 / 6 of a third derivative of at most some hundred
        assert abs(diff - dot) <= 0.02 + 0.01 * abs(dot), (k, diff, dot)


def test_steps_equal_a_whole_pass_and_inplace():
    """Token by token through the decode step, with the state in place, as one call over the tokens."""
    import burn_gdn2 as bg

    B, T, C = 3, 20, 70
    xs, gs, st, _, _ = _inputs(B * T, C, B, "f32", "f32", True, 8)
    x, g, s = xs.reshape(B, T, C).cuda(), gs.reshape(B, T, C).cuda(), st.cuda()
    want, bound = R.scan(xs, gs, st, [T] * B, True)
    state = s.clone()
    outs = []
    for t in range(T):
        h, back = bg.gated_scan(x[:, t:t + 1], g[:, t:t + 1], state, complement=True, inplace=True)
        assert back is state
        outs.append(h)
    _check({"h": torch.cat(outs, 1).reshape(-1, C), "state": state}, want, bound)
    # in two pieces, the second from the first's state, in place over a longer span
    h1, mid = bg.gated_scan(x[:, :7], g[:, :7], s, complement=True)
    h2, end = bg.gated_scan(x[:, 7:], g[:, 7:], mid, complement=True, inplace=True)
    assert end is mid
    _check({"h": torch.cat((h1, h2), 1).reshape(-1, C), "state": end}, want, bound)
    # packed, in place, an empty sequence keeps its state
    cu = torch.tensor([0, 0, 30, 60], dtype=torch.int32)
    s3 = s.clone()
    want, bound = R.scan(xs, gs, st, [0, 30, 30], True)
    h, back = bg.gated_scan(x.reshape(1, -1, C), g.reshape(1, -1, C), s3, cu_seqlens=cu, complement=True, inplace=True)
    _check({"h": h.reshape(-1, C), "state": s3}, want, bound)


def test_partial_gradients_and_repeatability():
    """Only some inputs or outputs take part; the same call twice gives the same bits."""
    import burn_gdn2 as bg

    B, T, C = 2, 150, 36
    xs, gs, st, dh, ds = _inputs(B * T, C, B, "bf16", "f32", True, 9)
    x, g, s = xs.reshape(B, T, C).cuda(), gs.reshape(B, T, C).cuda(), st.cuda()
    xg = x.clone().requires_grad_(True)
    h, last = bg.gated_scan(xg, g, s)
    assert h.requires_grad and last.requires_grad
    (a,) = torch.autograd.grad(last, xg, ds.cuda(), retain_graph=True)
    (b,) = torch.autograd.grad(h, xg, dh.reshape(B, T, C).cuda(), retain_graph=True)
    want, bound = R.scan(xs, gs, st, [T] * B, False, torch.zeros(B * T, C), ds)
    _check({"dx": a.reshape(-1, C)}, want, bound)
    want, bound = R.scan(xs, gs, st, [T] * B, False, dh, None)
    _check({"dx": b.reshape(-1, C)}, want, bound)
    h2, last2 = bg.gated_scan(xg, g, s)
    (b2,) = torch.autograd.grad(h2, xg, dh.reshape(B, T, C).cuda())
    assert torch.equal(h, h2) and torch.equal(last, last2) and torch.equal(b, b2)
    with torch.no_grad():
        h3, last3 = bg.gated_scan(xg, g, s)
    assert torch.equal(h, h3) and torch.equal(last, last3) and not h3.requires_grad


def test_side_stream_and_graph():
    """On another stream than the inputs', and captured and replayed on new values."""
    import burn_gdn2 as bg

    B, T, C = 2, 90, 64
    xs, gs, st, dh, ds = _inputs(B * T, C, B, "f32", "f32", True, 10)
    x, g, s = xs.reshape(B, T, C).cuda(), gs.reshape(B, T, C).cuda(), st.cuda()
    want, bound = R.scan(xs, gs, st, [T] * B, True, dh, ds)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h, last = bg.gated_scan(x, g, s, complement=True)
    torch.cuda.current_stream().wait_stream(side)
    _check({"h": h.reshape(-1, C), "state": last}, want, bound)

    static = [torch.zeros_like(t).requires_grad_(True) for t in (x, g, s)]
    d = [dh.reshape(B, T, C).cuda(), ds.cuda()]

    def step(*args):
        h, last = bg.gated_scan(*args, complement=True)
        return (h.detach(), last.detach()) + torch.autograd.grad((h, last), args, d)

    graph = bg.GraphedCall(step, *static)
    with torch.no_grad():
        for a, b in zip(static, (x, g, s)):
            a.copy_(b)
    for _ in range(2):
        out = graph.replay()
        got = dict(zip(("h", "state", "dx", "dg", "d_state"), out))
        _check({k: v.reshape(-1, C) for k, v in got.items()}, want, bound)


def test_exponential_over_its_range():
    """One token from state 1 with x = 0 gives e^g: within a step of it over the whole range, and 1 - e^g with x = 1
    from state 0 within a step and a half for small g, where 1 - e^g cancels."""
    import burn_gdn2 as bg

    g = torch.cat((-torch.logspace(-30, 1.9, 20000), torch.logspace(-30, 1.9, 20000), torch.linspace(-1, 1, 40001))).float()
    g = g.reshape(1, 1, -1).cuda().expand(1, 2, -1)  # two tokens: the scan's own exponential, not the step's
    zero, one = torch.zeros_like(g), torch.ones_like(g)
    h, _ = bg.gated_scan(zero, g, one[:, 0], complement=False)
    want = g[0, 0].double().exp()
    assert ((h[0, 0].double() - want).abs() <= 2.0 ** -23 * want).all()
    h, _ = bg.gated_scan(one, g, None, complement=True)
    want = -torch.expm1(g[0, 0].double())
    small = g[0, 0].abs() < 0.3
    assert ((h[0, 0].double() - want).abs() <= 1.5 * 2.0 ** -23 * want.abs())[small].all()
    assert ((h[0, 0].double() - want).abs() <= 2.0 ** -23 * (1 + want.abs()) * 1.5).all()


def test_rows_beyond_32_bit_offsets():
    """A buffer of more than 2^31 elements, strided so that the last rows lie beyond 32-bit offsets."""
    import burn_gdn2 as bg

    T, C, pitch = 3000, 32, 1 << 20
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GB of free device memory")
    big = torch.empty(T, pitch, dtype=torch.bfloat16, device="cuda")  # 6.3 GB, 3.1e9 elements
    gen = _gen(11)
    xs = torch.randn(T, C, generator=gen).bfloat16()
    gs = _decay(gen, T, C).bfloat16()
    big[:, 5:5 + C], big[:, 64:64 + C] = xs.cuda(), gs.cuda()
    want, bound = R.scan(xs, gs, None, [T], False)
    h, last = bg.gated_scan(big[None, :, 5:5 + C], big[None, :, 64:64 + C])
    _check({"h": h.reshape(-1, C), "state": last}, want, bound)

"""GPU: group_norm_gate against its formula in float64, forward and every
gradient, at the elementwise bound of f32 arithmetic (sequence_ref.group_norm)
plus one rounding to the output's type."""
import pytest
import torch

import sequence_ref as R

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _inputs(rows, groups, width, dtype, gate, affine, bias, seed):
    gen = torch.Generator().manual_seed(seed)
    C = groups * width
    x = (torch.randn(rows, C, generator=gen) * 1.5 + 0.5).to(DT[dtype])
    gt = torch.randn(rows, C, generator=gen).mul(2).to(DT[dtype]) if gate else None
    n = {"channel": C, "group": width, "none": 0}[affine]
    w = torch.randn(n, generator=gen) if n else None
    b = torch.randn(n, generator=gen) if n and bias else None
    return x, gt, w, b, torch.randn(rows, C, generator=gen).to(DT[dtype])


def _run(x, gt, w, b, d, groups, eps, center, train, shape=None):
    import burn_gdn2 as bg

    dev = lambda t: None if t is None else t.cuda()
    args = [dev(t) for t in (x, gt, w, b)]
    if shape is not None:
        args[:2] = [None if t is None else t.reshape(shape) for t in args[:2]]
    kw = dict(num_groups=groups, eps=eps, center=center)
    if not train:
        return {"y": bg.group_norm_gate(*args, **kw).reshape(x.shape)}
    leaves = [t.requires_grad_(True) for t in args if t is not None]
    y = bg.group_norm_gate(*args, **kw)
    assert y.shape == args[0].shape
    grads = list(torch.autograd.grad(y, leaves, dev(d).reshape(y.shape)))
    names = [n for n, t in zip(("dx", "d_gate", "d_weight", "d_bias"), args) if t is not None]
    return {"y": y.detach().reshape(x.shape), **{n: g.reshape(x.shape) if n in ("dx", "d_gate") else g for n, g in zip(names, grads)}}


def _check(got, want, bound):
    for k, v in got.items():
        R.check(v, want[k], bound[k], k)


SIZES = [(1, 1, 1), (5, 3, 1), (7, 2, 2), (3, 16, 128), (33, 7, 90), (9, 5, 33), (4, 1, 127), (70, 4, 16), (2, 3, 257),
         (6, 2, 520), (5, 1, 1021), (3, 2, 2048), (2, 1, 4096), (300, 1, 8), (2, 400, 4), (1000, 2, 64)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,groups,width", SIZES)
@pytest.mark.parametrize("gate,affine,bias,center", [(True, "channel", True, True), (False, "group", False, False),
                                                     (True, "none", False, False), (False, "channel", True, True)])
def test_sizes(dtype, rows, groups, width, gate, affine, bias, center):
    data = _inputs(rows, groups, width, dtype, gate, affine, bias, rows + width)
    want, bound = R.group_norm(*data[:4], groups, 1e-5, center, data[4])
    _check(_run(*data, groups, 1e-5, center, True), want, bound)
    _check(_run(*data, groups, 1e-5, center, False), want, bound)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,groups,width", [(3, 1, 1025), (2, 2, 1501), (5, 1, 4104), (700, 1, 4100), (3, 3, 8192), (1, 1, 10240), (3, 1, 30000)])
@pytest.mark.parametrize("gate,affine,bias,center", [(True, "channel", True, True), (False, "group", True, False),
                                                     (True, "group", False, True), (False, "none", False, True)])
def test_wide_groups(dtype, rows, groups, width, gate, affine, bias, center):
    """Groups that a block does not hold at once: the sums of weights' gradients in shared memory or, for the
    widest, not; at most 20 additions a thread, then trees."""
    test_sizes(dtype, rows, groups, width, gate, affine, bias, center)


def test_equals_rms_norm_gate_per_head():
    """The uncentered, gated norm with one weight for all heads is the layer's rms_norm_gate_per_head."""
    import burn_gdn2 as bg

    B, T, HV, V = 2, 9, 4, 64
    x, gt, w, _, _ = _inputs(B * T, HV, V, "f32", True, "group", False, 3)
    a = bg.group_norm_gate(x.cuda().reshape(B, T, HV * V), gt.cuda().reshape(B, T, HV * V), w.cuda(), num_groups=HV,
                           center=False)
    b = bg.rms_norm_gate_per_head(x.cuda().reshape(B, T, HV, V), gt.cuda().reshape(B, T, HV, V), w.cuda(), 1e-5)
    # both are within the bound of the formula
    _, bound = R.group_norm(x, gt, w, None, HV, 1e-5, False)
    assert ((a.reshape(-1, HV * V) - b.reshape(-1, HV * V)).abs().double().cpu() <= 2 * bound["y"] + 1e-38).all()


def test_strided_inputs_and_leading_dims():
    import burn_gdn2 as bg

    B, T, G, D = 2, 5, 3, 20
    x, gt, w, b, d = _inputs(B * T, G, D, "f32", True, "channel", True, 4)
    wide = torch.zeros(B, T, 2 * G * D + 2).cuda()
    wide[..., 1:1 + G * D], wide[..., 1 + G * D:1 + 2 * G * D] = x.reshape(B, T, -1).cuda(), gt.reshape(B, T, -1).cuda()
    xs, gs = wide[..., 1:1 + G * D], wide[..., 1 + G * D:1 + 2 * G * D]  # 4-byte aligned rows
    want, bound = R.group_norm(x, gt, w, b, G, 1e-3, True, d)
    y = bg.group_norm_gate(xs, gs, w.cuda(), b.cuda(), num_groups=G, eps=1e-3)
    R.check(y.reshape(B * T, -1), want["y"], bound["y"], "y")
    # transposed storage: copied, gradients find their way back
    xt = x.reshape(B, T, -1).transpose(0, 1).contiguous().cuda().requires_grad_(True)
    y = bg.group_norm_gate(xt.transpose(0, 1), gs, w.cuda(), b.cuda(), num_groups=G, eps=1e-3)
    (g,) = torch.autograd.grad(y, xt, d.reshape(B, T, -1).cuda())
    R.check(g.transpose(0, 1).reshape(B * T, -1), want["dx"], bound["dx"], "dx")
    # an expanded gradient (a plain sum), and a broadcast gate
    xl = x.cuda().requires_grad_(True)
    g1 = gt[:1].cuda().requires_grad_(True)
    y = bg.group_norm_gate(xl, g1.expand(B * T, -1), w.cuda(), b.cuda(), num_groups=G, eps=1e-3)
    gx, gg = torch.autograd.grad(y.sum(), (xl, g1))
    want, bound = R.group_norm(x, gt[:1].expand(B * T, -1), w, b, G, 1e-3, True, torch.ones_like(x))
    R.check(gx, want["dx"], bound["dx"], "dx")
    R.check(gg, want["d_gate"].sum(0, keepdim=True),
            bound["d_gate"].sum(0, keepdim=True) + B * T * R.EPS * want["d_gate"].abs().sum(0, keepdim=True), "d_gate")


def test_partial_gradients_empty_rows_and_repeatability():
    import burn_gdn2 as bg

    x, gt, w, b, d = _inputs(40, 4, 32, "bf16", True, "group", True, 5)
    want, bound = R.group_norm(x, gt, w, b, 4, 1e-5, True, d)
    names = ("dx", "d_gate", "d_weight", "d_bias")
    for k, name in enumerate(names):
        args = [t.cuda() for t in (x, gt, w, b)]
        args[k].requires_grad_(True)
        twice = []
        for _ in range(2):
            y = bg.group_norm_gate(*args, num_groups=4)
            twice.append(torch.autograd.grad(y, args[k], d.cuda())[0])
        assert torch.equal(*twice)
        R.check(twice[0], want[name], bound[name], name)
    args = [t.cuda().requires_grad_(True) for t in (x[:0], gt[:0], w, b)]
    y = bg.group_norm_gate(*args, num_groups=4)
    assert y.shape == (0, 128)
    grads = torch.autograd.grad(y, args, y.detach())
    assert not grads[2].any() and not grads[3].any()


def test_constant_rows_and_values_that_are_not_finite():
    """A group without variance gives z = bias; an infinity or NaN stays in its row's group."""
    import burn_gdn2 as bg

    x, gt, w, b, _ = _inputs(6, 3, 16, "f32", True, "channel", True, 6)
    x[1] = 2.0
    x[2, 3], x[3, 20], gt[4, 40] = float("inf"), float("nan"), -float("inf")
    want, bound = R.group_norm(x, gt, w, b, 3, 1e-5, True)
    y = bg.group_norm_gate(*(t.cuda() for t in (x, gt, w, b)), num_groups=3).cpu()
    fine = torch.ones(6, 48, dtype=torch.bool)
    fine[2, :16] = fine[3, 16:32] = False
    fine[4, 40] = False
    R.check(y[fine], want["y"][fine], bound["y"][fine], "y")
    assert not torch.isfinite(y[2, :16]).any() and torch.isnan(y[3, 16:32]).all()


def test_side_stream_and_graph():
    import burn_gdn2 as bg

    x, gt, w, b, d = (t.cuda() for t in _inputs(70, 4, 32, "f32", True, "channel", True, 7))
    want, bound = R.group_norm(*(t.cpu() for t in (x, gt, w, b)), 4, 1e-5, True, d.cpu())
    static = [torch.zeros_like(t).requires_grad_(True) for t in (x, gt, w, b)]

    def step(*args):
        y = bg.group_norm_gate(*args, num_groups=4)
        return (y.detach(),) + torch.autograd.grad(y, args, d)

    graph = bg.GraphedCall(step, *static)
    with torch.no_grad():
        for s, t in zip(static, (x, gt, w, b)):
            s.copy_(t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    _check(dict(zip(("y", "dx", "d_gate", "d_weight", "d_bias"), out)), want, bound)


def test_many_rows_beyond_32_bit_offsets():
    """More than 2^31 elements in x."""
    import burn_gdn2 as bg

    rows, C = (1 << 31) // 4096 + 3, 4096
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of free device memory")
    x = torch.zeros(rows, C, dtype=torch.bfloat16, device="cuda")
    tail, gt, w, b, _ = _inputs(3, 32, 128, "bf16", False, "channel", True, 8)
    x[-3:] = tail.cuda()
    y = bg.group_norm_gate(x, None, w.cuda(), b.cuda(), num_groups=32)
    want, bound = R.group_norm(tail, None, w, b, 32, 1e-5, True)
    R.check(y[-3:], want["y"], bound["y"], "y")


def test_refusals():
    import burn_gdn2 as bg

    x = torch.zeros(2, 12, device="cuda")
    w = torch.ones(12, device="cuda")
    call = lambda *a, **k: bg.group_norm_gate(*a, **{"num_groups": 3, **k})
    for bad in (dict(num_groups=5), dict(num_groups=0), dict(eps=0.0), dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            call(x, **bad)
    with pytest.raises(ValueError):
        call(x, x[:1])
    with pytest.raises(ValueError):
        call(x, x.bfloat16())
    with pytest.raises(ValueError):
        call(x, None, w[:5])
    with pytest.raises(ValueError):
        call(x, None, None, w)
    with pytest.raises(ValueError):
        call(x, None, w, w[:4])
    with pytest.raises(TypeError):
        call(x, None, w.bfloat16())
    with pytest.raises(TypeError):
        call(x.half())
    with pytest.raises(ValueError):
        call(x, None, w.cpu())
    with pytest.raises(bg.Gdn2Error, match="EUNSUPPORTED"):  # 2^31 channels, all the same stored one
        call(torch.zeros(1, device="cuda").as_strided((1, 1 << 31), (0, 0)), num_groups=1)

"""GPU: the sequence operators at the edges of what they take: nothing at all,
second derivatives, inference mode, two calls at once, in-place writes that
autograd has to know of, graphs that share nothing."""
import pytest
import torch

import sequence_ref as R

pytestmark = pytest.mark.gpu


def _calls(dtype=torch.float32, T=40, grad=True):
    """Each operator on fresh inputs: (name, call, leaves)."""
    import burn_gdn2 as bg

    gen = torch.Generator("cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, g, st = r(2, T, 24).to(dtype), -r(2, T, 24).abs(), r(2, 24)
    w, c = r(24, 4), r(2, 3, 24)
    xn, wn = r(2 * T, 24).to(dtype), r(24)
    leaves = ((x, g, st), (x.clone(), w, c), (xn, wn))
    if grad:
        for ls in leaves:
            for t in ls:
                t.requires_grad_(True)
    return [("scan", lambda: bg.gated_scan(*leaves[0])[0], leaves[0]),
            ("conv", lambda: bg.causal_conv_silu(*leaves[1])[0], leaves[1]),
            ("norm", lambda: bg.group_norm_gate(xn, None, wn, num_groups=4), leaves[2])]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nothing_to_do(dtype):
    import burn_gdn2 as bg

    z = lambda *s: torch.zeros(*s, dtype=dtype, device="cuda")
    f = lambda *s: torch.ones(*s, device="cuda")
    for B, T, C in ((2, 0, 8), (0, 5, 8), (2, 5, 0)):
        h, last = bg.gated_scan(z(B, T, C), z(B, T, C), f(B, C))
        assert h.shape == (B, T, C) and h.dtype == dtype and torch.equal(last, f(B, C))
        y, cache = bg.causal_conv_silu(z(B, T, C), f(C, 4), f(B, 3, C))
        assert y.shape == (B, T, C) and y.dtype == dtype and torch.equal(cache, f(B, 3, C))
    # a packed buffer without a row: every sequence is empty
    cu = torch.zeros(4, dtype=torch.int32)
    x, g, st = z(1, 0, 8).requires_grad_(True), z(1, 0, 8).requires_grad_(True), f(3, 8).requires_grad_(True)
    h, last = bg.gated_scan(x, g, st, cu_seqlens=cu)
    assert h.shape == (1, 0, 8) and torch.equal(last, st)
    grads = torch.autograd.grad((h, last), (x, g, st), (h.detach(), 2 * f(3, 8)))
    assert torch.equal(grads[2], 2 * f(3, 8))
    w, c = f(8, 4).requires_grad_(True), f(3, 3, 8).requires_grad_(True)
    y, cache = bg.causal_conv_silu(x, w, c, cu_seqlens=cu)
    grads = torch.autograd.grad((y, cache), (x, w, c), (y.detach(), 3 * f(3, 3, 8)))
    assert torch.equal(cache, c) and not grads[1].any() and torch.equal(grads[2], 3 * f(3, 3, 8))
    _, cache = bg.causal_conv_silu(x, w, None, cu_seqlens=cu)
    assert not cache.any()


def test_second_derivatives_are_refused():
    for name, call, leaves in _calls():
        (g,) = torch.autograd.grad(call().sum(), leaves[0], create_graph=True)
        with pytest.raises(RuntimeError):  # nothing to differentiate: the gradient has no graph
            torch.autograd.grad(g.sum(), leaves[0])
        (g,) = torch.autograd.grad(call().square().sum(), leaves[0], create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_the_layer_with_another_core_is_as_often_differentiable():
    import burn_gdn2 as bg
    from burn_gdn2 import training

    def core(q, k, v, g, b, w, scale, chunk):  # any torch core: all its inputs in a product
        return g.exp() * scale * (q + b * k) * v * w, None

    cfg = bg.Gdn2Config(mode=bg.Gdn2Mode.Chunk, chunk_size=64, hidden_size=64, num_heads=1, head_dim=32)
    m = bg.GatedDeltaNet2.new(cfg, device="cuda", dtype=torch.float32, seed=2)
    x = torch.randn(1, 6, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).requires_grad_(True)
    y = training.layer_forward(m.parameters(), cfg, x, core=core)
    (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    (gg,) = torch.autograd.grad(g.square().sum(), x)
    assert torch.isfinite(gg).all() and gg.any()


def test_inference_mode_and_in_place_versions():
    import burn_gdn2 as bg

    want = [call().detach() for _, call, _ in _calls(grad=False)]
    with torch.inference_mode():
        for (_, call, _), w in zip(_calls(grad=False), want):
            assert torch.equal(call(), w)
        s = torch.ones(2, 8, device="cuda")
        bg.gated_scan(torch.zeros(2, 1, 8, device="cuda"), torch.zeros(2, 1, 8, device="cuda"), s, inplace=True)
        bg.reorder_states(s, [1, 0])
    # a tensor that autograd has saved and a kernel then overwrites
    s = torch.ones(2, 8, device="cuda")
    leaf = torch.ones(2, 8, device="cuda", requires_grad=True)
    for write in (lambda: bg.reorder_states(s, [1, 0]),
                  lambda: bg.gated_scan(torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 3, 8, device="cuda"), s, inplace=True)):
        y = (leaf * s).sum()
        write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


@pytest.mark.parametrize("T", [40, 3000])
def test_two_calls_at_once(T):
    """The same operators on two streams at the same time, each on its own inputs: as one after the other."""
    jobs = [_calls(T=T), _calls(torch.bfloat16, T=T)]

    def run(calls):
        out = []
        for _, call, leaves in calls:
            y = call()
            out += [y.detach()] + list(torch.autograd.grad(y, leaves, torch.ones_like(y), allow_unused=True))
        return [t for t in out if t is not None]

    want = [run(c) for c in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[] for _ in jobs]
    for _ in range(3):
        for k, (s, c) in enumerate(zip(streams, jobs)):
            with torch.cuda.stream(s):
                got[k].append(run(c))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for again in g:
            assert len(again) == len(w) and all(torch.equal(a, b) for a, b in zip(again, w))


def test_two_graphs_of_the_same_leaves():
    """Forward and backward captured twice from the same inputs (each with its own workspaces), replayed in turn."""
    import burn_gdn2 as bg

    gen = torch.Generator("cuda").manual_seed(3)
    leaves = [torch.randn(1, 3000, 24, generator=gen, device="cuda").requires_grad_(True),
              (-torch.rand(1, 3000, 24, generator=gen, device="cuda")).requires_grad_(True)]

    def step(x, g):
        h, last = bg.gated_scan(x, g)
        return (h.detach(), last.detach()) + torch.autograd.grad((h, last), (x, g), (torch.ones_like(h), torch.ones_like(last)))

    want = step(*leaves)
    graphs = [bg.GraphedCall(step, *leaves) for _ in range(2)]
    for _ in range(2):
        for graph in graphs:
            assert all(torch.equal(a, b) for a, b in zip(graph.replay(), want))


def test_checked_against_the_formula_after_all_that():
    xs = torch.randn(50, 20, generator=torch.Generator().manual_seed(9))
    gs = -torch.rand(50, 20, generator=torch.Generator().manual_seed(10))
    import burn_gdn2 as bg

    h, last = bg.gated_scan(xs[None].cuda(), gs[None].cuda())
    want, bound = R.scan(xs, gs, None, [50], False)
    R.check(h[0], want["h"], bound["h"], "h")
    R.check(last, want["state"], bound["state"], "state")
    assert bg._lib.read_device_errors() == 0

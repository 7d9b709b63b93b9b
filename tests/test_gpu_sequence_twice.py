"""GPU: second derivatives.  An operator's gradient says that it has no further one wherever it is differentiated
again, also where the gradient that came in was a constant."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _calls():
    import burn_gdn2 as bg

    gen = torch.Generator("cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda").requires_grad_(True)
    x, g, st, w, c, gate, n, b = r(2, 40, 24), r(2, 40, 24), r(2, 24), r(24, 4), r(2, 3, 24), r(2, 40, 24), r(24), r(24)
    rows, turned = r(80, 24), r(2, 24, 40)
    return {"scan": (lambda: bg.gated_scan(x, -g.abs(), st)[0], (x, g, st)),
            "conv": (lambda: bg.causal_conv_silu(x, w, c)[0], (x, w, c)),
            "norm": (lambda: bg.group_norm_gate(x, gate, n, b, num_groups=4), (x, gate, n, b)),
            "norm of rows": (lambda: bg.group_norm_gate(rows, None, n, num_groups=4), (rows, n)),
            "norm of turned": (lambda: bg.group_norm_gate(turned.transpose(1, 2), None, n, num_groups=4), (turned, n))}


@pytest.mark.parametrize("name", ["scan", "conv", "norm", "norm of rows", "norm of turned"])
def test_a_penalty_on_a_gradient_is_not_dropped(name):
    call, leaves = _calls()[name]
    for k, leaf in enumerate(leaves):
        loss = call().sum()
        (g,) = torch.autograd.grad(loss, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (loss + g.square().sum()).backward()
        if k:  # where only this leaf wants a gradient
            for t in leaves:
                t.requires_grad_(t is leaf)
            (g,) = torch.autograd.grad(call().sum(), leaf, create_graph=True)
            with pytest.raises(RuntimeError, match="once_differentiable"):
                g.sum().backward()
            for t in leaves:
                t.requires_grad_(True)
    # once is what they are: the same values with a graph as without
    want = torch.autograd.grad(call().sum(), leaves)
    got = torch.autograd.grad(call().sum(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

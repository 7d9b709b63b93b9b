"""GPU: the sequence operators have no forward-mode derivative and say so, whichever input carries the tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def _operators():
    import burn_gdn2 as bg

    gen = torch.Generator("cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, g, st = r(2, 40, 24), -r(2, 40, 24).abs(), r(2, 24)
    one, g1 = r(2, 1, 24), -r(2, 1, 24).abs()
    w, c, gate, n, b = r(24, 4), r(2, 3, 24), r(2, 40, 24), r(24), r(24)
    norm = lambda x, gate, n, b: bg.group_norm_gate(x, gate, n, b, num_groups=4)
    return {"scan": (lambda *a: bg.gated_scan(*a)[0], (x, g, st)),
            "scan step": (lambda *a: bg.gated_scan(*a)[0], (one, g1, st)),
            "scan in place": (lambda x, g, s: bg.gated_scan(x, g, s, inplace=True)[0], (one, g1, st)),
            "conv": (lambda *a: bg.causal_conv_silu(*a)[0], (x, w, c)),
            "norm": (norm, (x, gate, n, b)),
            "reorder": (lambda s: bg.reorder_states(s, [1, 0]), (st,)),
            "select": (lambda s: bg.select_states(s, [1, 0, 1]), (st,))}


@pytest.mark.parametrize("name", ["scan", "scan step", "scan in place", "conv", "norm", "reorder", "select"])
@pytest.mark.parametrize("grad", [False, True])
def test_operators_refuse_a_tangent(name, grad):
    call, args = _operators()[name]
    for k in range(len(args)):
        with fwAD.dual_level():
            mine = [t.clone().requires_grad_(grad and name not in ("scan in place", "reorder", "select")) for t in args]
            mine[k] = fwAD.make_dual(mine[k], torch.ones_like(mine[k]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(*mine)
    call(*[t.clone() for t in args])  # and without one

"""GPU: second derivatives of the training layer where the recurrence takes no part in them: its gate, its norm and its
output projection, which the core's output enters as a constant (or through the core's first derivative)."""
import pytest
import torch

from training_ref import torch_loop_core

pytestmark = pytest.mark.gpu

GATE = ("o_norm_w", "g_proj_0", "g_proj_1_w", "g_proj_1_b", "o_proj")


@pytest.mark.parametrize("T", [40, 100])
def test_penalty_on_the_gate_gradients(T):
    """The gradient of a penalty on the gate's gradients, in every weight, against float64 autograd of the same graph:
    twice the bar of the layer's f32 gradients (1e-3 relative and of the RMS), for two passes."""
    import burn_gdn2 as bg
    from burn_gdn2 import training

    cfg = bg.Gdn2Config(mode=bg.Gdn2Mode.Chunk, chunk_size=64, hidden_size=128, num_heads=2, head_dim=64)
    m = bg.GatedDeltaNet2.new(cfg, device="cuda", dtype=torch.float32, seed=3)
    gen = torch.Generator("cuda").manual_seed(5)
    x, r = (torch.randn(2, T, 128, device="cuda", generator=gen) for _ in range(2))

    def penalty(P, x, r, core):
        y = training.layer_forward(P, cfg, x, core=core)
        grads = torch.autograd.grad((y * r).sum(), [P[n] for n in GATE], create_graph=True)
        # weighted, so that each kind of weight counts alike
        return sum(g.square().mean() for g in grads)

    P = {n: t.detach().clone().requires_grad_(True) for n, t in m.parameters().items()}
    P64 = {n: t.detach().double().cpu().requires_grad_(True) for n, t in P.items()}
    names = [n for n in P if n in GATE or n in ("q_proj", "v_proj", "v_conv_w", "w_proj")]
    got_p, want_p = penalty(P, x, r, training.cuda_core), penalty(P64, x.double().cpu(), r.double().cpu(), torch_loop_core)
    got = torch.autograd.grad(got_p, [P[n] for n in names])
    want = torch.autograd.grad(want_p, [P64[n] for n in names])
    for n, a, b in zip(names, got, want):
        a = a.double().cpu()
        assert ((a - b).abs() <= 2e-3 * b.abs() + 2e-3 * b.square().mean().sqrt()).all(), (n, float((a - b).norm() / b.norm()))


def test_gradients_with_and_without_a_graph():
    """create_graph takes the norm's gradient through torch ops: the same gradients at the layer's bar."""
    import burn_gdn2 as bg

    cfg = bg.Gdn2Config(mode=bg.Gdn2Mode.Chunk, chunk_size=64, hidden_size=128, num_heads=2, head_dim=64)
    m = bg.GatedDeltaNet2.new(cfg, device="cuda", dtype=torch.float32, seed=6)
    m.requires_grad_(True)
    gen = torch.Generator("cuda").manual_seed(7)
    x = torch.randn(2, 50, 128, device="cuda", generator=gen).requires_grad_(True)
    r = torch.randn(2, 50, 128, device="cuda", generator=gen)
    leaves = [x, *m.parameters().values()]
    leaves = [t for t in leaves if t.requires_grad]
    grads = [torch.autograd.grad((m.forward_train_autograd(x) * r).sum(), leaves, create_graph=c, allow_unused=True)
             for c in (False, True)]
    for a, b in zip(*grads):
        assert (a is None) == (b is None)
        if a is not None:
            assert ((a - b).abs() <= 1e-3 * a.abs() + 1e-3 * a.square().mean().sqrt()).all()

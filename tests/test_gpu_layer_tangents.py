"""GPU: forward-mode derivatives of the training layer.  Its gated norm runs on an operator that has none; its gate and
norm weights, which do not pass through the recurrence, have theirs all the same."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from training_ref import torch_loop_core

pytestmark = pytest.mark.gpu

GATE = ("o_norm_w", "g_proj_0", "g_proj_1_w", "g_proj_1_b")


@pytest.mark.parametrize("T", [40, 100])
@pytest.mark.parametrize("grad", [False, True])
def test_layer_tangents_of_the_gate_and_norm_weights(T, grad):
    """Against central differences of the float64 layer, at the bar of the layer's f32 gradients (1e-3 relative and of
    the RMS); a step of 1e-4 leaves the differences' own error near 1e-8."""
    import burn_gdn2 as bg
    from burn_gdn2 import training

    cfg = bg.Gdn2Config(mode=bg.Gdn2Mode.Chunk, chunk_size=64, hidden_size=128, num_heads=2, head_dim=64)
    m = bg.GatedDeltaNet2.new(cfg, device="cuda", dtype=torch.float32, seed=3)
    gen = torch.Generator("cuda").manual_seed(4)
    x = torch.randn(2, T, 128, device="cuda", generator=gen)
    P = dict(m.parameters())
    P64 = {n: t.detach().double().cpu() for n, t in P.items()}
    for n in GATE:
        way = torch.randn(P[n].shape, device="cuda", generator=gen)
        with fwAD.dual_level():
            Q = {k: t.detach().clone().requires_grad_(grad) for k, t in P.items()}
            Q[n] = fwAD.make_dual(Q[n], way)
            got = fwAD.unpack_dual(training.layer_forward(Q, cfg, x)).tangent
            assert got is not None, n
            got = got.detach().double().cpu()
        at = lambda s: training.layer_forward({**P64, n: P64[n] + s * way.double().cpu()}, cfg, x.double().cpu(), core=torch_loop_core)
        want = (at(1e-4) - at(-1e-4)) / 2e-4
        assert ((got - want).abs() <= 1e-3 * want.abs() + 1e-3 * want.square().mean().sqrt()).all(), n


def test_layer_refuses_the_recurrence_s_tangents():
    """What passes through the core has no forward derivative, in silence least of all."""
    import burn_gdn2 as bg
    from burn_gdn2 import training

    cfg = bg.Gdn2Config(mode=bg.Gdn2Mode.Chunk, chunk_size=64, hidden_size=128, num_heads=2, head_dim=64)
    m = bg.GatedDeltaNet2.new(cfg, device="cuda", dtype=torch.float32, seed=3)
    x = torch.randn(1, 30, 128, device="cuda")
    for n in ("q_conv_w", "v_proj", "A_log"):
        with fwAD.dual_level():
            Q = {k: t.detach() for k, t in m.parameters().items()}
            Q[n] = fwAD.make_dual(Q[n], torch.ones_like(Q[n]))
            with pytest.raises(RuntimeError):
                training.layer_forward(Q, cfg, x)

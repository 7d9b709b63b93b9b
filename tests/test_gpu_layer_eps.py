"""GPU: the training layer with a norm_eps that f32 does not hold (below its smallest number) normalises as with none."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [1e-50, 1e-40])
def test_norm_eps_below_f32(eps):
    import dataclasses

    import burn_gdn2 as bg
    from burn_gdn2 import training

    cfg = bg.Gdn2Config(mode=bg.Gdn2Mode.Chunk, chunk_size=64, hidden_size=128, num_heads=2, head_dim=64, norm_eps=eps)
    m = bg.GatedDeltaNet2.new(cfg, device="cuda", dtype=torch.float32, seed=3)
    x = torch.randn(1, 30, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    P = {n: t.detach().clone().requires_grad_(True) for n, t in m.parameters().items()}
    y = training.layer_forward(P, cfg, x)
    # an eps far below the mean squares here changes nothing that f32 holds
    near = dataclasses.replace(cfg, norm_eps=1e-30)
    want = training.layer_forward(P, near, x)
    assert ((y - want).abs() <= 1e-5 * want.abs() + 1e-5 * want.square().mean().sqrt()).all()
    (g,) = torch.autograd.grad(y.square().sum(), P["o_norm_w"])
    assert torch.isfinite(g).all() and g.any()

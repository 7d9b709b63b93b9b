"""GPU: the training layer without the sequence operators' torch extension warns and runs its convs and its norm as torch
ops: the same output and gradients at the layer's f32 bar (1e-3 relative and of the RMS)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_training_without_the_extension(monkeypatch):
    import burn_gdn2 as bg
    from burn_gdn2 import sequence

    cfg = bg.Gdn2Config(mode=bg.Gdn2Mode.Chunk, chunk_size=64, hidden_size=128, num_heads=2, head_dim=64)
    m = bg.GatedDeltaNet2.new(cfg, device="cuda", dtype=torch.float32, seed=3).requires_grad_(True)
    x = torch.randn(2, 100, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1))

    def train():
        y = m.forward_train_autograd(x)
        return [y.detach(), *torch.autograd.grad(y.square().sum(), list(m.parameters().values()))]

    with_it = train()
    monkeypatch.setattr(sequence, "_calls", sequence._NotBuilt(ImportError("not there")))
    with pytest.warns(UserWarning, match="build.py"):
        without = train()
    for a, b in zip(with_it, without):
        assert ((a - b).abs() <= 1e-3 * a.abs() + 1e-3 * a.square().mean().sqrt()).all()

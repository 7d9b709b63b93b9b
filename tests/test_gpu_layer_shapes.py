"""GPU: the training layer takes weights in the shapes that the fused layer takes: a convolution's as [C,1,4], the norm's
with leading ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_conv_and_norm_weights_with_more_dimensions():
    import burn_gdn2 as bg

    cfg = bg.Gdn2Config(mode=bg.Gdn2Mode.Chunk, chunk_size=64, hidden_size=128, num_heads=2, head_dim=64)
    plain = bg.GatedDeltaNet2.new(cfg, device="cuda", dtype=torch.float32, seed=3)
    W = plain.export_weights()
    other = dict(W, o_norm_w=W["o_norm_w"][None], **{n: W[n][:, None] for n in ("q_conv_w", "k_conv_w", "v_conv_w")})
    other = bg.GatedDeltaNet2(cfg, other, device="cuda")
    x = torch.randn(2, 30, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    assert torch.equal(other.forward_train(x), plain.forward_train(x))
    ys, grads = [], []
    for m in (plain, other):
        m.requires_grad_(True)
        y = m.forward_train_autograd(x)
        y.square().sum().backward()
        ys.append(y)
        grads.append([m.parameters()[n].grad for n in ("o_norm_w", "q_conv_w", "k_conv_w", "v_conv_w")])
    assert torch.equal(*ys)
    for a, b in zip(*grads):
        assert torch.equal(a.flatten(), b.flatten())

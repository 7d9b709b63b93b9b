"""GPU: the sequence operators together, as a gated-recurrence block uses them:
short convolution, scan with its decay, gated group norm, over packed
documents in training and token by token, with forks and freed sequences, in
serving, against the same block in float64.

The bound is normwise: worst case, the convolution is off by some 16 f32
roundings (2^-24) of its terms, a scan over 60 tokens by 4 * 60 + 8, the norm
by about 100, 372 together; a gradient passes the same again, 744, and the
norm may stretch what enters it (groups of unequal sizes) some three times:
3 * 744 * 2^-24 = 1.4e-4."""
import pytest
import torch

import sequence_ref as R

pytestmark = pytest.mark.gpu
TOL = 3 * 744 * 2.0 ** -24
C, G = 48, 3


def _weights(seed):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    return {"w_in": r(C, C) / C ** 0.5, "w_f": r(C, C) / C ** 0.5, "w_gate": r(C, C) / C ** 0.5, "conv": 0.5 * r(C, 4),
            "norm": 1 + 0.1 * r(C), "bias": 0.1 * r(C), "rate": torch.rand(C, generator=gen) * 2}


def _parts(x, W):
    softplus = torch.nn.functional.softplus
    return x @ W["w_in"], -W["rate"] * softplus(x @ W["w_f"]), x @ W["w_gate"]


def _block(x, W, cache, state, cu):
    import burn_gdn2 as bg

    u, g, gate = _parts(x, W)
    v, cache = bg.causal_conv_silu(u, W["conv"], cache, cu_seqlens=cu)
    h, state = bg.gated_scan(v, g, state, cu_seqlens=cu, complement=True)
    return bg.group_norm_gate(h, gate, W["norm"], W["bias"], num_groups=G), cache, state


def _block64(x, W, cache, state):
    """One sequence [T,C] in float64, by torch autograd."""
    u, g, gate = _parts(x, W)
    line = torch.cat((cache, u))
    v = torch.nn.functional.silu(sum(line[j:j + len(u)] * W["conv"][:, j] for j in range(4)))
    hs = []
    for t in range(len(u)):
        state = g[t].exp() * state - torch.expm1(g[t]) * v[t]
        hs.append(state)
    h = torch.stack(hs).reshape(-1, G, C // G)
    n = (h - h.mean(-1, keepdim=True)) * (h.var(-1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    y = (n.reshape(-1, C) * W["norm"] + W["bias"]) * torch.nn.functional.silu(gate)
    return y, line[len(u):], state


def _near(got, want, what):
    rel = float((got.double().cpu() - want).norm() / want.norm())
    assert rel <= TOL, (what, rel)


def test_packed_training():
    lens = [17, 60, 1, 33, 2]
    gen = torch.Generator().manual_seed(1)
    W, N, rows = _weights(2), len(lens), sum(lens)
    x, d = torch.randn(rows, C, generator=gen), torch.randn(rows, C, generator=gen)
    cache, state = torch.randn(N, 3, C, generator=gen), torch.randn(N, C, generator=gen)
    Wd = {k: t.cuda().requires_grad_(True) for k, t in W.items()}
    xd, cd, sd = (t.cuda().requires_grad_(True) for t in (x[None], cache, state))
    cu = torch.tensor([0] + lens).cumsum(0).int()
    y, c1, s1 = _block(xd, Wd, cd, sd, cu)
    leaves = [xd, cd, sd, *Wd.values()]
    grads = torch.autograd.grad((y, c1.sum() + s1.square().sum()), leaves, (d[None].cuda(), torch.ones((), device="cuda")))

    W64 = {k: t.double().requires_grad_(True) for k, t in W.items()}
    x64, c64, s64 = (t.double().requires_grad_(True) for t in (x, cache, state))
    outs, at = [], 0
    for n, length in enumerate(lens):
        outs.append(_block64(x64[at:at + length], W64, c64[n], s64[n]))
        at += length
    y64, cs, ss = torch.cat([o[0] for o in outs]), torch.stack([o[1] for o in outs]), torch.stack([o[2] for o in outs])
    want = torch.autograd.grad((y64, cs.sum() + ss.square().sum()), [x64, c64, s64, *W64.values()],
                               (d.double(), torch.ones((), dtype=torch.float64)))
    _near(y[0].detach(), y64.detach(), "y")
    _near(c1.detach(), cs.detach(), "cache")
    _near(s1.detach(), ss.detach(), "state")
    for name, a, b in zip(["x", "cache", "state", *W], grads, want):
        _near(a.reshape(b.shape), b, name)


def test_serving_with_forks_and_freed_sequences():
    """Prefill, decode steps, a fork and a freed row, more steps: each sequence as if alone from its start."""
    import burn_gdn2 as bg

    gen = torch.Generator().manual_seed(3)
    W = _weights(4)
    Wd, W64 = {k: t.cuda() for k, t in W.items()}, {k: t.double() for k, t in W.items()}
    x = torch.randn(3, 30, C, generator=gen)
    later = torch.randn(3, 6, C, generator=gen)
    with torch.no_grad():
        y, cache, state = _block(x.cuda(), Wd, torch.zeros(3, 3, C, device="cuda"), None, None)
        for t in range(2):
            y, cache, state = _block(later[:, t:t + 1].cuda(), Wd, cache, state, None)
        # row 1 goes on as a fork of row 2, row 2 starts again
        index = [0, 2, -1]
        bg.reorder_states([cache, state], index)
        steps = []
        for t in range(2, 6):
            y, cache, state = _block(later[:, t:t + 1].cuda(), Wd, cache, state, None)
            steps.append(y)
    got = torch.cat(steps, 1)
    for row, source in enumerate(index):
        past = torch.cat((x[source], later[source, :2])) if source >= 0 else x[0, :0]
        line = torch.cat((past, later[row, 2:])).double()
        want, c64, s64 = _block64(line, W64, torch.zeros(3, C, dtype=torch.float64), torch.zeros(C, dtype=torch.float64))
        _near(got[row], want[-4:], f"row {row}")
        _near(cache[row], c64, f"cache {row}")
        _near(state[row], s64, f"state {row}")


def test_captured_decode_step():
    """A decode step of the block in a CUDA graph, its states carried in place, as the eager steps."""
    import burn_gdn2 as bg

    Wd = {k: t.cuda() for k, t in _weights(5).items()}
    gen = torch.Generator("cuda").manual_seed(6)
    tokens = torch.randn(5, 4, 1, C, generator=gen, device="cuda")
    with torch.no_grad():
        cache, state = torch.zeros(4, 3, C, device="cuda"), torch.zeros(4, C, device="cuda")
        want = []
        for t in tokens:
            y, cache, state = _block(t, Wd, cache, state, None)
            want.append(y)
        held = [torch.zeros(4, 3, C, device="cuda"), torch.zeros(4, C, device="cuda")]

        def step(x):
            u, g, gate = _parts(x, Wd)
            v, new = bg.causal_conv_silu(u, Wd["conv"], held[0])
            held[0].copy_(new)
            h, _ = bg.gated_scan(v, g, held[1], complement=True, inplace=True)
            return bg.group_norm_gate(h, gate, Wd["norm"], Wd["bias"], num_groups=G)

        slot = torch.zeros(4, 1, C, device="cuda")
        graph = bg.GraphedCall(step, slot)
        for t in held:
            t.zero_()
        for t, w in zip(tokens, want):
            slot.copy_(t)
            assert torch.equal(graph.replay(), w)
    assert torch.equal(held[0], cache) and torch.equal(held[1], state)


def test_state_methods():
    import burn_gdn2 as bg

    s = bg.Gdn2State.zeros("cuda", 3, 2, 16, 16, 32, 32)
    for k, t in enumerate((s.recurrent, s.conv_q, s.conv_k, s.conv_v)):
        t += torch.arange(3, device="cuda").reshape(3, *[1] * (t.dim() - 1)) + 1 + 10 * k
    new = s.select([2, -1, 0, 2])
    assert isinstance(new, bg.Gdn2State) and new.recurrent.shape[0] == 4
    assert new.conv_v[:, 0, 0].tolist() == [33, 0, 31, 33] and new.recurrent[:, 0, 0, 0].tolist() == [3, 0, 1, 3]
    s.reorder([1, 0, -1])
    assert s.recurrent[:, 1, 2, 3].tolist() == [2, 1, 0] and s.conv_q[:, 2, 5].tolist() == [12, 11, 0]

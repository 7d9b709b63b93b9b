"""GPU: gated_scan where a reset (a decay of zero) stands beside growth whose product leaves f32's range: a reset
leaves nothing for the growth to multiply, however the time axis is cut, in either direction.  Bounds as in
test_gpu_scan.py (sequence_ref.scan_one)."""
import pytest
import torch

import sequence_ref as R
from test_gpu_scan import _check, _decay, _gen, _run

pytestmark = pytest.mark.gpu

# tokens, channels, sequences, spans of growth, rate: growth of one token beyond f32, of a run, of several runs of a
# segment, of a long segment's tiles, and in blocks of eight warps
CASES = [(10, 34, 1, [(3, 4)], 90.0), (16, 64, 1, [(2, 3), (9, 12)], 90.0), (60, 33, 1, [(3, 50)], 6.0),
         (200, 64, 1, [(5, 120), (140, 143)], 6.0), (5000, 12, 1, [(3, 2000), (2500, 2600), (3001, 4990)], 3.0),
         (24581, 6, 1, [(70, 200), (300, 301), (1000, 9000), (20000, 20100)], 6.0),
         (300, 66, 100, [(3, 50), (130, 260)], 6.0)]


def _inputs(T, C, B, spans, rate, reset):
    """Growth on every other channel, between a reset before it (the forward's) and one behind it (the adjoint's);
    neither x nor the gradient of h touches these tokens, the state and both its gradients are not zero."""
    gen = _gen(T + C)
    xs, gs, dh = torch.randn(B, T, C, generator=gen), _decay(gen, B, T, C), torch.randn(B, T, C, generator=gen)
    for a, b in spans:
        gs[:, a - 1, ::2] = gs[:, b, ::2] = reset
        gs[:, a:b, ::2] = rate
        xs[:, a - 1:b, ::2] = dh[:, a - 1:b, ::2] = 0.0
    st, ds = torch.randn(B, C, generator=gen), torch.randn(B, C, generator=gen)
    return [t.reshape(-1, C) for t in (xs, gs, st, dh, ds)]


@pytest.mark.parametrize("T,C,B,spans,rate", CASES)
@pytest.mark.parametrize("reset,comp", [(-float("inf"), False), (-float("inf"), True), (-1000.0, False)])
def test_dense(T, C, B, spans, rate, reset, comp):
    xs, gs, st, dh, ds = _inputs(T, C, B, spans, rate, reset)
    got = _run(xs, gs, st, dh, ds, (B, T), None, comp, True)
    for b in {0, B // 2, B - 1}:
        part = slice(b * T, (b + 1) * T)
        want, bound = R.scan(xs[part], gs[part], st[b:b + 1], [T], comp, dh[part], ds[b:b + 1])
        _check({k: v[part] if v.shape[0] == B * T else v[b:b + 1] for k, v in got.items()}, want, bound)


@pytest.mark.parametrize("T,C,B,spans,rate", [c for c in CASES if c[2] == 1])
def test_packed(T, C, B, spans, rate):
    """The same between two other sequences and an empty one."""
    xs, gs, st, dh, ds = _inputs(T, C, 1, spans, rate, -float("inf"))
    gen = _gen(1)
    more = lambda t, n: torch.cat((torch.randn(n, C, generator=gen), t, torch.randn(n, C, generator=gen)))
    xs, dh, gs = more(xs, 21), more(dh, 21), torch.cat((_decay(gen, 21, C), gs, _decay(gen, 21, C)))
    lens = [21, T, 0, 21]
    st, ds = torch.randn(4, C, generator=gen), torch.randn(4, C, generator=gen)
    cu = torch.tensor([0] + lens).cumsum(0).int()
    want, bound = R.scan(xs, gs, st, lens, False, dh, ds)
    _check(_run(xs, gs, st, dh, ds, (1, len(xs)), cu, False, True), want, bound)


def test_as_token_by_token():
    """Reset, then growth beyond f32, from a state: the decode step's result and a whole pass's."""
    import burn_gdn2 as bg

    x, st = torch.zeros(1, 2, 4, device="cuda"), torch.ones(1, 4, device="cuda")
    g = torch.tensor([-float("inf"), 90.0], device="cuda")[None, :, None].expand(1, 2, 4)
    h, last = bg.gated_scan(x, g, st)
    h0, s = bg.gated_scan(x[:, :1], g[:, :1], st)
    h1, s = bg.gated_scan(x[:, 1:], g[:, 1:], s)
    assert not h0.any() and not h1.any() and torch.equal(h, torch.cat((h0, h1), 1)) and torch.equal(last, s)
    # a decay that is not a number is none of this
    h, last = bg.gated_scan(x, g.clone().masked_fill_(g > 0, float("nan")), st)
    assert torch.isnan(last).all()

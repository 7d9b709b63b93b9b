"""Float64 restatements of the sequence operators, with the error that f32
arithmetic may add to each value.  Checker only."""
import torch

EPS = 2.0 ** -24  # half a step of f32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def scan_one(x, g, state, comp, d_h, d_state):
    """One sequence [T,C] of the gated scan, token by token, and its adjoint.

    Returns (values, bounds) as dicts.  A decay e^g is off by at most a step
    (2 EPS relative), the products of decays that join spans add EPS a factor
    and the sums EPS a step, so the part of h_t that comes from token s is
    off by at most (4 (t - s) + 8) EPS of its size: P sums the sizes, Q the
    sizes times t - s.  The adjoint is the same sum from the other end, and
    dg = e^g (h - x) l takes the errors of both factors."""
    T, C = x.shape
    a, w = g.exp(), (-torch.expm1(g) if comp else torch.ones_like(g))
    h = torch.empty_like(x)
    eh = torch.empty_like(x)
    now, P, Q = state.clone(), state.abs(), torch.zeros_like(state)
    before, e_before = torch.empty_like(x), torch.empty_like(x)
    for t in range(T):
        before[t], e_before[t] = now, EPS * (4 * Q + 8 * P)
        now = a[t] * now + w[t] * x[t]
        P, Q = a[t] * P + (w[t] * x[t]).abs(), a[t] * (Q + P)
        h[t], eh[t] = now, EPS * (4 * Q + 8 * P)
    values, bounds = {"h": h, "state": now}, {"h": eh, "state": EPS * (4 * Q + 8 * P)}
    if d_h is None:
        return values, bounds
    lam, el = torch.empty_like(x), torch.empty_like(x)
    mu, P, Q = d_state.clone(), d_state.abs(), torch.zeros_like(d_state)
    for t in range(T - 1, -1, -1):
        lam[t] = d_h[t] + mu
        P, Q = P + d_h[t].abs(), Q
        el[t] = EPS * (4 * Q + 8 * P)
        mu = a[t] * lam[t]
        P, Q = a[t] * P, a[t] * (Q + P)
    d = before - x if comp else before
    values.update(dx=w * lam, dg=a * d * lam, d_state=mu)
    size = before.abs() + (x.abs() if comp else 0)
    # |w (l + e) - w l| = |w| |e|: w = 1 - e^g is negative where g > 0, an error's bound never is
    bounds.update(dx=w.abs() * el + 4 * EPS * (w * lam).abs(),
                  dg=a * (d.abs() * el + e_before * lam.abs() + 8 * EPS * size * lam.abs()),
                  d_state=EPS * (4 * Q + 8 * P))
    return values, bounds


def scan(x, g, state, lens, comp, d_h=None, d_state=None):
    """Sequences of lens rows each of [R,C] (rows behind the last come out as
    zero); state, d_state [N,C] or None.  Float64 throughout."""
    R, C = x.shape
    N = len(lens)
    zero = lambda t, *s: torch.zeros(*s, dtype=torch.float64) if t is None else t.double()
    x, g, state = x.double(), g.double(), zero(state, N, C)
    keys_rows, keys_seq = ["h"] + (["dx", "dg"] if d_h is not None else []), ["state"] + (["d_state"] if d_h is not None else [])
    out = {k: torch.zeros(R, C, dtype=torch.float64) for k in keys_rows}
    out.update({k: torch.zeros(N, C, dtype=torch.float64) for k in keys_seq})
    tol = {k: torch.zeros_like(v) for k, v in out.items()}
    d_state = zero(d_state, N, C)
    at = 0
    for n, length in enumerate(lens):
        s = slice(at, at + length)
        v, b = scan_one(x[s], g[s], state[n], comp, None if d_h is None else d_h.double()[s], d_state[n])
        for k in keys_rows:
            out[k][s], tol[k][s] = v[k], b[k]
        for k in keys_seq:
            out[k][n], tol[k][n] = v[k], b[k]
        at += length
    return out, tol


def check(got, want, bound, what):
    """got (any dtype) within the bound of f32 arithmetic plus one rounding to its dtype."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    rounding = half_step(got.dtype) if got.dtype != torch.float32 else 0.0
    tiny = torch.finfo(torch.float32).tiny
    g = got.double().cpu()
    assert torch.equal(torch.isnan(g), torch.isnan(want)), f"{what}: NaN in other places"
    lim = bound + rounding * (want.abs() + bound) + tiny
    err = (g - want).abs()
    bad = (err > lim) & ~torch.isnan(want)
    if bad.any():
        i = int((err - lim).masked_fill(torch.isnan(err), -1).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())}/{bad.numel()} outside; worst at {i}: got {g.flatten()[i]:.9g} "
                             f"want {want.flatten()[i]:.9g}, allowed {lim.flatten()[i]:.3g}")

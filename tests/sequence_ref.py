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


def silu_parts(t):
    """sigmoid, silu, silu' and the absolute errors of the last two for an exact t: the fast exponential is within
    (4 + 2 |t|) EPS, the fast division within 4 EPS, relative."""
    sig = torch.sigmoid(t)
    act, slope = t * sig, sig * (1 + t * (1 - sig))
    rel = (16 + 2 * t.abs()) * EPS
    return act, slope, rel * act.abs(), rel * sig * (1 + 2 * t.abs())


def group_norm(x, gate, weight, bias, groups, eps, center, d=None):
    """[R,C] group norm with SiLU and its adjoint, with bounds.

    Sums over a group run at most 50 deep (16 values a lane, then trees), so a mean is off by 50 EPS of the mean
    size A.  A deviation is off by that and its own rounding; rstd, relative, by half the variance's error (twice
    the deviations' over sigma, and the sum's) and the root's 4 EPS.  Weight gradients are sums over the rows, at
    most one addition a row deep."""
    f64 = lambda t: None if t is None else t.double()
    x, gate, weight, bias, d = (f64(t) for t in (x, gate, weight, bias, d))
    rows, chan = x.shape
    per = lambda t: t.reshape(rows, groups, -1)
    wide = lambda t, default: torch.full((1, 1), default, dtype=torch.float64) if t is None else t.reshape(-1, chan // groups)
    v, w, b = per(x), wide(weight, 1.0), wide(bias, 0.0)
    A = v.abs().mean(-1, keepdim=True)
    dev = v - v.mean(-1, keepdim=True) if center else v
    e_dev = (50 * EPS * A if center else 0) + 2 * EPS * dev.abs()
    rstd = ((dev * dev).mean(-1, keepdim=True) + eps).rsqrt()
    rel_r = (50 * A * rstd if center else 0) * EPS + 31 * EPS
    n = dev * rstd
    e_n = rstd * e_dev + n.abs() * (rel_r + EPS)
    z = n * w + b
    e_z = w.abs() * e_n + 2 * EPS * ((n * w).abs() + b.abs())
    t = z if gate is None else per(gate)
    act, slope, e_act, e_slope = silu_parts(t)
    if gate is None:
        y, e_y = act, e_act + 1.1 * e_z + EPS * act.abs()
    else:
        y, e_y = z * act, z.abs() * e_act + act.abs() * e_z + 2 * EPS * (z * act).abs()
    flat = lambda t: t.reshape(rows, chan)
    out, tol = {"y": flat(y)}, {"y": flat(e_y)}
    if d is None:
        return out, tol
    d = per(d)
    if gate is None:
        dz, e_dz = d * slope, d.abs() * (e_slope + 0.5 * e_z) + EPS * (d * slope).abs()
    else:
        dz, e_dz = d * act, d.abs() * e_act + EPS * (d * act).abs()
        out["d_gate"] = flat(d * z * slope)
        tol["d_gate"] = flat(d.abs() * (e_z * slope.abs() + z.abs() * e_slope) + 3 * EPS * (d * z * slope).abs())
    dn = dz * w
    e_dn = w.abs() * e_dz + EPS * dn.abs()
    mean = lambda t: t.mean(-1, keepdim=True)
    m0, e_m0 = (mean(dn), mean(e_dn) + 50 * EPS * mean(dn.abs())) if center else (0, 0)
    m1 = mean(dn * n)
    e_m1 = mean(e_dn * n.abs() + dn.abs() * e_n) + 50 * EPS * mean((dn * n).abs())
    dx = rstd * (dn - m0 - n * m1)
    size = dn.abs() + (m0.abs() if center else 0) + (n * m1).abs()
    out["dx"] = flat(dx)
    tol["dx"] = flat(rstd * (e_dn + e_m0 + n.abs() * e_m1 + e_n * m1.abs() + 3 * EPS * size) + dx.abs() * (rel_r + EPS))
    for name, given, g, e in (("d_weight", weight, dz * n, e_dz * n.abs() + dz.abs() * e_n), ("d_bias", bias, dz, e_dz)):
        if given is not None:
            over = (0,) if given.numel() == chan else (0, 1)
            deep = (rows if given.numel() == chan else rows * groups) + 8
            out[name] = g.sum(over).reshape(given.shape)
            tol[name] = (e.sum(over) + deep * EPS * g.abs().sum(over)).reshape(given.shape)
    return out, tol


def conv(x, weight, cache, lens, d_y=None, d_cache=None):
    """Sequences of lens rows each of [R,C] through the 4-tap causal convolution with SiLU, and its adjoint, with
    bounds: a sum of n products is off by at most (n + 1) EPS of the sum of their sizes."""
    R, C = x.shape
    N = len(lens)
    x, w = x.double(), weight.double()
    train = d_y is not None
    out = {"y": torch.zeros(R, C, dtype=torch.float64), "cache": torch.zeros(N, 3, C, dtype=torch.float64)}
    if train:
        out.update(dx=torch.zeros(R, C, dtype=torch.float64), d_weight=torch.zeros(C, 4, dtype=torch.float64))
        if cache is not None:
            out["d_cache"] = torch.zeros(N, 3, C, dtype=torch.float64)
    tol = {k: torch.zeros_like(v) for k, v in out.items()}
    dw_size = torch.zeros(C, 4, dtype=torch.float64)
    at = 0
    for n, length in enumerate(lens):
        s = slice(at, at + length)
        at += length
        seq = x[s]
        if cache is not None:
            front = cache[n].double()
        else:
            front = seq[:1].expand(3, C) if length else torch.zeros(3, C, dtype=torch.float64)
        line = torch.cat((front, seq))
        out["cache"][n] = line[length:]
        taps = torch.stack([line[j:j + length] for j in range(4)], -1)  # [T,C,4]
        pre = (taps * w).sum(-1)
        e_pre = 5 * EPS * (taps * w).abs().sum(-1)
        act, slope, e_act, e_slope = silu_parts(pre)
        out["y"][s], tol["y"][s] = act, e_act + 1.1 * e_pre
        if not train:
            continue
        d = d_y.double()[s]
        dp, e_dp = d * slope, d.abs() * (e_slope + 0.5 * e_pre) + EPS * (d * slope).abs()
        d_line, e_line, size = (torch.zeros(length + 3, C, dtype=torch.float64) for _ in range(3))
        for j in range(4):
            d_line[j:j + length] += dp * w[:, j]
            e_line[j:j + length] += e_dp * w[:, j].abs()
            size[j:j + length] += (dp * w[:, j]).abs()
        if d_cache is not None:
            d_line[length:] += d_cache[n].double()
            size[length:] += d_cache[n].double().abs()
        out["dx"][s], tol["dx"][s] = d_line[3:], e_line[3:]
        count = 6 * size
        if cache is not None:
            out["d_cache"][n], tol["d_cache"][n] = d_line[:3], e_line[:3] + EPS * count[:3]
        elif length:  # copies of the first token: four values' sums come together
            out["dx"][s][0] += d_line[:3].sum(0)
            tol["dx"][s][0] += e_line[:3].sum(0) + 16 * EPS * size[:4].sum(0)
        tol["dx"][s] += EPS * count[3:]
        out["d_weight"] += (dp[..., None] * taps).sum(0)
        tol["d_weight"] += (e_dp[..., None] * taps.abs()).sum(0)
        dw_size += (dp[..., None] * taps).abs().sum(0)
    if train:
        tol["d_weight"] += (R + 8) * EPS * dw_size
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

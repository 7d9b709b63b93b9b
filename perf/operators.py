"""Cases that time the sequence operators around a gated recurrence.

Four operators, each in training (forward and every gradient) and in serving
form:

* ``gated_scan``: h_t = e^{g_t} h_{t-1} + s_t x_t over long sequences, one
  state per channel, with s_t = 1 or s_t = 1 - e^{g_t} ("complement"), from a
  given state, dense or packed;
* ``causal_conv_silu``: the 4-tap depthwise causal convolution with SiLU in
  front of such a recurrence, with its cache of three tokens, dense or packed;
* ``group_norm_gate``: the norm of each token's channel groups behind it
  (channels last), with an affine map and a SiLU, gated or not;
* ``reorder_states``: forking, compacting and freeing the rows of the state
  pool that a batch of running sequences keeps.

``run`` computes them in elementary torch operations in 32 bits, or, where
``own`` is set, calls the package.  ``exact`` gives the results in 64 bits.
"""
import math
import os
import sys

import torch

own = False

TAPS = 4  # taps of the short convolution; its cache holds TAPS - 1 tokens
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "burn-gdn2_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import burn_gdn2

    return burn_gdn2


# -- cases -------------------------------------------------------------------


def listed():
    return [
        # one decode step of a serving batch: 256 sequences, 2048 channels, a launch's latency
        {"name": "scan step", "op": "scan", "batch": 256, "len": 1, "lens": "", "chan": 2048, "x": "bf16", "g": "f32",
         "complement": False, "state": True, "train": False},
        # prefill of eight prompts of 4096 tokens into their states, forward alone
        {"name": "scan prefill", "op": "scan", "batch": 8, "len": 4096, "lens": "", "chan": 2048, "x": "bf16",
         "g": "f32", "complement": False, "state": True, "train": False},
        # a training step's pass, forward and backward, at the same size
        {"name": "scan train", "op": "scan", "batch": 8, "len": 4096, "lens": "", "chan": 2048, "x": "bf16",
         "g": "f32", "complement": False, "state": False, "train": True},
        # one long document: few chains, 65536 tokens, the whole axis scanned
        {"name": "scan long", "op": "scan", "batch": 1, "len": 65536, "lens": "", "chan": 1024, "x": "bf16",
         "g": "bf16", "complement": True, "state": False, "train": True},
        # documents of different lengths packed into one row, an empty and a one-token one among them, odd channels
        {"name": "scan packed", "op": "scan", "batch": 1, "len": 0, "lens": "700,1,4099,0,63,2048,5,129,7001,333",
         "chan": 1001, "x": "f32", "g": "f32", "complement": True, "state": True, "train": True},
        # the norm behind one decode step: 256 tokens of 16 heads of 128
        {"name": "norm step", "op": "norm", "rows": 256, "groups": 16, "width": 128, "x": "bf16", "gate": True,
         "affine": "channel", "bias": False, "center": True, "train": False},
        # the same norm in a training step over 8 sequences of 4096 tokens
        {"name": "norm train", "op": "norm", "rows": 32768, "groups": 16, "width": 128, "x": "bf16", "gate": True,
         "affine": "channel", "bias": True, "center": True, "train": True},
        # odd group widths in 32 bits, root mean square alone, weights shared by the groups, SiLU of the result
        {"name": "norm odd", "op": "norm", "rows": 5003, "groups": 7, "width": 90, "x": "f32", "gate": False,
         "affine": "group", "bias": False, "center": False, "train": True},
        # the convolution of one projection in a training step over 8 sequences of 4096 tokens
        {"name": "conv train", "op": "conv", "batch": 8, "len": 4096, "lens": "", "chan": 2048, "x": "bf16",
         "cache": False, "train": True},
        # packed documents that continue from their caches, shorter than the taps among them, odd channels
        {"name": "conv packed", "op": "conv", "batch": 1, "len": 0, "lens": "700,1,4099,0,63,2,5,129,3001,333",
         "chan": 1001, "x": "f32", "cache": True, "train": True},
        # a serving pool of 256 sequences after a third of them ended: live rows move down into the holes
        {"name": "pool compact", "op": "pool", "rows": 256, "heads": 16, "key": 128, "value": 128, "how": "compact"},
        # a small pool in which one sequence is forked into beams: the smallest call
        {"name": "pool fork", "op": "pool", "rows": 16, "heads": 4, "key": 64, "value": 64, "how": "fork"},
    ]


def _span(rng, low, high):
    """A size between low and high, even over its logarithm, odd as often as not."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(("scan", "scan", "conv", "norm", "norm", "pool"))
    if op == "pool":
        key = rng.choice((16, 32, 64, 80, 128))
        value = rng.choice((16, 48, 64, 128, 256))
        heads = _span(rng, 1, 32)
        rows = _span(rng, 2, max(2, min(512, (1 << 26) // (heads * key * value))))
        return {"op": op, "rows": rows, "heads": heads, "key": key, "value": value,
                "how": rng.choice(("compact", "fork", "shuffle"))}
    x = rng.choice(("f32", "bf16"))
    train = rng.random() < 0.7
    if op == "norm":
        width = _span(rng, 4, 512)
        groups = _span(rng, 1, max(1, min(64, 8192 // width)))
        rows = _span(rng, 1, max(1, min(32768, (1 << 25) // (width * groups))))
        return {"op": op, "rows": rows, "groups": groups, "width": width, "x": x, "gate": rng.random() < 0.6,
                "affine": rng.choice(("channel", "group", "none")), "bias": rng.random() < 0.4,
                "center": rng.random() < 0.6, "train": train}
    chan = _span(rng, 16, 4096)
    tokens = _span(rng, 1, max(1, min(65536, (1 << 25) // chan)))
    batch, length, lens = 1, 0, ""
    if rng.random() < 0.4:
        cuts = sorted(rng.randint(0, tokens) for _ in range(rng.randint(0, 12)))
        lens = ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [tokens]))
    else:
        batch = _span(rng, 1, min(256, tokens))
        length = max(1, tokens // batch)
    case = {"op": op, "batch": batch, "len": length, "lens": lens, "chan": chan, "x": x}
    if op == "scan":
        case.update(g=rng.choice(("f32", x)), complement=rng.random() < 0.5, state=rng.random() < 0.6, train=train)
    else:
        case.update(cache=rng.random() < 0.5, train=train)
    return case


def _lengths(case):
    return [int(v) for v in case["lens"].split(",")] if case["lens"] else [case["len"]] * case["batch"]


# -- inputs ------------------------------------------------------------------


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _decay(gen, chan, *shape):
    """Log decays as a trained gate gives them: -A softplus(f + bias), A from
    1 to 16 and the bias such that softplus(bias) lies between 1e-3 and 0.1."""
    rate = torch.exp(torch.rand(chan, generator=gen, device="cuda") * math.log(16.0))
    step = torch.exp(torch.rand(chan, generator=gen, device="cuda") * math.log(100.0) + math.log(1e-3))
    bias = step + torch.log(-torch.expm1(-step))
    return -rate * torch.nn.functional.softplus(0.5 * _normal(gen, *shape, chan) + bias)


def _sequence_rows(lens):
    """(first row of each sequence, rows in all)."""
    first, total = [], 0
    for n in lens:
        first.append(total)
        total += n
    return first, total


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    op, s = case["op"], dict(case)
    if op == "pool":
        rows = case["rows"]
        inner = case["heads"] * max(case["key"], case["value"])
        s["tensors"] = [_normal(gen, rows, case["heads"], case["key"], case["value"])] + \
            [_normal(gen, rows, TAPS - 1, inner) for _ in range(3)]
        s["index"] = torch.tensor(_pool_index(case), dtype=torch.int32, device="cuda")
        return s
    dt = DTYPES[case["x"]]
    train = case["train"]
    if op == "norm":
        rows, groups, width = case["rows"], case["groups"], case["width"]
        chan = groups * width
        # activations with a mean and a scale of their own in each group, as a recurrence hands them over
        scale = torch.exp(_normal(gen, groups, 1))
        s["x"] = ((_normal(gen, rows, groups, width) + 0.3 * _normal(gen, groups, 1)) * scale).reshape(rows, chan).to(dt)
        s["gate"] = _normal(gen, rows, chan, dtype=dt) if case["gate"] else None
        wide = {"channel": chan, "group": width, "none": 0}[case["affine"]]
        s["weight"] = 1 + 0.2 * _normal(gen, wide) if wide else None
        s["bias"] = 0.2 * _normal(gen, wide) if wide and case["bias"] else None
        s["eps"] = 1e-5
        s["inputs"] = [s["x"]] + [t for t in (s["gate"], s["weight"], s["bias"]) if t is not None]
        if train:
            s["d_out"] = _normal(gen, rows, chan, dtype=dt)
            for t in s["inputs"]:
                t.requires_grad_(True)
        return s
    lens, chan = _lengths(case), case["chan"]
    first, total = _sequence_rows(lens)
    packed = bool(case["lens"])
    shape = (1, total) if packed else (case["batch"], case["len"])
    s["cu"] = torch.tensor(first + [total], dtype=torch.int32, device="cuda") if packed else None
    s["x"] = _normal(gen, *shape, chan, dtype=dt)
    if op == "scan":
        s["g"] = _decay(gen, chan, *shape).to(DTYPES[case["g"]])
        s["state0"] = _normal(gen, len(lens), chan) if case["state"] else None
        s["d_state"] = _normal(gen, len(lens), chan) if train else None
        s["inputs"] = [s["x"], s["g"]] + ([s["state0"]] if case["state"] else [])
        rows = torch.zeros(shape[0] * shape[1], dtype=torch.bool, device="cuda")
        rows[[r for r, n in zip(first, lens) if n]] = True
        s["starts"] = rows.reshape(*shape, 1) if packed else None
    else:
        s["weight"] = torch.rand(chan, TAPS, generator=gen, device="cuda") - 0.5
        s["cache0"] = _normal(gen, len(lens), TAPS - 1, chan) if case["cache"] else None
        s["d_cache"] = _normal(gen, len(lens), TAPS - 1, chan) if train else None
        s["inputs"] = [s["x"], s["weight"]] + ([s["cache0"]] if case["cache"] else [])
        s["rows"], s["tail"] = (t.cuda() for t in _tap_rows(lens, case["cache"]))
    # sequences that hold a token, and their last rows
    s["live"] = torch.tensor([i for i, n in enumerate(lens) if n], device="cuda")
    s["first"] = torch.tensor([r for r, n in zip(first, lens) if n], device="cuda")
    s["last"] = torch.tensor([r + n - 1 for r, n in zip(first, lens) if n], device="cuda")
    if train:
        s["d_out"] = _normal(gen, *shape, chan, dtype=dt)
        for t in s["inputs"]:
            t.requires_grad_(True)
    return s


def _pool_index(case):
    """Where each row of the pool comes from: its old row, -1 for a row that is freed."""
    rows, how = case["rows"], case["how"]
    index = list(range(rows))
    if how == "fork":  # the first sequence's state goes to the second quarter of the pool, the last row is freed
        for d in range(rows // 4, rows // 2):
            index[d] = 0
        index[-1] = -1 if rows > 1 else 0
    elif how == "compact":  # every third sequence has ended: the last live ones move into the holes
        ended = [d for d in range(rows) if d % 3 == 1]
        live = [d for d in range(rows) if d % 3 != 1]
        for hole in ended:
            if hole >= len(live):
                break
            index[hole] = live.pop()
    else:  # every row changes its place: a turn of the whole pool
        index = [(d * 1 + 1) % rows for d in range(rows)]
    return index


def _tap_rows(lens, cached):
    """Row numbers, in a table of [cache rows; token rows; one row of zeros],
    that each token's taps read, and that the next cache keeps."""
    ahead = (TAPS - 1) * len(lens) if cached else 0
    first, total = _sequence_rows(lens)
    taps, tails = [], []
    for i, (start, n) in enumerate(zip(first, lens)):
        at = torch.arange(n + 1)[:, None] + torch.arange(TAPS)[None, :] - (TAPS - 1)
        if cached:
            before = i * (TAPS - 1) + at + (TAPS - 1)
        else:  # without a cache a sequence starts from copies of its own first token
            before = torch.full_like(at, ahead + start if n else ahead + total)
        at = torch.where(at < 0, before, ahead + start + at)
        taps.append(at[:n])
        tails.append(at[n, :TAPS - 1])
    return torch.cat(taps), torch.stack(tails)


# -- one pass ----------------------------------------------------------------


def run(state):
    s = state
    if own:
        return _run_own(s)
    return {"scan": _scan, "norm": _norm, "conv": _conv, "pool": _pool}[s["op"]](s)


def _gradients(s, outs, d_outs):
    return list(torch.autograd.grad(outs, s["inputs"], d_outs))


def _run_own(s):
    bg = _package()
    if s["op"] == "pool":
        bg.reorder_states(s["tensors"], s["index"])
        return s["tensors"]
    if s["op"] == "norm":
        y = bg.group_norm_gate(s["x"], s["gate"], s["weight"], s["bias"], num_groups=s["groups"], eps=s["eps"],
                               center=s["center"])
        return [y.detach()] + _gradients(s, [y], [s["d_out"]]) if s["train"] else [y]
    if s["op"] == "scan":
        h, last = bg.gated_scan(s["x"], s["g"], s["state0"], cu_seqlens=s["cu"], complement=s["complement"])
        grads = _gradients(s, [h, last], [s["d_out"], s["d_state"]]) if s["train"] else []
        return [h.detach(), last.detach()] + grads
    y, cache = bg.causal_conv_silu(s["x"], s["weight"], s["cache0"], cu_seqlens=s["cu"])
    grads = _gradients(s, [y, cache], [s["d_out"], s["d_cache"]]) if s["train"] else []
    return [y.detach(), cache.detach()] + grads


def _doubling(a, h, reverse):
    """h_t + a_t h_{t-1} + a_t a_{t-1} h_{t-2} + ... along dim 1 (from the other
    end with reverse): spans of 1, 2, 4, ... tokens joined, log2(T) steps."""
    if reverse:
        a, h = a.flip(1), h.flip(1)
    span, length = 1, a.shape[1]
    while span < length:
        h = torch.cat((h[:, :span], h[:, span:] + a[:, span:] * h[:, :-span]), 1)
        a = torch.cat((a[:, :span], a[:, span:] * a[:, :-span]), 1)
        span *= 2
    return h.flip(1) if reverse else h


@torch.no_grad()
def _scan(s):
    x, g = s["x"].float(), s["g"].float()
    shape, chan = x.shape, x.shape[2]
    a = torch.exp(g)
    scale = -torch.expm1(g) if s["complement"] else None
    u = x * scale if s["complement"] else x
    flat = lambda t: t.reshape(-1, chan)  # noqa: E731
    entering = torch.zeros(shape[0] if s["cu"] is None else len(s["cu"]) - 1, chan, device=x.device)
    if s["state0"] is not None:
        entering = s["state0"].float()
    if s["starts"] is None:
        u = torch.cat((u[:, :1] + a[:, :1] * entering[:, None], u[:, 1:]), 1)
        kept = a
    else:  # a sequence's first token takes its own state in place of its neighbour's
        u = u.clone()
        flat(u)[s["first"]] += flat(a)[s["first"]] * entering[s["live"]]
        kept = a * ~s["starts"]
    h = _doubling(kept, u, False)
    last = entering.clone()
    last[s["live"]] = flat(h)[s["last"]]
    out = [h.to(s["x"].dtype), last]
    if not s["train"]:
        return out
    d_h = s["d_out"].float().clone()
    flat(d_h)[s["last"]] += s["d_state"][s["live"]]
    after = torch.cat((kept[:, 1:], torch.zeros_like(kept[:, :1])), 1)
    lam = _doubling(after, d_h, True)
    before = torch.cat((torch.zeros_like(h[:, :1]), h[:, :-1]), 1)
    flat(before)[s["first"]] = entering[s["live"]]
    d_x = lam * scale if s["complement"] else lam
    d_g = a * lam * (before - x if s["complement"] else before)
    out += [d_x.to(s["x"].dtype), d_g.to(s["g"].dtype)]
    if s["state0"] is not None:
        d_state = s["d_state"].clone()
        d_state[s["live"]] = flat(a)[s["first"]] * flat(lam)[s["first"]]
        out.append(d_state)
    return out


@torch.no_grad()
def _norm(s):
    groups, width = s["groups"], s["width"]
    per = lambda t: t.float().reshape(-1, groups, width)  # noqa: E731
    wide = lambda t: t.reshape(-1, width)  # [groups or 1, width]  # noqa: E731
    x = per(s["x"])
    if s["center"]:
        x = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"])
    n = x * rstd
    z = n if s["weight"] is None else n * wide(s["weight"])
    z = z if s["bias"] is None else z + wide(s["bias"])
    t = z if s["gate"] is None else per(s["gate"])
    sig = 1 / (1 + torch.exp(-t))
    act = t * sig
    y = act if s["gate"] is None else z * act
    out = [y.reshape(s["x"].shape).to(s["x"].dtype)]
    if not s["train"]:
        return out
    d = per(s["d_out"])
    slope = sig * (1 + t * (1 - sig))
    d_z = d * (slope if s["gate"] is None else act)
    d_n = d_z if s["weight"] is None else d_z * wide(s["weight"])
    d_x = d_n - n * (d_n * n).mean(-1, keepdim=True)
    if s["center"]:
        d_x = d_x - d_n.mean(-1, keepdim=True)
    out.append((d_x * rstd).reshape(s["x"].shape).to(s["x"].dtype))
    if s["gate"] is not None:
        out.append((d * z * slope).reshape(s["x"].shape).to(s["x"].dtype))
    over = (0, 1) if s["affine"] == "group" else (0,)
    if s["weight"] is not None:
        out.append((d_z * n).sum(over).reshape(s["weight"].shape))
    if s["bias"] is not None:
        out.append(d_z.sum(over).reshape(s["bias"].shape))
    return out


@torch.no_grad()
def _conv(s):
    x, w = s["x"].float(), s["weight"].float()
    chan = x.shape[2]
    ahead = [] if s["cache0"] is None else [s["cache0"].reshape(-1, chan)]
    table = torch.cat(ahead + [x.reshape(-1, chan), torch.zeros(1, chan, device=x.device)])
    taps = table[s["rows"]]  # [tokens, TAPS, chan]
    pre = (taps * w.t()).sum(1)
    sig = 1 / (1 + torch.exp(-pre))
    out = [(pre * sig).reshape(x.shape).to(s["x"].dtype), table[s["tail"]]]
    if not s["train"]:
        return out
    d_pre = s["d_out"].float().reshape(-1, chan) * sig * (1 + pre * (1 - sig))
    d_table = torch.zeros_like(table)
    d_table.index_add_(0, s["rows"].reshape(-1), (d_pre[:, None] * w.t()).reshape(-1, chan))
    d_table.index_add_(0, s["tail"].reshape(-1), s["d_cache"].reshape(-1, chan))
    held = 0 if s["cache0"] is None else (TAPS - 1) * s["cache0"].shape[0]
    out.append(d_table[held:-1].reshape(x.shape).to(s["x"].dtype))
    out.append((taps * d_pre[:, None]).sum(0).t().contiguous())
    if s["cache0"] is not None:
        out.append(d_table[:held].reshape(s["cache0"].shape))
    return out


@torch.no_grad()
def _pool(s):
    source = s["index"].long()
    freed = source < 0
    for t in s["tensors"]:
        moved = t.index_select(0, source.clamp(min=0))
        moved[freed] = 0
        t.copy_(moved)
    return s["tensors"]


# -- what a pass cannot do without ---------------------------------------------


def work(case):
    """Inputs read once, outputs written once; arithmetic in multiplications,
    additions and functions."""
    size = lambda n: 2 if n == "bf16" else 4  # noqa: E731
    if case["op"] == "pool":
        index = _pool_index(case)
        row = 4 * (case["heads"] * case["key"] * case["value"]
                   + 3 * (TAPS - 1) * case["heads"] * max(case["key"], case["value"]))
        sources = {i for d, i in enumerate(index) if i >= 0 and i != d}
        return {"bytes": row * (len(sources) + sum(i != d for d, i in enumerate(index))) + 4 * len(index), "flops": 0}
    x, train = size(case["x"]), case["train"]
    if case["op"] == "norm":
        n = case["rows"] * case["groups"] * case["width"]
        small = {"channel": case["groups"] * case["width"], "group": case["width"], "none": 0}[case["affine"]]
        small *= 4 * (2 if case["bias"] else 1) * (2 if train else 1)
        tensors = 2 + case["gate"] + (2 + case["gate"] if train else 0)
        return {"bytes": n * x * tensors + small, "flops": n * (14 + (24 if train else 0))}
    lens, chan = _lengths(case), case["chan"]
    n = sum(lens) * chan
    if case["op"] == "scan":
        g = size(case["g"])
        states = 4 * len(lens) * chan * (1 + case["state"] + (1 + case["state"] if train else 0))
        per = 2 * x + g + (2 * x + g if train else 0)
        return {"bytes": n * per + states, "flops": n * (12 + (16 if train else 0))}
    caches = 4 * len(lens) * (TAPS - 1) * chan * (1 + case["cache"] + (1 + case["cache"] if train else 0))
    return {"bytes": n * x * (4 if train else 2) + caches + 4 * chan * TAPS * (2 if train else 1),
            "flops": n * (2 * TAPS + 6 + (6 * TAPS + 8 if train else 0))}


# -- 64 bits -------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"scan": _exact_scan, "norm": _exact_norm, "conv": _exact_conv, "pool": _exact_pool}[case["op"]](case, s)


def _exact_scan(case, s):
    """The recurrence and its adjoint, one token after the other."""
    f64 = lambda t: None if t is None else t.detach().double()  # noqa: E731
    x, g, state, d_out, d_state = (f64(s.get(n)) for n in ("x", "g", "state0", "d_out", "d_state"))
    lens, chan = _lengths(case), case["chan"]
    count, train, comp = len(lens), case["train"], case["complement"]
    if count * max(lens) * chan > 1 << 28 or max(sum(lens) if case["lens"] else max(lens), 1) > 70000:
        return None
    batch, length = x.shape[:2]
    # the tokens as columns [T, B, C]; sequence number and place in it of each column's entries
    x, g = x.transpose(0, 1).contiguous(), g.transpose(0, 1).contiguous()
    a, weight = g.exp(), (-torch.expm1(g) if comp else torch.ones_like(g))
    del g
    start = state if state is not None else x.new_zeros(count, chan)
    opens, closes = {}, {}
    if case["lens"]:
        at = 0
        for i, n in enumerate(lens):
            if n:
                opens[at], closes[at + n - 1] = i, i
            at += n
    else:
        opens[0] = closes[length - 1] = slice(None)
    h, ends = torch.empty_like(x), start.clone()
    now = None
    for t in range(length):
        if t in opens:
            now = start[opens[t]].reshape(batch, chan)
        now = torch.addcmul(weight[t] * x[t], a[t], now)
        h[t] = now
        if t in closes:
            ends[closes[t]] = now.reshape(ends[closes[t]].shape)
    out = [h.transpose(0, 1), ends]
    if not train:
        return out
    d_out = d_out.transpose(0, 1)
    lam, d_start, flow = torch.empty_like(x), d_state.clone(), None
    before = torch.cat((x.new_zeros(1, batch, chan), h[:-1]))
    for t in opens:
        before[t] = start[opens[t]].reshape(batch, chan)
    for t in range(length - 1, -1, -1):
        if t in closes:
            flow = d_state[closes[t]].reshape(batch, chan)
        now = d_out[t] + flow
        lam[t] = now
        flow = a[t] * now
        if t in opens:
            d_start[opens[t]] = flow.reshape(d_start[opens[t]].shape)
    d_x = lam * weight
    d_g = lam * a * (before - x if comp else before)
    out += [d_x.transpose(0, 1), d_g.transpose(0, 1)]
    return out + ([d_start] if state is not None else [])


def _leaf(t):
    return None if t is None else t.detach().double().requires_grad_(True)


def _exact_norm(case, s):
    x, gate, weight, bias = (_leaf(s[n]) for n in ("x", "gate", "weight", "bias"))
    groups, width = case["groups"], case["width"]
    v = x.reshape(-1, groups, width)
    var, mean = torch.var_mean(v, dim=-1, unbiased=False, keepdim=True)
    z = (v - mean) / (var + s["eps"]).sqrt() if case["center"] else v / (var + mean * mean + s["eps"]).sqrt()
    if weight is not None:
        z = z * weight.reshape(-1, width)
    if bias is not None:
        z = z + bias.reshape(-1, width)
    z = z.reshape(x.shape)
    y = torch.nn.functional.silu(z) if gate is None else z * torch.nn.functional.silu(gate)
    if not case["train"]:
        return [y.detach()]
    leaves = [t for t in (x, gate, weight, bias) if t is not None]
    return [y.detach()] + list(torch.autograd.grad(y, leaves, s["d_out"].double()))


def _exact_conv(case, s):
    """A library convolution over each sequence with its three tokens in front."""
    x, weight, cache = (_leaf(s[n]) for n in ("x", "weight", "cache0"))
    lens, chan, rows = _lengths(case), case["chan"], x.reshape(-1, x.shape[2])
    ys, tails, at = [], [], 0
    for i, n in enumerate(lens):
        part = rows[at:at + n]
        if cache is not None:
            front = cache[i]
        else:
            front = part[:1].expand(TAPS - 1, chan) if n else x.new_zeros(TAPS - 1, chan)
        line = torch.cat((front, part))
        if n:
            ys.append(torch.nn.functional.conv1d(line.t()[None], weight[:, None], groups=chan)[0].t())
        tails.append(line[n:])
        at += n
    y = torch.nn.functional.silu(torch.cat(ys)).reshape(x.shape)
    tail = torch.stack(tails)
    if not case["train"]:
        return [y.detach(), tail.detach()]
    leaves = [t for t in (x, weight, cache) if t is not None]
    grads = torch.autograd.grad([y, tail], leaves, [s["d_out"].double(), s["d_cache"].double()])
    return [y.detach(), tail.detach()] + list(grads)


def _exact_pool(case, s):
    """The rows one by one."""
    out = []
    for t in s["tensors"]:
        new = t.double()
        for row, source in enumerate(_pool_index(case)):
            new[row] = t[source].double() if source >= 0 else 0.0
        out.append(new)
    return out

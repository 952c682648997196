"""Measured calls of the attention block's operators: rotary positions, the norms of queries and
keys with the rotation in the same pass, and attention with a sliding window and a few first
tokens that stay visible.

`own` chooses what `run` computes with: the plain formulas in elementary torch operations (false)
or the calls that a user makes of spar_b200.ops (true). Heads are addressed as
[batch, tokens, heads, head_dim] views of the packed projection [batch, tokens, (H + 2 K) D].
"""
import math

import torch

own = False

DEVICE = "cuda"
FLOAT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # One new token of eight sequences on its way into the cache: launch latency.
        dict(name="rotate one token", op="rotary", dtype="bfloat16", batch=8, seq=1, heads=16, kv=4,
             dim=64, rotary=64, layout="half", inverse=False, positions=True, rows=4096),
        # The benchmark decoder's packed projection (16 x 1024 tokens, 16 heads of 64), fp32.
        dict(name="rotate the projection", op="rotary", dtype="float32", batch=16, seq=1024, heads=16,
             kv=16, dim=64, rotary=64, layout="interleaved", inverse=False, positions=False,
             rows=1024),
        # Gradients of a long ragged batch, half of each head rotated, packed positions.
        dict(name="rotate back part of a head", op="rotary", dtype="bfloat16", batch=3, seq=8191,
             heads=32, kv=8, dim=128, rotary=64, layout="half", inverse=True, positions=True,
             rows=32768),
        # The angle table of a context stretched by eight.
        dict(name="table for a long context", op="table", rows=131072, rotary=128, theta=10000.0,
             start=0, scaling="parts", factor=8.0, original=16384),
        # Query and key norms of one new token of sixteen sequences.
        dict(name="norm and rotate one token", op="norm", dtype="bfloat16", batch=16, seq=1, heads=16,
             kv=4, dim=64, rotary=64, layout="half", backward=False, positions=True, rows=8192),
        # The Spar family's projection at the benchmark decoder's widths.
        dict(name="norm and rotate forward", op="norm", dtype="float32", batch=16, seq=1024, heads=16,
             kv=16, dim=64, rotary=64, layout="interleaved", backward=False, positions=False,
             rows=1024),
        # Its backward at a long odd length, grouped heads of 128.
        dict(name="norm and rotate backward", op="norm", dtype="bfloat16", batch=2, seq=4095, heads=32,
             kv=8, dim=128, rotary=128, layout="half", backward=True, positions=False, rows=4096),
        # One token of one sequence against a short fp32 cache (12 heads of 64).
        dict(name="one token, short cache", op="window", dtype="float32", batch=1, q_len=1, kv_len=1000,
             heads=12, kv=12, dim=64, window=256, sinks=4, ragged=0, backward=False, decode=True),
        # One token of each of 32 sequences against caches of different fill.
        dict(name="one token, long caches", op="window", dtype="bfloat16", batch=32, q_len=1,
             kv_len=16384, heads=32, kv=8, dim=128, window=4096, sinks=4, ragged=201, backward=False,
             decode=True),
        # A long prompt.
        dict(name="window forward, long", op="window", dtype="bfloat16", batch=1, q_len=8192,
             kv_len=8192, heads=32, kv=8, dim=128, window=1024, sinks=4, ragged=0, backward=False,
             decode=False),
        # A training pass, forward and backward, over grouped heads of 64.
        dict(name="window training", op="window", dtype="bfloat16", batch=2, q_len=4096, kv_len=4096,
             heads=16, kv=4, dim=64, window=512, sinks=4, ragged=0, backward=True, decode=False),
        # The same in fp32 at the benchmark decoder's widths with a padded batch of odd lengths.
        dict(name="window training, fp32", op="window", dtype="float32", batch=4, q_len=1023,
             kv_len=1023, heads=16, kv=16, dim=64, window=256, sinks=2, ragged=101, backward=True,
             decode=False),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    limit = max(_cost(c) for c in listed())
    op = rng.choice(["rotary", "table", "norm", "norm", "window", "window", "window"])
    while True:
        dtype = rng.choice(["float32", "bfloat16"])
        kv = rng.choice([1, 2, 4, 8, 12, 16])
        heads = kv * rng.choice([1, 2, 4, 8]) if kv < 12 else kv
        dim = rng.choice([32, 64, 64, 128, 128])
        if op == "table":
            scaling = rng.choice(["none", "linear", "base", "parts"])
            case = dict(op=op, rows=_log(rng, 16, 131072), rotary=rng.choice([16, 32, 64, 96, 128]),
                        theta=rng.choice([10000.0, 500000.0]), start=rng.choice([0, 0, 7, 4096]),
                        scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]),
                        original=rng.choice([2048, 8192]))
        elif op == "rotary":
            seq = _log(rng, 1, 8192)
            case = dict(op=op, dtype=dtype, batch=_log(rng, 1, 16), seq=seq, heads=heads, kv=kv, dim=dim,
                        rotary=dim if rng.random() < 0.6 else dim // 2,
                        layout=rng.choice(["interleaved", "half"]), inverse=rng.random() < 0.5,
                        positions=rng.random() < 0.5, rows=seq + _log(rng, 1, 4096))
        elif op == "norm":
            seq = _log(rng, 1, 8192)
            case = dict(op=op, dtype=dtype, batch=_log(rng, 1, 16), seq=seq, heads=heads, kv=kv, dim=dim,
                        rotary=dim if rng.random() < 0.6 else dim // 2,
                        layout=rng.choice(["interleaved", "half"]), backward=rng.random() < 0.5,
                        positions=rng.random() < 0.5, rows=seq + _log(rng, 1, 4096))
        else:
            decode = rng.random() < 0.35
            kv_len = _log(rng, 16, 16384 if decode else 8192)
            batch = _log(rng, 1, 32 if decode else 8)
            backward = not decode and rng.random() < 0.5
            case = dict(op=op, dtype=dtype, batch=batch, q_len=rng.choice([1, 1, 2, 5]) if decode else kv_len,
                        kv_len=kv_len, heads=heads, kv=kv, dim=dim, window=_log(rng, 16, 4096),
                        sinks=rng.choice([0, 1, 4, 4, 64]),
                        ragged=_log(rng, 1, max(1, kv_len // (2 * batch))) if rng.random() < 0.5 else 0,
                        backward=backward, decode=decode)
            # the plain form holds whole score matrices
            if batch * heads * case["q_len"] * kv_len > 32 * 8192 * 8192 // (4 if backward else 1):
                continue
        if _cost(case) <= limit:
            return case


# ------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Keys of each sequence: the whole capacity, less `ragged` more for each further one."""
    return [max(case["q_len"] if case["decode"] else 1, case["kv_len"] - b * case["ragged"])
            for b in range(case["batch"])]


def _frequencies(case):
    """Angle per position of each pair, float64, and the factor on cos and sin."""
    d, theta, factor = case["rotary"], case["theta"], case["factor"]
    i = torch.arange(d // 2, dtype=torch.float64, device=DEVICE)
    if case["scaling"] == "base":
        theta = theta * factor ** (d / (d - 2))
    f = theta ** (-2.0 * i / d)
    magnitude = 1.0
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "parts":
        turns = case["original"] * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        magnitude = 0.1 * math.log(factor) + 1.0
    return f, magnitude


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _heads_of(case, g, scale=1.0):
    """q, k, v views of a packed projection, as the model's product leaves them."""
    h, k, d = case["heads"], case["kv"], case["dim"]
    b, t = case["batch"], case.get("seq", case.get("kv_len"))
    packed = torch.randn(b, t, (h + 2 * k) * d, generator=g, device=DEVICE) * scale
    packed = packed.to(FLOAT[case["dtype"]])
    return (packed[..., :h * d].view(b, t, h, d), packed[..., h * d:(h + k) * d].view(b, t, k, d),
            packed[..., (h + k) * d:].view(b, t, k, d))


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    op = case["op"]
    if op == "table":  # its only input is the base
        s["theta"] = case["theta"] * (1.0 + 0.001 * (seed % 97))
        return s
    b = case["batch"]
    if op in ("rotary", "norm"):
        t, d = case["seq"], case["rotary"]
        s["q"], s["k"], _ = _heads_of(case, g, 1.0 if op == "rotary" else 2.0)
        f = 10000.0 ** (-2.0 * torch.arange(d // 2, dtype=torch.float64, device=DEVICE) / d)
        angle = torch.arange(case["rows"], dtype=torch.float64, device=DEVICE)[:, None] * f
        s["table"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
        s["positions"] = None
        if case["positions"]:
            first = torch.randint(0, case["rows"] - t + 1, (b, 1), generator=g, device=DEVICE)
            s["positions"] = (first + torch.arange(t, device=DEVICE)).to(torch.int32).contiguous()
        if op == "norm":
            s["wq"] = 1.0 + 0.2 * torch.randn(case["dim"], generator=g, device=DEVICE)
            s["wk"] = 1.0 + 0.2 * torch.randn(case["dim"], generator=g, device=DEVICE)
            if case["backward"]:
                s["dq"], s["dk"], _ = _heads_of(case, g)
        return s
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)
    if case["decode"]:
        h, k, d, t = case["heads"], case["kv"], case["dim"], case["q_len"]
        kind = FLOAT[case["dtype"]]
        s["q"] = torch.randn(b, t, h, d, generator=g, device=DEVICE).to(kind)
        s["k"] = torch.randn(b, case["kv_len"], k, d, generator=g, device=DEVICE).to(kind)
        s["v"] = torch.randn(b, case["kv_len"], k, d, generator=g, device=DEVICE).to(kind)
        s["lengths"], s["first"] = lengths, lengths - t
    else:
        s["q"], s["k"], s["v"] = _heads_of(case, g)
        s["lengths"], s["first"] = (lengths if case["ragged"] else None), None
        if case["backward"]:
            s["dout"] = torch.randn(b, case["q_len"], case["heads"], case["dim"], generator=g,
                                    device=DEVICE).to(FLOAT[case["dtype"]])
    return s


# ------------------------------------------------------------------------------------- plain forms
def _cos_sin(s, tokens):
    """cos, sin [batch or 1, tokens, 1, pairs] of each token."""
    if s["positions"] is not None:
        row = s["table"][s["positions"].long()]
    else:
        row = s["table"][:tokens][None]
    return row[:, :, None, :, 0], row[:, :, None, :, 1]


def _rotate(x, cos, sin, rotary, layout):
    """Pairs of the first `rotary` elements turned by their angle; the rest as it is."""
    r = x[..., :rotary]
    if layout == "half":
        a, b = r[..., :rotary // 2], r[..., rotary // 2:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, x[..., rotary:]], -1)


EPS = 1e-6


def _norm_backward(x, w, g):
    """Gradients of x / sqrt(mean(x^2) + eps) * w for the gradient g: (dx, dw)."""
    inv = 1.0 / ((x * x).mean(-1, keepdim=True) + EPS).sqrt()
    unit = x * inv
    gw = g * w
    return inv * (gw - unit * (gw * unit).mean(-1, keepdim=True)), (g * unit).flatten(0, 2).sum(0)


def _visible(case, s):
    """[batch or 1, 1, q_len, kv_len]: key j is seen from position p iff j <= p and it is within
    the window or among the first `sinks`; neither p nor j reaches a sequence's length."""
    dev = s["q"].device
    p = torch.arange(case["q_len"], device=dev)[None, :, None]
    if s["first"] is not None:
        p = p + s["first"].long()[:, None, None]
    j = torch.arange(case["kv_len"], device=dev)[None, None, :]
    see = (j <= p) & ((j > p - case["window"]) | (j < case["sinks"]))
    if s["lengths"] is not None:
        n = s["lengths"].long()[:, None, None]
        see = see & (j < n) & (p < n)
    return see[:, None]


def _window_plain(s):
    case = s["case"]
    group = case["heads"] // case["kv"]
    q = s["q"].float().transpose(1, 2)
    k = s["k"].float().transpose(1, 2).repeat_interleave(group, 1)
    v = s["v"].float().transpose(1, 2).repeat_interleave(group, 1)
    scale = 1.0 / math.sqrt(case["dim"])
    see = _visible(case, s)
    score = (q @ k.transpose(-1, -2) * scale).masked_fill_(~see, -math.inf)
    top = score.amax(-1, keepdim=True)
    base = torch.where(top == -math.inf, 0.0, top)
    p = (score - base).exp_()
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ v
    got = {"out": out.transpose(1, 2).to(s["q"].dtype).contiguous(),
           "lse": (total.log() + base)[..., 0]}
    if not case["backward"]:
        return got
    do = s["dout"].float().transpose(1, 2)
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (do * out).sum(-1, keepdim=True)) * scale
    b, n, d = case["batch"], case["kv_len"], case["dim"]
    for name, full in (("dq", ds @ k), ("dk", ds.transpose(-1, -2) @ q), ("dv", p.transpose(-1, -2) @ do)):
        if name != "dq":
            full = full.view(b, case["kv"], group, n, d).sum(2)
        got[name] = full.transpose(1, 2).to(s["q"].dtype).contiguous()
    return got


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "table":
        f, magnitude = _frequencies(dict(case, theta=s["theta"]))
        pos = torch.arange(case["rows"], dtype=torch.float64, device=DEVICE) + case["start"]
        angle = pos[:, None] * f
        return torch.stack([angle.cos() * magnitude, angle.sin() * magnitude], -1).float()
    if op == "window":
        return _window_plain(s)
    cos, sin = _cos_sin(s, case["seq"])
    kind, n, layout = s["q"].dtype, case["rotary"], case["layout"]
    if op == "rotary":
        sin = -sin if case["inverse"] else sin
        return {"q": _rotate(s["q"].float(), cos, sin, n, layout).to(kind),
                "k": _rotate(s["k"].float(), cos, sin, n, layout).to(kind)}
    got = {}
    for name in ("q", "k"):
        x, w = s[name].float(), s["w" + name]
        if case["backward"]:
            g = _rotate(s["d" + name].float(), cos, -sin, n, layout)
            dx, got["dw" + name] = _norm_backward(x, w, g)
            got["d" + name] = dx.to(kind)
        else:
            y = x * (1.0 / ((x * x).mean(-1, keepdim=True) + EPS).sqrt()) * w
            got[name] = _rotate(y, cos, sin, n, layout).to(kind)
    return got


# ------------------------------------------------------------------------------------- own calls
def _own(s):
    from spar_b200 import ops

    case = s["case"]
    op = case["op"]
    if op == "table":
        scaling = None
        if case["scaling"] != "none":
            scaling = ops.RotaryScaling(case["scaling"], case["factor"], case["original"])
        return ops.rotary_table(case["rows"], case["rotary"], s["theta"], case["start"], scaling,
                                device=DEVICE)
    if op == "rotary":
        q, k = ops.rotary(s["q"], s["k"], s["table"], layout=case["layout"], positions=s["positions"],
                          inverse=case["inverse"])
        return {"q": q, "k": k}
    if op == "norm":
        if not case["backward"]:
            q, k = ops.qk_norm_rotary_forward(s["q"], s["k"], s["wq"], s["wk"], s["table"], EPS,
                                              layout=case["layout"], positions=s["positions"])
            return {"q": q, "k": k}
        dq, dk, dwq, dwk = ops.qk_norm_rotary_backward(
            s["dq"], s["dk"], s["q"], s["k"], s["wq"], s["wk"], s["table"], EPS,
            layout=case["layout"], positions=s["positions"])
        return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    where = {"window": case["window"], "sinks": case["sinks"], "lengths": s["lengths"],
             "first": s["first"]}
    out, lse = ops.window_attention_forward(s["q"], s["k"], s["v"], **where)
    got = {"out": out, "lse": lse}
    if case["backward"]:
        got["dq"], got["dk"], got["dv"] = ops.window_attention_backward(
            s["dout"], s["q"], s["k"], s["v"], out, lse, **where)
    return got


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------- work
def _up_to(x, most):
    """The sum of min(p + 1, most) over positions 0 <= p < x."""
    m = min(x, most)
    return m * (m + 1) // 2 + (x - m) * most


def _pairs_and_keys(case):
    """Visible (query, key) pairs of one head over the batch, and the keys that some query sees."""
    pairs = keys = 0
    w, sinks = case["window"], case["sinks"]
    for n in _lengths(case):
        lo = n - case["q_len"] if case["decode"] else 0
        pairs += _up_to(n, w) - _up_to(lo, w)
        pairs += _up_to(max(0, n - w), sinks) - _up_to(max(0, lo - w), sinks)  # behind the window
        start = max(0, lo - w + 1)
        keys += n - start + min(sinks, start)
    return pairs, keys


def work(case):
    if case["op"] == "table":
        n = case["rows"] * case["rotary"] // 2
        return {"bytes": 8.0 * n, "flops": 4.0 * n}
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] in ("rotary", "norm"):
        tokens = case["batch"] * case["seq"]
        n = tokens * (case["heads"] + case["kv"]) * case["dim"]
        table = 4.0 * case["rotary"] * (tokens if case["positions"] else case["seq"])
        table += 4.0 * tokens if case["positions"] else 0.0
        if case["op"] == "rotary":
            return {"bytes": 2.0 * n * size + table, "flops": 3.0 * n}
        back = case["backward"]
        return {"bytes": (3.0 if back else 2.0) * n * size + table + (16.0 if back else 8.0) * case["dim"],
                "flops": (14.0 if back else 7.0) * n}
    pairs, keys = _pairs_and_keys(case)
    h, d = case["heads"], case["dim"]
    rows = case["batch"] * case["q_len"] * h
    moved = 2.0 * rows * d * size + 2.0 * keys * case["kv"] * d * size + 4.0 * rows
    flops = 4.0 * pairs * h * d
    if case["backward"]:
        moved += 2.0 * rows * d * size + 2.0 * case["batch"] * case["kv_len"] * case["kv"] * d * size
        flops += 10.0 * pairs * h * d
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------------------- 64 bits
def _turn(case):
    """Index of each element's partner and its sign in y = x cos + sign x[partner] sin, and the
    pair that each element belongs to."""
    n, d = case["rotary"], case["dim"]
    partner, sign, pair = list(range(d)), [0.0] * d, [0] * d
    for i in range(n // 2):
        a, b = (i, i + n // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
        partner[a], partner[b], sign[a], sign[b], pair[a], pair[b] = b, a, -1.0, 1.0, i, i
    return (torch.tensor(partner, device=DEVICE), torch.tensor(sign, dtype=torch.float64, device=DEVICE),
            torch.tensor(pair, device=DEVICE))


def _turned(x, case, angles, back):
    partner, sign, pair = _turn(case)
    moved = (sign != 0).double()
    cos = angles[:, :, None, :, 0][..., pair] * moved + (1.0 - moved)
    sin = angles[:, :, None, :, 1][..., pair] * sign
    return x * cos + x[..., partner] * (-sin if back else sin)


def _exact_window(s):
    case = s["case"]
    group, scale = case["heads"] // case["kv"], case["dim"] ** -0.5
    back = case["backward"]
    names = ["q", "k", "v"]
    full = {n: s[n].double() for n in names}
    out = torch.zeros(full["q"].shape, dtype=torch.float64, device=DEVICE)
    lse = torch.full((case["batch"], case["heads"], case["q_len"]), -math.inf, dtype=torch.float64,
                     device=DEVICE)
    grad = {n: torch.zeros_like(full[n]) for n in names}
    lengths = _lengths(case) if s["lengths"] is not None else [case["kv_len"]] * case["batch"]
    for b in range(case["batch"]):
        n = lengths[b]
        first = n - case["q_len"] if case["decode"] else 0
        rows = min(case["q_len"], n - first)
        p = torch.arange(first, first + rows, device=DEVICE)
        j = torch.arange(n, device=DEVICE)
        age = p[:, None] - j[None, :]
        hidden = (age < 0) | ((age >= case["window"]) & (j[None, :] >= case["sinks"]))
        for h in range(case["heads"]):
            qh = full["q"][b, :rows, h].clone().requires_grad_(back)
            kh = full["k"][b, :n, h // group].clone().requires_grad_(back)
            vh = full["v"][b, :n, h // group].clone().requires_grad_(back)
            score = torch.einsum("id,jd->ij", qh, kh).mul(scale).masked_fill(hidden, -math.inf)
            o = torch.einsum("ij,jd->id", torch.softmax(score, -1), vh)
            out[b, :rows, h] = o.detach()
            lse[b, h, :rows] = torch.logsumexp(score.detach(), -1)
            if back:
                o.backward(s["dout"][b, :rows, h].double())
                grad["q"][b, :rows, h] += qh.grad
                grad["k"][b, :n, h // group] += kh.grad
                grad["v"][b, :n, h // group] += vh.grad
    got = {"out": out, "lse": lse}
    if back:
        got.update({"d" + n: grad[n] for n in names})
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "table":
        # numpy's long double would cost seconds here; 64 bits leave 1e-11 of the farthest angle
        f, magnitude = _frequencies(dict(case, theta=s["theta"]))
        turn = torch.outer(torch.arange(case["start"], case["start"] + case["rows"], device=DEVICE).double(),
                           f / (2 * math.pi))
        turn = (turn - turn.floor()) * (2 * math.pi)
        return torch.stack([torch.sin(turn + math.pi / 2), torch.sin(turn)], -1) * magnitude
    if case["op"] == "window":
        return _exact_window(s)
    t = case["seq"]
    if s["positions"] is None:
        angles = s["table"][:t].double()[None]
    else:
        angles = s["table"].double()[s["positions"].long()]
    got = {}
    for name in ("q", "k"):
        x = s[name].double()
        if case["op"] == "rotary":
            got[name] = _turned(x, case, angles, case["inverse"])
            continue
        x.requires_grad_(case["backward"])
        w = s["w" + name].double().requires_grad_(case["backward"])
        y = _turned(torch.nn.functional.rms_norm(x, (case["dim"],), eps=EPS) * w, case, angles, False)
        if not case["backward"]:
            got[name] = y
            continue
        y.backward(s["d" + name].double())
        got["d" + name], got["dw" + name] = x.grad, w.grad
    return got

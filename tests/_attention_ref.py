"""Plain 64-bit forms of the attention block's operators (rotation, qk-norm, window attention) with
their gradients, and what an implementation in fewer bits may be off by, element by element.

Error model. u = 2^-24 is half a step of fp32, h = eps(type) / 2 half a step of the stored type
(2^-8 for bf16, u for fp32). All sums are in fp32.
"""
import torch

U = 2.0 ** -24
TINY = 2.0 ** -126  # a weight exp(s - lse) below the smallest normal fp32 may become zero, so every
                    # weight, and every stored value, may be off by this much whatever its size


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------- rotation
def rotate(x, angles, rotary, layout, sign=1.0):
    """x [B, T, H, D] float64, angles [B or 1, T, rotary / 2, 2] (cos, sin)."""
    c, s = angles[:, :, None, :, 0], angles[:, :, None, :, 1] * sign
    y = x.clone()
    if layout == "half":
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        y[..., :rotary // 2], y[..., rotary // 2:rotary] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        y[..., 0:rotary:2], y[..., 1:rotary:2] = a * c - b * s, b * c + a * s
    return y


def norm_rotate(x, w, angles, rotary, layout, eps):
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return rotate(x * r * w, angles, rotary, layout)


def norm_rotate_backward(dy, x, w, angles, rotary, layout, eps):
    """(dx, dw, and the sums of magnitudes that bound their rounding errors)."""
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    u = x * r
    g = rotate(dy, angles, rotary, layout, -1.0)
    gw = g * w
    dx = r * (gw - u * (gw * u).mean(-1, keepdim=True))
    # |g| from its two terms, so that cancellation in the rotation counts
    ga = rotate(dy.abs(), angles.abs(), rotary, layout, -1.0).abs() + rotate(dy.abs(), angles.abs(),
                                                                             rotary, layout).abs()
    size = r * (ga * w.abs() + u.abs() * (ga * w.abs() * u.abs()).mean(-1, keepdim=True))
    return dx, (g * u).sum((0, 1, 2)), size, (ga * u.abs()).sum((0, 1, 2))


# ------------------------------------------------------------------------------------- attention
def visible(q_len, kv_len, window, sinks, length, first):
    p = torch.arange(q_len)[:, None] + first
    j = torch.arange(kv_len)[None, :]
    return (j <= p) & ((j > p - window) | (j < sinks)) & (j < length) & (p < length)


def window_attention(q, k, v, window, sinks, scale=None, lengths=None, first=None, dout=None, h=U,
                     logit_u=48.0):
    """q [B, Q, H, D], k, v [B, K, KV, D], dout like q or None, float64.
    Returns ({name: value}, {name: bound}). `h`: half a step of the stored type, by which P and dS
    may be rounded before their products too. `logit_u`: error of scale q.k in units of
    u * scale * sum |q| |k| (a sum of at most 256 products in any order of pieces of 16 is off by
    at most 16 + 16 units; a tensor core that cuts instead of rounding doubles the second half).
    """
    B, Q, H, D = q.shape
    K, KV = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    val = {"out": torch.zeros_like(q), "lse": torch.full((B, H, Q), -float("inf"), dtype=q.dtype)}
    off = {"out": torch.zeros_like(q), "lse": torch.zeros(B, H, Q, dtype=q.dtype)}
    if dout is not None:
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            val[n], off[n] = torch.zeros_like(t), torch.zeros_like(t)
    for b in range(B):
        n = K if lengths is None else min(max(int(lengths[b]), 0), K)
        f = K - Q if first is None else int(first[b])
        see = visible(Q, n, window, sinks, n, f)
        rows = see.any(1)
        if not rows.any():
            continue
        see = see[rows]
        for a in range(H):
            g = a // (H // KV)
            qq, kk, vv = q[b, rows, a], k[b, :n, g], v[b, :n, g]
            s = (qq @ kk.T * scale).masked_fill(~see, -float("inf"))
            lse = torch.logsumexp(s, -1)
            p = torch.exp(s - lse[:, None])
            o = p @ vv
            ds = torch.where(see, logit_u * U * scale * (qq.abs() @ kk.abs().T), 0.0)
            es = ds.amax(-1) + 16 * U * (1 + lse.abs())      # a row's logits, its max and its sum
            pv = p @ vv.abs()
            # 2 es: weights off by exp(es) each, and the sum; cut accumulators and the divide: 64 u
            eo = h * o.abs() + (h + 2 * es[:, None] + 64 * U) * pv + TINY * (1 + see.double() @ vv.abs())
            val["out"][b, rows, a], off["out"][b, rows, a] = o, eo
            val["lse"][b, a, rows], off["lse"][b, a, rows] = lse, es + 4 * U
            if dout is None:
                continue
            do = dout[b, rows, a]
            dp = do @ vv.T
            delta = (do * o).sum(-1, keepdim=True)
            dS = p * (dp - delta)
            ep = 2 * es[:, None] * p + TINY * see            # P against the saved lse
            edp = logit_u * U * (do.abs() @ vv.abs().T)
            ed = (do.abs() * eo).sum(-1, keepdim=True) + logit_u * U * (do.abs() * o.abs()).sum(-1, keepdim=True)
            eS = h * dS.abs() + ep * (dp.abs() + delta.abs()) + p * (edp + ed) + 8 * U * p * (dp.abs() + delta.abs())
            eP = h * p + ep
            acc = 64 * U                                      # sums of the products themselves
            val["dq"][b, rows, a] = scale * dS @ kk
            off["dq"][b, rows, a] = scale * ((eS + acc * dS.abs()) @ kk.abs())
            val["dk"][b, :n, g] += scale * dS.T @ qq
            off["dk"][b, :n, g] += scale * ((eS + acc * dS.abs()).T @ qq.abs())
            val["dv"][b, :n, g] += p.T @ do
            off["dv"][b, :n, g] += (eP + acc * p).T @ do.abs()
    if dout is not None:
        for n in ("dq", "dk", "dv"):
            off[n] += h * val[n].abs() + TINY
    return val, off


def assert_within(got, want, bound, name=""):
    """|got - want| <= bound everywhere, infinities equal and no NaN; the largest ratio."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine]), name
    d = (got[fine] - want[fine]).abs()
    assert bool(torch.isfinite(d).all()), f"{name}: not finite"
    over = d > bound[fine] + 1e-300
    if over.any():
        worst = int((d / (bound[fine] + 1e-300)).argmax())
        raise AssertionError(f"{name}: {int(over.sum())} of {over.numel()} off, worst "
                             f"{float(d[worst]):.3g} against {float(bound[fine][worst]):.3g}")

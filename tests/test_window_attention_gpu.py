"""Attention with a sliding window and first tokens that stay visible, forward and backward, against
the 64-bit form, with element-wise bounds that follow from the roundings (see _attention_ref)."""
import math

import pytest
import torch

from _attention_ref import assert_within, half_step, window_attention

pytestmark = pytest.mark.gpu


def _packed(cuda, g, dtype, b, t, h, kv, d, offset=0):
    width = (h + 2 * kv) * d
    x = torch.randn(b * t * width + offset, generator=g, device=cuda).to(dtype)[offset:].view(b, t, width)
    return (x[..., :h * d].unflatten(-1, (h, d)), x[..., h * d:(h + kv) * d].unflatten(-1, (kv, d)),
            x[..., (h + kv) * d:].unflatten(-1, (kv, d)))


def _check(q, k, v, window, sinks, dout=None, **where):
    from spar_b200 import ops

    out, lse = ops.window_attention_forward(q, k, v, window, sinks, **where)
    got = {"out": out, "lse": lse}
    if dout is not None:
        got["dq"], got["dk"], got["dv"] = ops.window_attention_backward(dout, q, k, v, out, lse, window,
                                                                        sinks, **where)
    torch.cuda.synchronize()
    assert ops.attention_error() == 0
    want, bound = window_attention(
        *(x.double().cpu() for x in (q, k, v)), window, sinks, where.get("scale"), where.get("lengths"),
        where.get("first"), None if dout is None else dout.double().cpu(), half_step(q.dtype))
    for name in want:
        assert_within(got[name], want[name], bound[name], name)
    return got


SELF = [
    # b, t, heads, kv, dim, window, sinks
    (1, 1, 1, 1, 64, 1, 0),
    (2, 2, 2, 1, 64, 1, 1),
    (1, 5, 4, 2, 32, 3, 2),
    (2, 63, 2, 2, 64, 16, 4),
    (1, 128, 4, 1, 64, 128, 0),     # one tile
    (1, 129, 2, 1, 64, 64, 4),      # one row behind it
    (2, 200, 3, 1, 128, 50, 3),     # a group of three
    (1, 257, 2, 2, 128, 1000, 0),   # plain causal
    (1, 300, 2, 1, 64, 1, 0),       # each row sees itself
    (1, 300, 2, 1, 64, 1, 300),     # everything is a first token
    (1, 520, 4, 4, 32, 100, 130),   # first tokens over more than a tile
    (2, 513, 2, 1, 128, 127, 1),
    (1, 700, 2, 1, 64, 300, 64),
    (1, 150, 2, 1, 96, 40, 5),
    (1, 150, 2, 1, 80, 40, 5),
    (1, 140, 2, 2, 33, 20, 2),      # odd head: element by element
    (1, 70, 1, 1, 200, 30, 2),
    (1, 1400, 2, 1, 64, 200, 4),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SELF)
def test_self_attention(cuda, shape, dtype):
    b, t, h, kv, d, window, sinks = shape
    g = torch.Generator(device=cuda)
    g.manual_seed(t * 3 + d)
    q, k, v = _packed(cuda, g, dtype, b, t, h, kv, d)
    dout = torch.randn(b, t, h, d, generator=g, device=cuda).to(dtype)
    _check(q, k, v, window, sinks, dout)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [1, 4])
def test_rows_that_are_not_aligned(cuda, dtype, offset):
    g = torch.Generator(device=cuda)
    g.manual_seed(5)
    q, k, v = _packed(cuda, g, dtype, 2, 140, 4, 2, 64, offset)
    dout = torch.randn(2, 140, 4, 64, generator=g, device=cuda).to(dtype)
    _check(q, k, v, 33, 3, dout)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_padded_batch_ignores_what_lies_behind_the_lengths(cuda, dtype, dim):
    """Lengths 0, 1, inside a tile and whole; NaN and infinities behind them, in the gradients too."""
    g = torch.Generator(device=cuda)
    g.manual_seed(6)
    lengths = [300, 0, 1, 131, 128, 299, 500, -4]
    q, k, v = _packed(cuda, g, dtype, len(lengths), 300, 4, 2, dim)
    dout = torch.randn(q.shape, generator=g, device=cuda).to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    clean = _check(q, k, v, 70, 4, dout, lengths=n)
    for b, m in enumerate(lengths):
        for x, bad in ((q, math.nan), (k, math.nan), (v, math.inf), (dout, math.nan)):
            x[b, max(m, 0):] = bad
    from spar_b200 import ops

    out, lse = ops.window_attention_forward(q, k, v, 70, 4, lengths=n)
    grads = ops.window_attention_backward(dout, q, k, v, out, lse, 70, 4, lengths=n)
    for x, name in zip((out, lse, *grads), ("out", "lse", "dq", "dk", "dv")):
        assert torch.equal(x, clean[name]), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(32, 8), (24, 8)])  # pairs of heads, and (groups of three) of tiles
def test_several_items_for_every_cta(cuda, heads, kv, dim, dtype):
    """More items than SMs, of differing numbers of key tiles and some of none: what a CTA carries from
    one to the next (the rings' phases, both stationary buffers, drawn items, scores that run ahead)."""
    from spar_b200 import ops

    lengths = [400, 0, 217, 385, 1, 129, 400, 384]
    g = torch.Generator(device=cuda)
    g.manual_seed(35)
    q, k, v = _packed(cuda, g, dtype, len(lengths), 400, heads, kv, dim)
    dout = torch.randn(q.shape, generator=g, device=cuda).to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    # sum over sequences of tiles of 128 rows that are not empty, times two tiles or heads an item
    items = sum(-(-x // 128) for x in lengths) * heads // 2
    assert items > 1.5 * torch.cuda.get_device_properties(cuda).multi_processor_count
    for window, sinks in ((100, 4), (260, 0)):
        one = _check(q, k, v, window, sinks, dout, lengths=n)
        out, lse = ops.window_attention_forward(q, k, v, window, sinks, lengths=n)
        grads = ops.window_attention_backward(dout, q, k, v, out, lse, window, sinks, lengths=n)
        for x, name in zip((out, lse, *grads), ("out", "lse", "dq", "dk", "dv")):
            assert torch.equal(x, one[name]), name


CACHE = [
    # b, q_len, kv_len, heads, kv, dim, window, sinks
    (1, 1, 1, 1, 1, 64, 5, 0),
    (3, 1, 40, 4, 4, 64, 16, 4),
    (2, 1, 1000, 8, 2, 128, 256, 4),
    (4, 1, 2100, 16, 1, 64, 5000, 0),   # sixteen heads of one cache
    (2, 3, 777, 8, 2, 64, 100, 1),      # a few tokens at once
    (1, 5, 600, 16, 2, 64, 1000, 4),    # 40 rows of a long cache: still a decoding step
    (2, 64, 700, 2, 2, 128, 600, 3),    # 64
    (2, 64, 500, 2, 2, 128, 600, 3),    # too short beside its rows: tiled
    (1, 65, 900, 1, 1, 64, 900, 0),     # one row more: tiled
    (3, 6, 30, 4, 1, 96, 20, 2),        # 24 rows of a short cache: tiled
    (1, 5, 640, 32, 4, 128, 600, 64),
    (2, 1, 300, 6, 3, 96, 100, 3),
    (1, 2, 500, 3, 1, 50, 100, 3),
    (2, 1, 700, 2, 1, 256, 300, 4),
    (1, 1, 9001, 2, 1, 128, 9001, 0),   # ranges joined by a launch of their own
    (1, 1, 5003, 3, 3, 32, 4000, 70),
    (1, 1, 3001, 2, 2, 256, 2500, 4),
    (1, 40, 900, 4, 2, 64, 300, 4),     # a chunk of a prompt
    (1, 200, 700, 4, 2, 128, 130, 4),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", CACHE)
def test_tokens_against_a_cache(cuda, shape, dtype):
    b, t, n, h, kv, d, window, sinks = shape
    g = torch.Generator(device=cuda)
    g.manual_seed(n + d)
    q = torch.randn(b, t, h, d, generator=g, device=cuda).to(dtype)
    k = torch.randn(b, n, kv, d, generator=g, device=cuda).to(dtype)
    v = torch.randn(b, n, kv, d, generator=g, device=cuda).to(dtype)
    dout = torch.randn(q.shape, generator=g, device=cuda).to(dtype)
    _check(q, k, v, window, sinks, dout)
    lengths = torch.tensor([n - (x * 37) % max(n - t, 1) for x in range(b)], dtype=torch.int32, device=cuda)
    for x in range(b):
        k[x, int(lengths[x]):] = math.nan
        v[x, int(lengths[x]):] = math.nan
    _check(q, k, v, window, sinks, dout, lengths=lengths, first=lengths - t)


def test_positions_of_the_first_row(cuda):
    """Rows before position 0, rows behind the length, and positions far outside."""
    g = torch.Generator(device=cuda)
    g.manual_seed(11)
    for dtype in (torch.float32, torch.bfloat16):
        for t, n in ((4, 200), (160, 200), (200, 90)):
            first = [0, -3, n - 2, n + 5, 2 ** 31 - 1, -2 ** 31, n - t]
            q = torch.randn(len(first), t, 2, 64, generator=g, device=cuda).to(dtype)
            k = torch.randn(len(first), n, 1, 64, generator=g, device=cuda).to(dtype)
            v = torch.randn(len(first), n, 1, 64, generator=g, device=cuda).to(dtype)
            dout = torch.randn(q.shape, generator=g, device=cuda).to(dtype)
            _check(q, k, v, 50, 3, dout, first=torch.tensor(first, dtype=torch.int32, device=cuda))
            if t > n:
                _check(q, k, v, 50, 3, dout)  # default: the first rows stand before position 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,dim", [(200, 64), (130, 128), (70, 96), (3, 64), (90, 33)])
def test_what_no_row_sees_may_hold_anything(cuda, rows, dim, dtype):
    """A chunk of a prompt against a cache whose fill only `first` tells: the slots behind the chunk, those
    older than its first row's window, and rows before position 0 or behind the length reach no result."""
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(33)
    first = torch.tensor([300, 0, 411, -50], dtype=torch.int32, device=cuda)
    q, dout = (torch.randn(4, rows, 4, dim, generator=g, device=cuda).to(dtype) for _ in range(2))
    k, v = (torch.randn(4, 700, 2, dim, generator=g, device=cuda).to(dtype) for _ in range(2))
    longer = torch.tensor([600, 700, 690, 700], dtype=torch.int32, device=cuda)
    inside = torch.tensor([310, 1, 500, 40], dtype=torch.int32, device=cuda)
    for lengths in (None, longer, inside):
        for window, sinks in ((60, 4), (130, 0), (1000, 0)):
            where = dict(lengths=lengths, first=first)
            clean = _check(q, k, v, window, sinks, dout, **where)
            bad = [x.clone() for x in (q, k, v, dout)]
            for b, f in enumerate(first.tolist()):
                n = 700 if lengths is None else int(lengths[b])
                for x in bad[1:3]:
                    x[b, min(max(f + rows, 0), n):] = math.nan
                    x[b, min(max(f + rows, 0), n)::2] = math.inf
                    x[b, sinks:max(max(f, 0) - window + 1, sinks)] = math.nan
                for x in (bad[0], bad[3]):
                    x[b, :max(-f, 0)] = math.nan
                    x[b, max(n - f, 0):] = math.inf
            bq, bk, bv, bdout = bad
            out, lse = ops.window_attention_forward(bq, bk, bv, window, sinks, **where)
            grads = ops.window_attention_backward(bdout, bq, bk, bv, out, lse, window, sinks, **where)
            for x, name in zip((out, lse, *grads), ("out", "lse", "dq", "dk", "dv")):
                assert torch.equal(x, clean[name]), (name, window, sinks)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 20])
def test_nan_in_a_visible_key_or_value(cuda, dim, dtype):
    """It makes every row that sees it NaN, whichever column of a tile it falls on, and no row of
    another head or sequence, nor one far behind the window."""
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(21)
    for place in range(100, 108):
        for part in (1, 2):
            q, k, v = (x.clone() for x in _packed(cuda, g, dtype, 2, 700, 2, 2, dim))
            (k if part == 1 else v)[0, place, 0] = math.nan
            out, lse = ops.window_attention_forward(q, k, v, 90, 2)
            seen = out[0, place:place + 90, 0]
            assert bool(torch.isnan(seen).all()), (place, part)
            if part == 1:
                assert bool(torch.isnan(lse[0, 0, place:place + 90]).all())
            assert bool(torch.isfinite(out[0, :, 1]).all() and torch.isfinite(out[1]).all())
            assert bool(torch.isfinite(out[0, place + 90 + 256:, 0]).all())
            one, one_lse = ops.window_attention_forward(q[:, :1], k[:, :place + 20], v[:, :place + 20], 90, 2)
            assert bool(torch.isnan(one[0, 0, 0]).all() and torch.isfinite(one[0, 0, 1]).all())
            grads = ops.window_attention_backward(torch.ones_like(q), q, k, v, torch.nan_to_num(out),
                                                  torch.nan_to_num(lse), 90, 2)
            assert bool(torch.isfinite(grads[0][0, place + 90 + 256:, 0]).all())
            for x in grads:
                assert bool(torch.isfinite(x[0, :, 1]).all() and torch.isfinite(x[1]).all())


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("part", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("dtype,rows,dim", [(torch.bfloat16, 900, 64), (torch.bfloat16, 900, 128),
                                            (torch.float32, 900, 64), (torch.float32, 900, 128),
                                            (torch.bfloat16, 900, 20), (torch.bfloat16, 5, 64),
                                            (torch.float32, 5, 64)])
def test_how_far_one_bad_value_reaches(cuda, dtype, rows, dim, part, bad):
    """Results that it does not enter keep their bits, or become NaN within 256 positions; those of a
    value's or query's column that it enters are not finite."""
    from spar_b200 import ops

    n, window, sinks = 900, 100, 3
    g = torch.Generator(device=cuda)
    g.manual_seed(34)
    x = {m: torch.randn(2, rows, 4, dim, generator=g, device=cuda).to(dtype) for m in ("q", "dout")}
    x |= {m: torch.randn(2, n, 2, dim, generator=g, device=cuda).to(dtype) for m in ("k", "v")}
    out, lse = ops.window_attention_forward(x["q"], x["k"], x["v"], window, sinks)
    clean = [out, *ops.window_attention_backward(x["dout"], x["q"], x["k"], x["v"], out, lse, window, sinks)]
    row, key = torch.arange(n - rows, n, device=cuda), torch.arange(n, device=cuda)
    see = (key <= row[:, None]) & ((key > row[:, None] - window) | (key < sinks))
    for place in ((1, 433, 897) if part in "kv" else (rows // 2, rows - 2)):
        y = {m: t.clone() for m, t in x.items()}
        y[part][0, place, 1, 0] = bad  # head 1: of the first group as a query, of the second as a key
        heads, kv = (slice(0, 2), slice(0, 1)) if part in ("q", "dout") else (slice(2, 4), slice(1, 2))
        got = ops.window_attention_forward(y["q"], y["k"], y["v"], window, sinks)
        grads = ops.window_attention_backward(y["dout"], y["q"], y["k"], y["v"], *got, window, sinks)
        if part in "kv":  # rows that see it or are near those, and the keys that such a row sees
            rows_in = ((row[:, None] - row[see[:, place]]).abs() <= 256).any(1)
            enter = [see[:, place], see[rows_in].any(0)]
        else:
            enter = [row == row[place], see[place]]
        for t, was, name in zip((got[0], *grads), clean, ("out", "dq", "dk", "dv")):
            at, entered, own = (row, enter[0], heads) if name in ("out", "dq") else (key, enter[1], kv)
            near = ((at[:, None] - at[entered]).abs() <= 256).any(1)
            reach = torch.zeros(t.shape[:3], dtype=torch.bool, device=cuda)
            reach[0, near, own] = True
            changed = ~((t == was) | (torch.isnan(t) & torch.isnan(was)))
            assert not changed[~reach].any(), (name, place)
            reach[0, entered, own] = False
            assert bool(torch.isnan(t[reach])[changed[reach]].all()), (name, place)
            if (part, name) in (("v", "out"), ("dout", "dv"), ("q", "dq")):
                own = own if part == "v" else 1 if part == "q" else kv
                assert not torch.isfinite(t[0, entered][:, own, 0]).any(), (name, place)
                if name != "dq":
                    keep = t[0, entered][:, own, 1:] == was[0, entered][:, own, 1:]
                    assert bool(keep.all()), (name, place)


@pytest.mark.parametrize("dtype,rows,dim", [(torch.bfloat16, 300, 64), (torch.bfloat16, 1, 64),
                                            (torch.bfloat16, 1, 40), (torch.float32, 1, 64),
                                            (torch.float32, 40, 33), (torch.bfloat16, 40, 33)])
def test_scores_of_minus_infinity(cuda, dtype, rows, dim):
    """Keys whose scores are -infinity have no weight; a row that sees only such keys is 0 / 0, and its
    lse is -infinity. (In the tiled, the decoding and the row path.)"""
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(27)
    q = torch.rand(1, rows, 2, dim, generator=g, device=cuda).to(dtype) + 0.5
    k, v = (torch.randn(1, 300, 1, dim, generator=g, device=cuda).to(dtype) for _ in range(2))
    k[0, 298:, :, 0] = -math.inf
    out, lse = ops.window_attention_forward(q, k, v, 2)
    assert torch.isnan(out[0, -1]).all() and torch.isneginf(lse[0, :, -1]).all()
    out, lse = ops.window_attention_forward(q, k, v, 290)
    want, bound = window_attention(*(x.double().cpu() for x in (q[:, -1:], k[:, 10:298], v[:, 10:298])), 300, 0,
                                   h=half_step(dtype))
    assert_within(out[:, -1:], want["out"], bound["out"], "out")
    assert_within(lse[..., -1:], want["lse"], bound["lse"], "lse")
    assert torch.isfinite(lse).all()
    torch.cuda.synchronize()
    assert ops.attention_error() == 0


@pytest.mark.parametrize("rows", [1, 100])
def test_cache_offsets_beyond_32_bits(cuda, rows):
    """70000 tokens 2^16 elements apart: the visible rows lie beyond 2^32 elements of the cache."""
    from spar_b200 import ops

    n, d, apart = 70000, 64, 1 << 16
    cache = torch.zeros(n, apart, device=cuda, dtype=torch.bfloat16)
    g = torch.Generator(device=cuda)
    g.manual_seed(28)
    cache[-400:, :2 * d] = torch.randn(400, 2 * d, generator=g, device=cuda).bfloat16()
    k, v = (cache[None, :, None, i * d:(i + 1) * d] for i in range(2))
    q, dout = (torch.randn(1, rows, 2, d, generator=g, device=cuda).bfloat16() for _ in range(2))
    dk, dv = (cache[None, :, None, i * d:(i + 1) * d] for i in range(2, 4))
    out, lse = ops.window_attention_forward(q, k, v, 250, 3)
    dq, _, _ = ops.window_attention_backward(dout, q, k, v, out, lse, 250, 3, dk=dk, dv=dv)
    torch.cuda.synchronize()
    assert ops.attention_error() == 0
    # all that a row sees: the first tokens (zeros) and the last 400
    pick = [*range(3), *range(n - 400, n)]
    want, bound = window_attention(*(x.double().cpu() for x in (q, k[:, pick], v[:, pick])), 250, 3,
                                   dout=dout.double().cpu(), h=half_step(q.dtype))
    got = {"out": out, "lse": lse, "dq": dq, "dk": dk[:, pick], "dv": dv[:, pick]}
    for name in want:
        assert_within(got[name], want[name], bound[name], name)
    assert not dk[:, 3:n - 400].any() and not dv[:, 3:n - 400].any()


@pytest.mark.parametrize("n,window,dim", [(16, 16, 32), (24, 300, 64), (40, 16, 128), (300, 16, 64),
                                          (300, 16, 128), (600, 200, 64), (60, 16, 36)])
def test_bf16_is_off_by_two_roundings(cuda, n, window, dim):
    """In the 2-norm: the stored result's rounding, and that of P or dS before its product, of the same
    size and independent: sqrt(2) of the one that every bf16 result has, 1.5 with what chance adds. (D
    from the rounded `out` alone would be a third in dq and dk: 1.5 to 1.75.)"""
    g = torch.Generator(device=cuda)
    g.manual_seed(36)
    b = max(1, 4800 // n)
    q, k, v = _packed(cuda, g, torch.bfloat16, b, n, 4, 4, dim)
    dout = torch.randn(q.shape, generator=g, device=cuda).bfloat16()
    got = _check(q, k, v, window, 0, dout)
    want, _ = window_attention(*(x.double().cpu() for x in (q, k, v)), window, 0, dout=dout.double().cpu())
    for name in ("out", "dq", "dk", "dv"):
        once = (want[name].bfloat16().double() - want[name]).norm()
        off = (got[name].double().cpu() - want[name]).norm()
        assert off <= 1.5 * once, (name, float(off / once))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_logits_and_a_given_scale(cuda, dtype):
    g = torch.Generator(device=cuda)
    g.manual_seed(12)
    q, k, v = _packed(cuda, g, dtype, 1, 260, 2, 1, 64)
    dout = torch.randn(q.shape, generator=g, device=cuda).to(dtype)
    _check(q * 6, k * 6, v, 90, 4, dout)
    _check(q, k, v, 90, 4, dout, scale=0.9)
    rising = (k * torch.linspace(0, 8, 260, device=cuda)[None, :, None, None]).to(dtype)
    _check(q, rising, v, 260, 0, dout)  # the maximum keeps moving


def test_outputs_into_a_packed_buffer_leave_the_rest(cuda):
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(13)
    for dtype in (torch.float32, torch.bfloat16):
        for d in (64, 33):
            q, k, v = _packed(cuda, g, dtype, 2, 135, 4, 2, d)
            dout = torch.randn(q.shape, generator=g, device=cuda).to(dtype)
            out, lse = ops.window_attention_forward(q, k, v, 40, 2)
            want = ops.window_attention_backward(dout, q, k, v, out, lse, 40, 2)
            wide = torch.full((2, 137, 11, d + 8), 7.0, device=cuda, dtype=dtype)
            o = wide[:, 1:136, 0:4, :d]
            ops.window_attention_forward(q, k, v, 40, 2, out=o)
            assert torch.equal(o, out)
            o.fill_(7.0)
            assert bool((wide == 7.0).all())
            dq, dk, dv = (wide[:, 1:136, s, :d] for s in (slice(0, 4), slice(4, 6), slice(7, 9)))
            got = ops.window_attention_backward(dout, q, k, v, out, lse, 40, 2, dq=dq, dk=dk, dv=dv)
            for x, y in zip(got, want):
                assert torch.equal(x, y)
                x.fill_(7.0)
            assert bool((wide == 7.0).all())


def test_repeats_streams_and_captured_graphs(cuda):
    """The same bits on every run; two captured graphs and an eager call share nothing."""
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(14)
    sets = []
    for b, t, n in ((2, 260, 260), (1, 1, 900)):
        for dtype in (torch.float32, torch.bfloat16):
            q = torch.randn(b, t, 8, 64, generator=g, device=cuda).to(dtype)
            k = torch.randn(b, n, 2, 64, generator=g, device=cuda).to(dtype)
            v = torch.randn(b, n, 2, 64, generator=g, device=cuda).to(dtype)
            sets.append((q, k, v, torch.randn(q.shape, generator=g, device=cuda).to(dtype)))

    def block(s):
        q, k, v, dout = s
        out, lse = ops.window_attention_forward(q, k, v, 100, 4)
        return (out, lse, *ops.window_attention_backward(dout, q, k, v, out, lse, 100, 4))

    want = [block(s) for s in sets]
    for s, w in zip(sets, want):
        assert all(torch.equal(a, b) for a, b in zip(block(s), w))
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, block(s)))
        graphs[-1] = (graph, graphs[-1][1])
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for (graph, _), stream in zip(graphs, streams):
        with torch.cuda.stream(stream):
            graph.replay()
    eager = [block(s) for s in sets]
    torch.cuda.synchronize()
    for (_, held), e, w in zip(graphs, eager, want):
        assert all(torch.equal(a, b) for a, b in zip(held, w))
        assert all(torch.equal(a, b) for a, b in zip(e, w))


def test_first_call_of_a_process_may_be_captured():
    """Nothing needs a call outside a capture first (the kernels' set-up is not stream work)."""
    import subprocess
    import sys

    code = """
import torch
from spar_b200 import ops
q = torch.randn(2, 200, 4, 64, device="cuda").bfloat16()
k, one = torch.randn_like(q[:, :, :2]), torch.randn(2, 1, 4, 64, device="cuda").bfloat16()
w, table = torch.ones(64, device="cuda"), torch.zeros(200, 32, 2, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
def block():
    a, b = ops.qk_norm_rotary_forward(q, k, w, w, table)
    out, lse = ops.window_attention_forward(a, b, k, 50, 4)
    return (out, *ops.window_attention_backward(out, a, b, k, out, lse, 50, 4),
            *ops.window_attention_forward(one, b, k, 50, 4), ops.rotary_table(9, 64, device="cuda"))
with torch.cuda.graph(graph):
    held = block()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(x, y) for x, y in zip(held, block()))
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


def test_nothing_to_do(cuda):
    from spar_b200 import ops

    empty = torch.empty(2, 0, 4, 64, device=cuda)
    some = torch.ones(2, 5, 2, 64, device=cuda)
    out, lse = ops.window_attention_forward(empty, some, some, 4)
    assert out.shape == empty.shape and lse.shape == (2, 4, 0)
    dq, dk, dv = ops.window_attention_backward(empty, empty, some, some, out, lse, 4)
    assert not dk.any() and not dv.any()
    q = torch.ones(2, 3, 4, 64, device=cuda)
    none = torch.empty(2, 0, 2, 64, device=cuda)
    out, lse = ops.window_attention_forward(q, none, none, 4)
    assert not out.any() and bool((lse == -math.inf).all())
    dq, dk, dv = ops.window_attention_backward(q, q, none, none, out, lse, 4)
    assert not dq.any() and dk.shape == none.shape


def test_wide_window_is_the_framework_causal_attention(cuda):
    """With a window over everything this is attention_forward / attention_backward, within the
    2e-3 of their TF32 products."""
    from _util import rel_l2
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(15)
    b, t, h, kv, d = 2, 200, 4, 2, 64
    x = torch.randn(b, t, (h + 2 * kv) * d, generator=g, device=cuda)
    dout = torch.randn(b, t, h * d, generator=g, device=cuda)
    ctx, top, inv = ops.attention_forward(x, h, kv)
    dx = ops.attention_backward(dout, x, ctx, top, inv, h, kv_heads=kv)
    parts = lambda y: (y[..., :h * d].unflatten(-1, (h, d)), y[..., h * d:(h + kv) * d].unflatten(-1, (kv, d)),  # noqa: E731
                       y[..., (h + kv) * d:].unflatten(-1, (kv, d)))
    q, k, v = parts(x)
    out, lse = ops.window_attention_forward(q, k, v, t)
    mine = torch.empty_like(x)
    dq, dk, dv = parts(mine)
    ops.window_attention_backward(dout.unflatten(-1, (h, d)), q, k, v, out, lse, t, dq=dq, dk=dk, dv=dv)
    assert rel_l2(out.flatten(2).cpu(), ctx.cpu()) <= 2e-3
    for a, b_ in zip(parts(mine), parts(dx)):
        assert rel_l2(a.cpu(), b_.cpu()) <= 3e-3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_block_forward_and_backward(cuda, dtype):
    """Norm and rotation of the packed projection's queries and keys, window attention, and back to
    the gradient of the projection, as a layer runs them; then one token against the cache that the
    layer's keys and values make, at its position in the table."""
    from _attention_ref import norm_rotate
    from _util import rel_l2
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(16)
    b, t, h, kv, d, window, sinks = 2, 190, 8, 2, 64, 60, 4
    width = (h + 2 * kv) * d
    x = (2 * torch.randn(b, t, width, generator=g, device=cuda)).to(dtype)
    dout = torch.randn(b, t, h, d, generator=g, device=cuda).to(dtype)
    w = [1 + 0.2 * torch.randn(d, generator=g, device=cuda) for _ in range(2)]
    scaling = ops.RotaryScaling("parts", 4.0, 64)
    table = ops.rotary_table(t, d // 2, scaling=scaling, device=cuda)
    parts = lambda y: (y[..., :h * d].unflatten(-1, (h, d)), y[..., h * d:(h + kv) * d].unflatten(-1, (kv, d)),  # noqa: E731
                       y[..., (h + kv) * d:].unflatten(-1, (kv, d)))
    q, k, v = parts(x)
    rq, rk = ops.qk_norm_rotary_forward(q, k, *w, table, layout="half")
    out, lse = ops.window_attention_forward(rq, rk, v, window, sinks)
    dx = torch.empty_like(x)
    dq, dk, dv = parts(dx)
    ops.window_attention_backward(dout, rq, rk, v, out, lse, window, sinks, dq=dq, dk=dk, dv=dv)
    _, _, dwq, dwk = ops.qk_norm_rotary_backward(dq, dk, q, k, *w, table, layout="half", dq=dq, dk=dk)

    x64 = x.double().cpu().requires_grad_()
    w64 = [y.double().cpu().requires_grad_() for y in w]
    angles = table.double().cpu()[None]
    q64, k64, v64 = parts(x64)
    q64 = norm_rotate(q64, w64[0], angles, d // 2, "half", 1e-6)
    k64 = norm_rotate(k64, w64[1], angles, d // 2, "half", 1e-6)
    p = torch.arange(t)
    see = (p[None] <= p[:, None]) & ((p[None] > p[:, None] - window) | (p[None] < sinks))
    s = torch.einsum("bihd,bjhd->bhij", q64, k64.repeat_interleave(h // kv, 2)) * d ** -0.5
    o64 = torch.einsum("bhij,bjhd->bihd", torch.softmax(s.masked_fill(~see, -math.inf), -1),
                       v64.repeat_interleave(h // kv, 2))
    o64.backward(dout.double().cpu())
    # A chain of a handful of roundings to the stored type (rotated q, k, P, dS, out, the gradients
    # twice): at most eight half steps in the 2-norm, and 2^-20 for the sums in 32 bits.
    tol = 8 * half_step(dtype) + 2.0 ** -20
    for got, want in ((out, o64), (dx, x64.grad), (dwq, w64[0].grad), (dwk, w64[1].grad)):
        assert rel_l2(got.detach().double().cpu(), want.detach()) <= tol

    token = torch.full((b, 1), t - 1, dtype=torch.int32, device=cuda)
    q1, _ = ops.qk_norm_rotary_forward(q[:, t - 1:], None, w[0], None, table, layout="half",
                                       positions=token)
    assert torch.equal(q1, rq[:, t - 1:])
    o1, lse1 = ops.window_attention_forward(q1, rk, v, window, sinks)
    assert rel_l2(o1.double().cpu(), o64[:, t - 1:].detach()) <= tol
    assert float((lse1[..., 0] - lse[..., t - 1]).abs().max()) <= 2.0 ** -18


def test_wrong_calls_are_refused(cuda):
    from spar_b200 import ops

    q, k = torch.zeros(2, 4, 4, 64, device=cuda), torch.zeros(2, 9, 2, 64, device=cuda)
    n = torch.zeros(2, dtype=torch.int32, device=cuda)
    f = ops.window_attention_forward
    bad = [lambda: f(q, k, k, 0), lambda: f(q, k, k, 4, -1), lambda: f(q, k, k[:, :8], 4),
           lambda: f(q, k.bfloat16(), k.bfloat16(), 4), lambda: f(q.double(), k.double(), k.double(), 4),
           lambda: f(q[:, :, :3], k, k, 4), lambda: f(q, k[..., :32], k[..., :32], 4),
           lambda: f(q, k, k, 4, scale=0.0), lambda: f(q, k, k, 4, lengths=n[:1]),
           lambda: f(q, k, k, 4, first=n.long()), lambda: f(q.cpu(), k.cpu(), k.cpu(), 4),
           lambda: f(q, k, k, 4, out=torch.zeros(2, 4, 4, 64, device=cuda, dtype=torch.bfloat16)),
           lambda: f(q[:1], k, k, 4)]
    for call in bad:
        with pytest.raises(ValueError):
            call()

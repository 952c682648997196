"""Rotary positions and qk-norm with the rotation, forward and backward, against 64-bit forms.

Bounds (u = 2^-24, h half a step of the stored type): a rotation is two products and a sum, off by
at most 3 u (|a cos| + |b sin|) before it is stored; the norm adds 1/rms, a sum of at most 256
squares in pieces of 16 (under 24 u after the square root, with divide and root), and two products.
"""
import pytest
import torch

from _attention_ref import (U, assert_within, half_step, norm_rotate, norm_rotate_backward, rotate)

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _views(cuda, g, dtype, b, t, h, kv, d, packed=True, offset=0):
    """q and k as parts of a packed projection, `offset` elements from its start."""
    width = (h + 2 * kv) * d
    flat = torch.randn(b * t * width + offset, generator=g, device=cuda).to(dtype)
    x = flat[offset:].view(b, t, width)
    q, k = x[..., :h * d].unflatten(-1, (h, d)), x[..., h * d:(h + kv) * d].unflatten(-1, (kv, d))
    return (q, k) if packed else (q.contiguous(), k.contiguous())


def _table(cuda, rows, rotary, g):
    angle = torch.rand(rows, rotary // 2, generator=g, device=cuda, dtype=torch.float64) * 6.3
    return torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()


def _angles(table, positions, start, t):
    table = table.double().cpu()
    return table[start:start + t][None] if positions is None else table[positions.long().cpu()]


def _size(x, angles, rotary, layout):
    a = rotate(x.abs(), angles.abs(), rotary, layout, -1.0).abs()
    return torch.maximum(a, rotate(x.abs(), angles.abs(), rotary, layout).abs())


SHAPES = [
    # b, t, heads, kv, dim, rotary, offset
    (1, 1, 1, 1, 2, 2, 0),       # one pair
    (1, 1, 12, 12, 64, 64, 0),
    (3, 17, 8, 2, 64, 32, 0),    # part of the head
    (2, 33, 6, 3, 128, 128, 0),  # head chunks that do not fill
    (2, 5, 4, 1, 96, 48, 0),
    (1, 7, 3, 2, 256, 256, 0),
    (1, 9, 2, 1, 256, 64, 0),
    (2, 11, 2, 1, 33, 10, 0),    # odd head, element by element
    (1, 13, 5, 1, 80, 20, 0),
    (2, 6, 4, 2, 64, 64, 1),     # rows that are not aligned to 16 bytes
    (1, 700, 16, 4, 64, 64, 0),  # enough work for whole head chunks
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotary(cuda, shape, layout, dtype):
    from spar_b200 import ops

    b, t, h, kv, d, r, offset = shape
    g = torch.Generator(device=cuda)
    g.manual_seed(d * 7 + t)
    q, k = _views(cuda, g, dtype, b, t, h, kv, d, offset=offset)
    table = _table(cuda, t + 40, r, g)
    positions = torch.randint(0, t + 40, (b, t), generator=g, device=cuda).to(torch.int32)
    for pos, start, inverse in ((positions, 0, False), (None, 5, True)):
        got = ops.rotary(q, k, table, layout=layout, positions=pos, start=start, inverse=inverse)
        angles = _angles(table, pos, start, t)
        for x, y in zip((q, k), got):
            x = x.double().cpu()
            want = rotate(x, angles, r, layout, -1.0 if inverse else 1.0)
            turned = 3 * U * _size(x, angles, r, layout)
            turned[..., r:] = 0
            assert_within(y, want, half_step(dtype) * want.abs() + (1 + half_step(dtype)) * turned)


def test_rotary_back_and_forth_in_place_matches_out_of_place(cuda):
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(3)
    q, k = _views(cuda, g, torch.float32, 2, 31, 8, 2, 64)
    table = _table(cuda, 31, 64, g)
    out_q, out_k = ops.rotary(q, k, table, layout="half")
    whole = q.clone(), k.clone()
    got = ops.rotary(q, k, table, layout="half", q_out=q, k_out=k)
    assert got[0] is q and torch.equal(q, out_q) and torch.equal(k, out_k)
    ops.rotary(q, k, table, layout="half", inverse=True, q_out=q, k_out=k)
    for x, y in zip(whole, (q, k)):  # two rotations with a table of 2^-25 absolute error
        assert float((x - y).abs().max()) <= 16 * U * float(x.abs().max())


def test_rotary_matches_the_framework_rotation(cuda):
    """The interleaved layout with the plain table is spar_b200_rope_apply's rotation."""
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(4)
    q, _ = _views(cuda, g, torch.float32, 2, 50, 4, 1, 64, packed=False)
    table = ops.rope_table(50, 64, device=cuda)
    mine = ops.rotary_table(50, 64, device=cuda)
    assert float((table - mine).abs().max()) <= 2 * U
    got, none = ops.rotary(q, None, table)
    assert none is None
    want = ops.rope_apply_(q.clone(), table, 2, 50, 4, 64, 256)
    assert float((got - want).abs().max()) <= 4 * U * float(want.abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("shape", SHAPES)
def test_qk_norm_rotary(cuda, shape, layout, dtype):
    from spar_b200 import ops

    b, t, h, kv, d, r, offset = shape
    g = torch.Generator(device=cuda)
    g.manual_seed(d * 5 + t)
    q, k = _views(cuda, g, dtype, b, t, h, kv, d, offset=offset)
    dq, dk = _views(cuda, g, dtype, b, t, h, kv, d, offset=offset)
    table = _table(cuda, t + 9, r, g)
    positions = torch.randint(0, t + 9, (b, t), generator=g, device=cuda).to(torch.int32)
    w = [1 + 0.3 * torch.randn(d, generator=g, device=cuda) for _ in range(2)]
    got = ops.qk_norm_rotary_forward(q, k, *w, table, EPS, layout=layout, positions=positions)
    back = ops.qk_norm_rotary_backward(dq, dk, q, k, *w, table, EPS, layout=layout, positions=positions)
    angles, hs = _angles(table, positions, 0, t), half_step(dtype)
    for x, dy, ww, y, dx, dw in zip((q, k), (dq, dk), w, got, back[:2], back[2:]):
        x, dy, ww = x.double().cpu(), dy.double().cpu(), ww.double().cpu()
        want = norm_rotate(x, ww, angles, r, layout, EPS)
        inv = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        size = _size(x * inv * ww, angles, r, layout)
        assert_within(y, want, hs * want.abs() + 32 * U * size, "y")
        wdx, wdw, sdx, sdw = norm_rotate_backward(dy, x, ww, angles, r, layout, EPS)
        # the mean and 1/rms are each under 32 u off, on both terms
        assert_within(dx, wdx, hs * wdx.abs() + 96 * U * sdx, "dx")
        # a sum of b t heads terms in any order, each under 40 u off
        assert_within(dw, wdw, (40 + b * t * x.shape[2]) * U * sdw, "dw")


def test_qk_norm_rotary_backward_matches_differences(cuda):
    """The 64-bit gradients the kernels are held to, against central differences of the 64-bit
    forward: step 1e-5 leaves 1e-10 of curvature and 1e-11 of rounding; 1e-7 is allowed."""
    g = torch.Generator()
    g.manual_seed(8)
    x = torch.randn(1, 3, 2, 12, generator=g, dtype=torch.float64)
    w = 1 + 0.3 * torch.randn(12, generator=g, dtype=torch.float64)
    dy = torch.randn(1, 3, 2, 12, generator=g, dtype=torch.float64)
    a = torch.rand(1, 3, 4, generator=g, dtype=torch.float64) * 6
    angles = torch.stack([a.cos(), a.sin()], -1)
    for layout in ("half", "interleaved"):
        dx, dw, _, _ = norm_rotate_backward(dy, x, w, angles, 8, layout, EPS)
        f = lambda x, w: float((norm_rotate(x, w, angles, 8, layout, EPS) * dy).sum())  # noqa: E731,B023
        for grad, at in ((dx, 0), (dw, 1)):
            v = torch.randn(grad.shape, generator=g, dtype=torch.float64)
            args = [[x, w], [x, w]]
            args[0][at], args[1][at] = args[0][at] + 1e-5 * v, args[1][at] - 1e-5 * v
            assert abs((f(*args[0]) - f(*args[1])) / 2e-5 - float((grad * v).sum())) <= 1e-7


def test_qk_norm_rotary_accumulates_repeats_and_takes_no_keys(cuda):
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(9)
    q, k = _views(cuda, g, torch.bfloat16, 2, 300, 8, 2, 64)
    dq, dk = _views(cuda, g, torch.bfloat16, 2, 300, 8, 2, 64)
    table = _table(cuda, 300, 64, g)
    w = [torch.ones(64, device=cuda), torch.ones(64, device=cuda)]
    one = ops.qk_norm_rotary_backward(dq, dk, q, k, *w, table, layout="half")
    two = ops.qk_norm_rotary_backward(dq, dk, q, k, *w, table, layout="half")
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    held = [torch.full((64,), 3.0, device=cuda) for _ in range(2)]
    ops.qk_norm_rotary_backward(dq, dk, q, k, *w, table, layout="half", dq_weight=held[0],
                                dk_weight=held[1], accumulate_params=True)
    assert torch.equal(held[0], 3.0 + one[2]) and torch.equal(held[1], 3.0 + one[3])
    only = ops.qk_norm_rotary_backward(dq, None, q, None, w[0], None, table, layout="half")
    assert torch.equal(only[0], one[0]) and only[1] is None and only[3] is None
    y = ops.qk_norm_rotary_forward(q, k, *w, table, layout="half")
    alone, _ = ops.qk_norm_rotary_forward(q, None, w[0], None, table, layout="half")
    assert torch.equal(y[0], alone)
    inplace = dq.clone(), dk.clone()
    ops.qk_norm_rotary_backward(*inplace, q, k, *w, table, layout="half", dq=inplace[0], dk=inplace[1])
    assert torch.equal(inplace[0], one[0]) and torch.equal(inplace[1], one[1])


def test_positions_outside_the_table_give_zeros_and_set_the_flag(cuda):
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(10)
    for d, r in ((64, 64), (33, 10)):
        q, k = _views(cuda, g, torch.float32, 2, 6, 4, 2, d)
        table = _table(cuda, 8, r, g)
        good = torch.randint(0, 8, (2, 6), generator=g, device=cuda).to(torch.int32)
        bad = good.clone()
        bad[0, 3], bad[1, 0] = 8, -1
        flag = torch.zeros(1, dtype=torch.int32, device=cuda)
        want = ops.rotary(q, k, table, positions=good, invalid=flag)
        assert int(flag) == 0
        got = ops.rotary(q, k, table, positions=bad, invalid=flag)
        assert int(flag) == 1
        ones = torch.ones(d, device=cuda)
        flag.zero_()
        back = ops.qk_norm_rotary_backward(q, k, q, k, ones, ones, table, positions=bad, invalid=flag)
        assert int(flag) == 1
        mask = torch.ones(2, 6, dtype=torch.bool, device=cuda)
        mask[0, 3] = mask[1, 0] = False
        for x, y, dx, dw in zip(want, got, back[:2], back[2:]):
            assert torch.equal(y[mask], x[mask]) and not y[~mask].any() and not dx[~mask].any()
            assert bool(torch.isfinite(dw).all())


@pytest.mark.parametrize("d,r", [(64, 64), (64, 32), (33, 10)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_table_without_rows_has_no_position_inside(cuda, dtype, d, r):
    """Every position lies outside it: zeros, the flag, weight gradients of zero; nothing of it is read
    (there may be no table at all)."""
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(31)
    q, k = _views(cuda, g, dtype, 2, 6, 4, 2, d)
    ones = torch.ones(d, device=cuda)
    positions = torch.zeros(2, 6, dtype=torch.int32, device=cuda)
    table = torch.empty(0, r // 2, 2, device=cuda)
    for layout in ("interleaved", "half"):
        where = dict(layout=layout, positions=positions)
        for call in (lambda f: ops.rotary(q, k, table, invalid=f, **where),
                     lambda f: ops.qk_norm_rotary_forward(q, k, ones, ones, table, invalid=f, **where),
                     lambda f: ops.qk_norm_rotary_backward(q, k, q, k, ones, ones, table, invalid=f, **where)):
            flag = torch.zeros(1, dtype=torch.int32, device=cuda)
            got = call(flag)
            assert int(flag) == 1
            for x in got:
                assert not x.any()


def test_no_tokens(cuda):
    from spar_b200 import ops

    q, k = torch.empty(2, 0, 4, 64, device=cuda), torch.empty(2, 0, 2, 64, device=cuda)
    table = torch.zeros(3, 32, 2, device=cuda)
    w = torch.ones(64, device=cuda)
    assert ops.rotary(q, k, table)[0].shape == q.shape
    assert ops.qk_norm_rotary_forward(q, k, w, w, table)[1].shape == k.shape
    _, _, dwq, dwk = ops.qk_norm_rotary_backward(q, k, q, k, w, w, table)
    assert not dwq.any() and not dwk.any()
    assert ops.rotary_table(0, 64, device=cuda).shape == (0, 32, 2)


def test_keys_without_heads(cuda):
    from spar_b200 import ops

    q, k = torch.ones(2, 3, 4, 64, device=cuda), torch.ones(2, 3, 0, 64, device=cuda)
    table, w = torch.ones(3, 32, 2, device=cuda), torch.ones(64, device=cuda)
    held = torch.full((64,), 7.0, device=cuda)
    dq, dk, dwq, dwk = ops.qk_norm_rotary_backward(q, k, q, k, w, w, table, dk_weight=held)
    alone = ops.qk_norm_rotary_backward(q, None, q, None, w, None, table)
    assert torch.equal(dq, alone[0]) and torch.equal(dwq, alone[2])
    assert dk.shape == k.shape and dwk is held and not held.any()
    held.fill_(7.0)
    ops.qk_norm_rotary_backward(q, k, q, k, w, w, table, dq_weight=w.clone(), dk_weight=held, accumulate_params=True)
    assert bool((held == 7.0).all())


@pytest.mark.parametrize("kind", ["none", "linear", "base", "parts"])
@pytest.mark.parametrize("rows,rotary,start", [(1, 4, 0), (33, 64, 0), (500, 96, 7), (70, 128, 1 << 20)])
def test_rotary_table(cuda, rows, rotary, start, kind):
    """cos and sin to half a step of fp32, plus the angle's own 64-bit error: position times
    frequency is off by 2^-52 of itself (and pow by a few of its last places)."""
    import math

    from spar_b200 import ops

    theta, factor, length = 10000.0, 8.0, 2048.0
    i = torch.arange(rotary // 2, dtype=torch.float64)
    f, magnitude = theta ** (-2 * i / rotary), 1.0
    if kind == "linear":
        f = f / factor
    elif kind == "base":
        f = (theta * factor ** (rotary / (rotary - 2))) ** (-2 * i / rotary)
    elif kind == "parts":
        keep = ((length * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f, magnitude = f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1
    angle = (torch.arange(rows, dtype=torch.float64) + start)[:, None] * f
    want = torch.stack([angle.cos(), angle.sin()], -1) * magnitude
    scaling = None if kind == "none" else ops.RotaryScaling(kind, factor, length)
    got = ops.rotary_table(rows, rotary, theta, start, scaling, device=cuda)
    slack = 2.0 ** -49 * (1 + angle.abs())[..., None]
    assert_within(got, want, U * want.abs() + slack)


def _lanes(dim, rotary, dtype):
    """Lanes of a head's group in the vectorised forms: the power of two that holds its slots."""
    v = 4 if dtype == torch.float32 else 8
    slots = rotary // 2 // v + ((dim - rotary) // v + 1) // 2
    return 1 << (slots - 1).bit_length()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("rotary", [64, 32])
def test_enough_tokens_that_heads_share_their_angles(cuda, rotary, layout, dtype):
    """From 64 warps an SM on, a lane group takes two or four heads of a token; 17 and 3 heads leave
    chunks that are not full, and the tokens do not fill the last block."""
    from spar_b200 import ops

    h, kv, d, b = 17, 3, 64, 3
    warps = 64 * torch.cuda.get_device_properties(cuda).multi_processor_count
    t = warps * 32 // (b * (h + kv) * _lanes(d, rotary, dtype)) + 3
    g = torch.Generator(device=cuda)
    g.manual_seed(41)
    q, k = _views(cuda, g, dtype, b, t, h, kv, d)
    table = _table(cuda, t + 40, rotary, g)
    positions = torch.randint(0, t + 40, (b, t), generator=g, device=cuda).to(torch.int32)
    w = [1 + 0.3 * torch.randn(d, generator=g, device=cuda) for _ in range(2)]
    for pos, start, inverse in ((positions, 0, False), (None, 5, True)):
        where = dict(layout=layout, positions=pos, start=start)
        turned = ops.rotary(q, k, table, inverse=inverse, **where)
        normed = ops.qk_norm_rotary_forward(q, k, *w, table, EPS, **where)
        angles, hs = _angles(table, pos, start, t), half_step(dtype)
        for x, ww, y, z in zip((q, k), w, turned, normed):
            x, ww = x.double().cpu(), ww.double().cpu()
            want = rotate(x, angles, rotary, layout, -1.0 if inverse else 1.0)
            off = 3 * U * _size(x, angles, rotary, layout)
            off[..., rotary:] = 0
            assert_within(y, want, hs * want.abs() + (1 + hs) * off, "turned")
            want = norm_rotate(x, ww, angles, rotary, layout, EPS)
            inv = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            assert_within(z, want, hs * want.abs() + 32 * U * _size(x * inv * ww, angles, rotary, layout), "normed")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 32), (33, 10)])
def test_backward_over_more_units_than_the_grid_has_groups(cuda, dim, rotary, layout, dtype):
    """Sixteen blocks of 128 threads an SM, split between queries and keys, walk the tokens: here every
    lane group takes two or three units of either side, and the sums of the weights stay in registers."""
    from spar_b200 import ops

    h, kv, b = 9, 3, 2
    lanes = 32 if dim == 33 else _lanes(dim, rotary, dtype)
    shared = 2 if dtype == torch.float32 and dim != 33 else 1  # heads of a unit
    blocks = 16 * torch.cuda.get_device_properties(cuda).multi_processor_count
    chunks = -(-h // shared) + -(-kv // shared)
    t = int(2.5 * blocks * (128 // lanes) / (b * chunks)) + 1
    g = torch.Generator(device=cuda)
    g.manual_seed(42)
    q, k = _views(cuda, g, dtype, b, t, h, kv, dim)
    dq, dk = _views(cuda, g, dtype, b, t, h, kv, dim)
    table = _table(cuda, t + 9, rotary, g)
    w = [1 + 0.3 * torch.randn(dim, generator=g, device=cuda) for _ in range(2)]
    back = ops.qk_norm_rotary_backward(dq, dk, q, k, *w, table, EPS, layout=layout, start=7)
    again = ops.qk_norm_rotary_backward(dq, dk, q, k, *w, table, EPS, layout=layout, start=7)
    assert all(torch.equal(x, y) for x, y in zip(back, again))
    angles, hs = table.double()[7:7 + t][None], half_step(dtype)
    for x, dy, ww, dx, dw in zip((q, k), (dq, dk), w, back[:2], back[2:]):
        wdx, wdw, sdx, sdw = (y.cpu() for y in norm_rotate_backward(dy.double(), x.double(), ww.double(), angles,
                                                                    rotary, layout, EPS))
        assert_within(dx, wdx, hs * wdx.abs() + 96 * U * sdx, "dx")
        # Each term is under 40 u off; their sum goes through at most 3 units x 2 heads of a lane, the
        # groups of a block and the blocks: fewer additions than blocks + 128 + 8.
        assert_within(dw, wdw, (40 + blocks + 136) * U * sdw, "dw")


def test_captured_on_another_stream_and_replayed(cuda):
    from spar_b200 import ops

    g = torch.Generator(device=cuda)
    g.manual_seed(12)
    q, k = _views(cuda, g, torch.bfloat16, 2, 65, 8, 2, 64)
    dq, dk = _views(cuda, g, torch.bfloat16, 2, 65, 8, 2, 64)
    table = _table(cuda, 65, 64, g)
    w = [1 + 0.3 * torch.randn(64, generator=g, device=cuda) for _ in range(2)]

    def block():
        y = ops.qk_norm_rotary_forward(q, k, *w, table, layout="half")
        return (*y, *ops.qk_norm_rotary_backward(dq, dk, q, k, *w, table, layout="half"),
                *ops.rotary(*y, table, layout="half", inverse=True))

    block()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = block()
    q.copy_(torch.randn(q.shape, generator=g, device=cuda))
    graph.replay()
    torch.cuda.synchronize()
    want = block()
    assert all(torch.equal(a, b) for a, b in zip(held, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = block()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))


def test_wrong_calls_are_refused(cuda):
    from spar_b200 import ops
    from spar_b200._lib import SparError

    q, k = torch.zeros(2, 4, 4, 64, device=cuda), torch.zeros(2, 4, 2, 64, device=cuda)
    table, w = torch.zeros(4, 32, 2, device=cuda), torch.ones(64, device=cuda)
    with pytest.raises(SparError):
        ops.rotary(q, k, table, start=1)  # the last token lies behind the table
    with pytest.raises(SparError):
        ops.rotary(q, k, torch.zeros(4, 33, 2, device=cuda))  # more pairs than the head has
    bad = [lambda: ops.rotary(q, k.bfloat16(), table), lambda: ops.rotary(q.half(), k.half(), table),
           lambda: ops.rotary(q, k[:, :3], table), lambda: ops.rotary(q, k, table, layout="other"),
           lambda: ops.rotary(q.cpu(), k.cpu(), table), lambda: ops.rotary(q[0], k[0], table),
           lambda: ops.rotary(q.transpose(2, 3), k, table), lambda: ops.rotary(q, k, table.double()),
           lambda: ops.rotary(q, k, table, positions=torch.zeros(2, 4, device=cuda)),
           lambda: ops.rotary(q, k, table, q_out=torch.zeros(2, 4, 4, 32, device=cuda)),
           lambda: ops.qk_norm_rotary_forward(q, k, w[:32], w, table),
           lambda: ops.qk_norm_rotary_backward(q, k, q, k, w, w, table, accumulate_params=True),
           lambda: ops.rotary_table(4, 64, scaling=ops.RotaryScaling("other", 2.0), device=cuda)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for scaling in (ops.RotaryScaling("linear", 0.0), ops.RotaryScaling("parts", 2.0),
                    ops.RotaryScaling("parts", 2.0, 2048, 1.0, 1.0),
                    ops.RotaryScaling("linear", 2.0, magnitude=-1.0)):
        with pytest.raises(SparError):
            ops.rotary_table(4, 64, scaling=scaling, device=cuda)
    with pytest.raises(SparError):
        ops.rotary_table(4, 2, scaling=ops.RotaryScaling("base", 2.0), device=cuda)

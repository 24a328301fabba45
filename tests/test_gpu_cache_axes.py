"""Rotation and append with positions of several axes.

Two kinds of check.  Against 64 bits: pair j of a token is a complex product by the table's entry at its
axis's position; a product and a sum in 32 bits are off by 3 * 2^-24 of |a c| + |b s|, the result by its own
type's rounding.  And to the bit against the calls of one axis: with a table that holds, row by row, the roots
of each token (entry j of row t is ``table[positions[axis(j), t], j]``) they do the same arithmetic.
"""
import math
import struct

import pytest
import torch

import bfft
from bfft import _lib, cache
from test_gpu_cache import BF16, F16, F32, HALF_UNIT, Pages, cumulative, generator, ints, normal

pytestmark = pytest.mark.gpu


def dealt(axes, order):
    """The axis of each pair, dealt one at a time."""
    left = list(axes)
    if order == "blocks":
        return [a for a, n in enumerate(axes) for _ in range(n)]
    out = []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


def token_table(table, positions, axes, order):
    """(tokens, pairs, 2): the roots of each token; positions (axes, tokens)."""
    axis = torch.tensor(dealt(axes, order), device="cuda")
    rows = positions.long()[axis].T
    return table[rows, torch.arange(len(axis), device="cuda")].contiguous()


def check_turned(got, x, roots, layout, sign=1.0):
    """x (tokens, heads, dim) rotated by roots (tokens, pairs, 2) in 64 bits."""
    pairs = roots.shape[1]
    c, s = roots.double()[:, None].unbind(-1)
    s = sign * s
    part = x.double()[..., :2 * pairs]
    a, b = (part[..., :pairs], part[..., pairs:]) if layout == "half" else (part[..., 0::2], part[..., 1::2])
    z = [a * c - b * s, a * s + b * c]
    size = [(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()]
    got = got.double()
    first, second = ((got[..., :pairs], got[..., pairs:2 * pairs]) if layout == "half"
                     else (got[..., 0:2 * pairs:2], got[..., 1:2 * pairs:2]))
    for y, want, rough in ((first, z[0], size[0]), (second, z[1], size[1])):
        tol = 3 * 2.0 ** -24 * rough + (HALF_UNIT[x.dtype] * want.abs() + 2.0 ** -25 if x.dtype != F32 else 0.0)
        assert ((y - want).abs() <= tol).all()
    assert torch.equal(got[..., 2 * pairs:], x.double()[..., 2 * pairs:])


SHAPES = [  # tokens, heads, dim, axes
    (1, 1, 2, (1,)), (1, 32, 128, (16, 24, 24)), (5, 3, 80, (7, 1, 12)), (17, 7, 96, (24, 20, 4)), (3, 2, 130, (1, 63)),
    (33, 5, 512, (100, 56, 60, 40)), (1000, 9, 64, (8, 8, 16)), (2, 1, 14, (0, 3)), (40, 20, 96, (16, 0, 16, 16)),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("order", ["blocks", "cyclic"])
@pytest.mark.parametrize("tokens, heads, dim, axes", SHAPES)
def test_rotate_axes(dtype, layout, order, tokens, heads, dim, axes):
    g = generator(tokens * heads + dim)
    table = bfft.rotary_table(5000, 2 * sum(axes))
    x = normal(g, tokens, heads, dim, dtype=dtype)
    positions = torch.randint(0, 5000, (len(axes), tokens), device="cuda", generator=g)
    roots = token_table(table, positions, axes, order)
    y = bfft.rotate_positions(x, positions, table, layout=layout, axes=axes, axis_order=order)
    check_turned(y, x, roots, layout)
    where = torch.arange(tokens, device="cuda")
    assert torch.equal(y, bfft.rotate_positions(x, where, roots, layout=layout))
    back = bfft.rotate_positions(x, positions.int(), table, layout=layout, axes=axes, axis_order=order,
                                 transform_direction="inverse")
    check_turned(back, x, roots, layout, -1.0)
    same = positions[:1].expand(len(axes), tokens)             # one position on every axis, and a stride of 0
    assert torch.equal(bfft.rotate_positions(x, same, table, layout=layout, axes=axes, axis_order=order),
                       bfft.rotate_positions(x, positions[0], table, layout=layout))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotate_axes_batches_views_and_in_place(layout):
    g = generator(3)
    axes = (10, 11, 11)
    table = bfft.rotary_table(300, 64, amplitude=1.3, axes=axes, axis_order="cyclic", spectrum="axial")
    wide = normal(g, 2, 5, 11, 3 * 64, dtype=BF16)            # (batch, heads, tokens, packed q k v)
    x = wide[..., 64:128].transpose(1, 2)                      # heads before tokens, rows 192 apart
    rows = torch.randint(0, 300, (3, 2, 11), device="cuda", generator=g)
    how = {"layout": layout, "axes": axes, "axis_order": "cyclic"}
    y = bfft.rotate_positions(x, rows, table, **how)
    for b in range(2):
        check_turned(y[b], x[b], token_table(table, rows[:, b], axes, "cyclic"), layout)
    one = rows[:, 0]                                           # the same positions for the whole batch
    assert torch.equal(bfft.rotate_positions(x, one, table, **how),
                       bfft.rotate_positions(x, one[:, None].expand(3, 2, 11), table, **how))
    last = rows.permute(1, 2, 0).contiguous().permute(2, 0, 1)  # axes innermost in memory
    assert torch.equal(bfft.rotate_positions(x, last, table, **how), y)
    odd = normal(g, 11, 3, 65, dtype=BF16)[..., 1:]            # element-aligned rows only
    check_turned(bfft.rotate_positions(odd, one, table, **how), odd, token_table(table, one, axes, "cyclic"), layout)
    other = wide.clone()
    assert bfft.rotate_positions(x, rows, table, out=x, **how) is x
    assert torch.equal(x, y)
    assert torch.equal(wide[..., :64], other[..., :64]) and torch.equal(wide[..., 128:], other[..., 128:])
    assert bfft.rotate_positions(x[:, :0], rows[..., :0], table, **how).shape == (2, 0, 5, 64)
    assert bfft.rotate_positions(x, rows, table, layout=layout, axes=list(axes)).shape == x.shape  # a list will do


@pytest.mark.parametrize("order", ["blocks", "cyclic"])
def test_positions_outside_the_table_spoil_their_axis_only(order):
    axes = (3, 5)
    table = bfft.rotary_table(10, 16)
    x = normal(generator(1), 4, 2, 20)
    positions = torch.tensor([[-1, 3, 2 ** 40, 9], [0, 10, 4, -2 ** 33]], device="cuda")
    y = bfft.rotate_positions(x, positions, table, layout="interleaved", axes=axes, axis_order=order)
    bad = ((positions < 0) | (positions >= 10))[torch.tensor(dealt(axes, order), device="cuda")].T
    assert (y[..., :16].isnan() == bad.repeat_interleave(2, 1)[:, None]).all()
    assert torch.equal(y[..., 16:], x[..., 16:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("order", ["blocks", "cyclic"])
def test_rotate_axes_gradient(layout, order):
    g = generator(11)
    axes = (4, 5, 3)
    table = bfft.rotary_table(100, 24, amplitude=0.9)
    positions = torch.randint(0, 100, (3, 13), device="cuda", generator=g)
    how = {"layout": layout, "axes": axes, "axis_order": order}
    x = normal(g, 13, 3, 32).requires_grad_(True)
    w = normal(g, 13, 3, 32)
    dx, = torch.autograd.grad(bfft.rotate_positions(x, positions, table, **how), x, w)
    check_turned(dx, w, token_table(table, positions, axes, order), layout, -1.0)
    # differences: y is linear in x, so a step of any size gives the derivative but for roundings
    u = normal(g, 13, 3, 32)
    with torch.no_grad():
        ahead = bfft.rotate_positions(x + u, positions, table, **how).double()
        behind = bfft.rotate_positions(x - u, positions, table, **how).double()
    slope = ((ahead - behind) * w.double()).sum() / 2
    size = (w.double().abs() * (x.double().abs() + u.double().abs()).amax()).sum()
    assert abs(slope - (dx.double() * u.double()).sum()) <= 8 * 2.0 ** -24 * 2 * size
    # a broadcast input collects the heads' gradients; twice differentiable
    base = normal(g, 13, 1, 32).requires_grad_(True)
    y = bfft.rotate_positions(base.expand(13, 3, 32), positions, table, **how)
    db, = torch.autograd.grad(y.square().sum(), base, create_graph=True)
    # |y|^2 = 0.81 |x|^2 in the rotated part: the gradient is 6 * 0.81 x there, 6 x behind it
    slope = torch.where(torch.arange(32, device="cuda") < 24, 6 * 0.81, 6.0)
    assert torch.allclose(db, slope * base, rtol=1e-5, atol=1e-5)
    ddb, = torch.autograd.grad(db.sum(), base)
    assert torch.allclose(ddb, slope.expand_as(ddb), rtol=1e-5, atol=1e-5)


def test_backward_of_axes_in_a_graph_and_on_another_stream():
    g = generator(5)
    axes, table = (16, 24, 24), bfft.rotary_table(512, 128)
    positions = torch.randint(0, 512, (3, 50), device="cuda", generator=g)
    x = normal(g, 50, 4, 128, dtype=BF16).requires_grad_(True)
    w = normal(g, 50, 4, 128, dtype=BF16)

    def step():
        y = bfft.rotate_positions(x, positions, table, axes=axes)
        return y.detach(), *torch.autograd.grad(y, x, w)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        elsewhere = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, elsewhere):
        assert torch.equal(a, b) and torch.equal(a, c)


# ------------------------------------------------------------------------------- append

@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("order", ["blocks", "cyclic"])
@pytest.mark.parametrize("dtype, layout, page, heads, dim, axes, q_heads", [
    (BF16, "half", 64, 8, 128, (16, 24, 24), 32), (F16, "interleaved", 32, 3, 96, (10, 7, 7), 9),
    (F32, "half", 16, 1, 16, (1, 1), 1), (BF16, "half", 128, 2, 80, (5, 5, 5, 5), 4),
    (F32, "interleaved", 16, 5, 256, (128,), 0), (BF16, "interleaved", 16, 1, 48, (20, 3), 3),
    (F16, "half", 64, 2, 64, (16, 16), 40),
])
@pytest.mark.parametrize("new", [[1, 63, 1, 100, 2, 0, 64], [1, 1, 1, 1, 1, 1, 1], [0, 300, 0, 0, 411, 90, 120]])
def test_append_axes(code, order, dtype, layout, page, heads, dim, axes, q_heads, new):
    held = [0, 1, page - 1, page, 2 * page + 5, 7, 300]
    kw = {"code": code, "page": page, "heads": heads, "dim": dim}
    a, b = (Pages(dim + page, held, [2 * n for n in new], **kw) for _ in range(2))
    table = bfft.rotary_table(4096, 2 * sum(axes))
    tokens, starts = sum(new), ints(cumulative(new))
    for turn in range(2):
        positions = torch.randint(0, 4096, (len(axes), tokens), device="cuda", generator=a.g)
        if turn:
            positions = positions.int()
        packed = normal(a.g, tokens, q_heads + 2 * heads, dim + 16, dtype=dtype)[..., :dim] * (1 + 3 * turn)
        q, k, v = packed.split([q_heads, heads, heads], 1)
        q = q if q_heads else None
        got = bfft.append_rotated(a.cache, k, v, a.table, ints(held), starts, table, layout=layout, positions=positions,
                                  axes=axes, axis_order=order, q=q)
        roots = token_table(table, positions, axes, order)
        want = bfft.append_rotated(b.cache, k, v, b.table, ints(held), starts, roots, layout=layout,
                                   positions=torch.arange(tokens, device="cuda"), q=q)
        for x, y in zip(a.cache, b.cache):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        if q_heads:
            assert torch.equal(got, want)
            check_turned(got, q, roots, layout)
        held = [h + n for h, n in zip(held, new)]


def test_append_axes_outside_the_table():
    p = Pages(4, [0, 3], [2, 2], code="int8", page=16, heads=2, dim=32)
    k = normal(p.g, 2, 2, 32, dtype=BF16)
    table = bfft.rotary_table(8, 32)
    positions = ints([[1, 8], [2, 2]])
    q = bfft.append_rotated(p.cache, k, k, p.table, ints([0, 3]), ints([0, 1, 2]), table, positions=positions,
                            axes=(8, 8), q=k)
    assert q[0].isfinite().all()
    assert (q[1].isnan() == (torch.arange(32, device="cuda") % 16 < 8)).all()
    assert p.values(0, 0, 0, 1)[0].isfinite().all() and p.values(1, 1, 0, 4)[0].isfinite().all()
    assert p.values(0, 1, 0, 4)[0].isnan().all()              # the block of the token's keys reads as NaN


# ------------------------------------------------------------------------------- refusals

def test_refusals_of_axes_come_before_any_launch():
    p = Pages(1, [20, 3], [4, 4], code="int8", page=16, heads=2, dim=32)
    table, one, held = bfft.rotary_table(64, 32), ints([0, 1, 2]), ints([20, 3])
    x = normal(p.g, 2, 2, 32, dtype=BF16)
    positions = ints([[1, 2], [3, 4], [5, 6]])
    count = _lib.launch_counter()

    def refuses(exc, fn, *args, **kw):
        with pytest.raises(exc):
            fn(*args, **kw)

    rot, app = bfft.rotate_positions, bfft.append_rotated
    for bad in ((8, 8), (4, 4, 4, 4, 0), (), (4, 4, -1, 9), (4.0, 6, 6), (6, 6, 5), (True, 9, 6), 16, "axes"):
        refuses((ValueError, TypeError), rot, x, positions, table, axes=bad)
        refuses((ValueError, TypeError), app, p.cache, x, x, p.table, held, one, table, positions=positions, axes=bad)
    axes = (4, 6, 6)
    refuses(ValueError, rot, x, positions, table, axes=axes, axis_order="spiral")
    refuses(ValueError, rot, x, positions[:2], table, axes=axes)
    refuses(ValueError, rot, x, positions[0], table, axes=axes)
    refuses(ValueError, rot, x, positions[:, :1], table, axes=axes)
    refuses(ValueError, rot, x, positions[:, None], table, axes=axes)        # a batch that x lacks
    refuses(ValueError, rot, x, positions, table)
    refuses(TypeError, rot, x, positions.float(), table, axes=axes)
    refuses(ValueError, rot, x, positions.cpu(), table, axes=axes)
    refuses(ValueError, rot, x.float().requires_grad_(True), positions, table, axes=axes, out=x.float())
    refuses(ValueError, app, p.cache, x, x, p.table, held, one, table, axes=axes)              # no positions
    refuses(ValueError, app, p.cache, x, x, p.table, held, one, positions=positions, axes=axes)  # no table
    refuses(ValueError, app, p.cache, x, x, p.table, held, one, table, positions=positions)
    refuses(ValueError, app, p.cache, x, x, p.table, held, one, table, positions=positions[:2], axes=axes)
    refuses(ValueError, app, p.cache, x, x, p.table, held, one, table, positions=positions.T.contiguous().T, axes=axes)
    assert _lib.launch_counter() == count
    assert app(p.cache, x[:0], x[:0], p.table, held, ints([0, 0, 0]), table, positions=positions[:, :0], axes=axes) is None


def test_the_calls_of_one_axis_are_those_of_equal_positions():
    """axes of one entry, and the C entry point with a map of its own, name the same rows as a plain call."""
    g = generator(2)
    table, x = bfft.rotary_table(50, 16), normal(g, 6, 2, 16)
    where = torch.randint(0, 50, (6,), device="cuda", generator=g).int()
    want = bfft.rotate_positions(x, where, table)
    assert torch.equal(bfft.rotate_positions(x, where[None], table, axes=(8,)), want)
    lib = _lib.load()
    cache._load()
    import ctypes
    axis = (ctypes.c_uint8 * 8)(1, 0, 1, 1, 0, 0, 1, 0)
    pos = torch.stack((where, where.flip(0))).contiguous()
    desc = struct.pack("19q", 1, 6, 2, 16, 16, 0, 32, 16, 0, 32, 16, 0, 1, 50, 0, 0, 0, 0, 0)
    y = torch.empty_like(x)
    assert lib.bfft_rotate_axes(desc, struct.pack("Qqq", ctypes.addressof(axis), 2, 6), x.data_ptr(), pos.data_ptr(),
                                table.data_ptr(), y.data_ptr(), torch.cuda.current_stream().cuda_stream) == _lib.OK
    roots = table[pos.long()[torch.tensor(list(axis))].T, torch.arange(8, device="cuda")]
    check_turned(y, x, roots, "half")
    assert math.isfinite(float(y.sum()))

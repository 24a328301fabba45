"""Position and cache calls on each path that the plans can take: the row tiles with windows, odd scales, direct
output and odd strides, and the append by runs with all types, layouts and packs.

Each test says by the plan's own rule that it gets to the path it names.
"""
import pytest
import torch

import bfft
from test_gpu_cache import (BF16, F16, F32, MOST, Pages, check_attention, check_rotated, code_error, cumulative, ints,
                            normal, rotate64)
from test_gpu_cache_edges import check_relative, takes_tiles

pytestmark = pytest.mark.gpu

SMS = 148


def tiles_chunks(p, q, table, group):
    """Chunks of the axis by the plan of the row tiles, without a window."""
    units = -(-q.shape[0] // (256 // group)) * p.heads
    chunk = max(512, -(-table.shape[1] * p.page // (1 if units >= SMS else SMS // units)))
    return -(-table.shape[1] * p.page // (-(-chunk // 128) * 128))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype, page, dim, group, window", [
    (BF16, 16, 64, 8, 129), (F16, 64, 128, 4, 517), (BF16, 128, 96, 4, 1000), (BF16, 32, 48, 16, 200), (F16, 16, 128, 8, 64),
    (BF16, 64, 80, 5, 3000),
])
def test_tiles_with_a_window(code, dtype, page, dim, group, window):
    lens, new = [4100, 0, 1333, 77], [2000, 60, 1000, 77]
    p = Pages(dim + page, lens, [0] * 4, code=code, page=page, heads=2, dim=dim)
    q = normal(p.g, sum(new), 2 * group, dim, dtype=dtype) * 1.5
    assert takes_tiles(p, q, new, p.table, window=window)
    check_attention(p, q, lens, new, window=window)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dim, page, window", [(64, 16, 33), (128, 64, 700), (112, 128, 5000)])
def test_tiles_that_see_behind_themselves(code, dim, page, window):
    """Rows that are not causal see from their window's first token to the sequence's end."""
    lens, new = [4100, 333], [600, 333]
    p = Pages(dim, lens, [0] * 2, code=code, page=page, heads=2, dim=dim)
    q = normal(p.g, sum(new), 8, dim, dtype=BF16)
    assert takes_tiles(p, q, new, p.table, causal=False, window=window)
    check_attention(p, q, lens, new, causal=False, window=window)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0, 1e-4])
@pytest.mark.parametrize("new", [[300], [4100]])
def test_tiles_with_scales_over_decades(code, scale, new):
    p = Pages(78, [4100], [0], code=code, page=32, heads=2, dim=128)
    p.cache.v_scale.mul_(torch.logspace(-6, 6, p.cache.v_scale.numel(), device="cuda").view_as(p.cache.v_scale))
    p.cache.v_scale[p.ids[0][3]] = 0.0                       # zero values count in the sum, and as 2^-64 in the maximum
    q = normal(p.g, new[0], 8, 128, dtype=BF16)
    check_relative(p, q, [4100], new, tiles=True, scale=scale, zero_as=2.0 ** -64)


@pytest.mark.parametrize("dtype, page, dim, group, rows", [
    (BF16, 64, 128, 4, 4100), (F16, 16, 64, 4, 4100), (BF16, 128, 96, 2, 9000), (F16, 32, 16, 32, 1000),
])
def test_tiles_write_their_rows_themselves(dtype, page, dim, group, rows):
    """One chunk: no joining kernel; rows of q and of out that start on any element."""
    lens = [rows + 50]
    p = Pages(dim, lens, [0], code="int8", page=page, heads=2, dim=dim)
    q = normal(p.g, rows, 2 * group, dim, dtype=dtype)
    assert takes_tiles(p, q, [rows], p.table) and tiles_chunks(p, q, p.table, group) == 1
    want, want_lse = check_attention(p, q, lens, [rows])
    odd = torch.zeros(rows, 2 * group, dim + 3, dtype=dtype, device="cuda")
    odd[..., 1:dim + 1] = q
    out = torch.full((rows, 2 * group, dim + 1), 7.0, dtype=dtype, device="cuda")
    got, lse = bfft.cache_attention(odd[..., 1:dim + 1], p.cache, p.table, ints(lens), ints([0, rows]), return_lse=True,
                                    out=out[..., 1:])
    assert torch.equal(got, want) and torch.equal(lse, want_lse) and (out[..., 0] == 7).all()
    assert bfft.cache_attention(q, p.cache, p.table, ints(lens), ints([0, rows]), out=q) is not None
    assert torch.equal(q, want)                              # in place


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("new, tiles", [([1], False), ([300], True), ([4100], True)])
def test_values_near_the_largest_float(code, new, tiles):
    p = Pages(79, [4100], [0], code=code, page=32, heads=2, dim=128)
    p.cache.v_scale.mul_(1e34)
    q = normal(p.g, new[0], 8, 128, dtype=BF16)
    out, _ = check_relative(p, q, [4100], new, tiles=tiles)
    assert out.abs().amax() > 1e33


@pytest.mark.parametrize("dim, heads, group, rows", [(64, 1, 129, 70), (256, 2, 4, 200), (144, 1, 40, 130)])
def test_prompts_that_the_tiles_do_not_take(dim, heads, group, rows):
    lens, new = [1500, 90], [rows, 30]
    p = Pages(dim, lens, [0] * 2, code="e4m3", page=32, heads=heads, dim=dim)
    q = normal(p.g, sum(new), heads * group, dim, dtype=BF16)
    assert not takes_tiles(p, q, new, p.table)
    check_attention(p, q, lens, new)
    check_attention(p, q, lens, new, window=100)


# ------------------------------------------------------------------------------- append by runs

def append_and_check(p, new, *, dtype=BF16, layout="half", rotated=0, q_heads=0, given=False, factor=1.0):
    """Appends random rows by runs.  A value is off by its code's error and, as codes are chosen from the rotated
    value in 32 bits, by the rotation's roundings: 3 * 2^-24 of |a c| + |b s|."""
    tokens, slots = sum(new), sum(new) // p.page + 2 * len(new)
    assert tokens > slots and tokens >= 48 * len(new) and slots * 2 * p.heads < 4096   # by runs, not by tokens or warps
    table = bfft.rotary_table(4096, rotated) if rotated else None
    packed = (normal(p.g, tokens, q_heads + 2 * p.heads, p.dim + 16, dtype=dtype) * factor)[..., :p.dim]
    q, k, v = packed.split([q_heads, p.heads, p.heads], 1)
    starts = cumulative(new)
    place = torch.cat([torch.arange(h, h + n) for h, n in zip(p.held, new)]).cuda()
    at = torch.randint(0, 4096, (tokens,), device="cuda", generator=p.g) if given else place
    old = [[p.values(w, s, 0, h) for s, h in enumerate(p.held)] for w in (0, 1)]
    before = [t.clone() for t in p.cache]
    got_q = bfft.append_rotated(p.cache, k, v, p.table, ints(p.held), ints(starts), table, layout=layout,
                                positions=at if given else None, q=q if q_heads else None)
    if q_heads and rotated:
        check_rotated(got_q, q, at, table, layout)
    elif q_heads:
        assert torch.equal(got_q, q)
    keys, size = rotate64(k, at, table, layout) if rotated else (k.double(), torch.zeros_like(k.double()))
    for w, x, rough in ((0, keys, 3 * 2.0 ** -24 * size), (1, v.double(), torch.zeros_like(size))):
        written = torch.zeros(before[w].shape[0], p.page, dtype=torch.bool, device="cuda")
        for s, (h, n) in enumerate(zip(p.held, new)):
            rows = slice(starts[s], starts[s + 1])
            got, scale = p.values(w, s, h, n)
            error = code_error(p.code, x[rows], scale[..., None]) + 2.0 ** -22 * x[rows].abs() + rough[rows]
            assert ((got - x[rows]).abs() <= error).all()
            first = h - h % p.page
            kept, now = p.values(w, s, first, h - first)
            was, then = old[w][s][0][first:], old[w][s][1][first:]
            grown = (now != then)[..., None]
            assert (now >= then).all()
            assert ((kept - was).abs() <= torch.where(grown, code_error(p.code, was, now[..., None]), 0.0)).all()
            assert torch.equal(p.values(w, s, 0, first)[0], old[w][s][0][:first])
            for page in range(first // p.page, (h + n - 1) // p.page + 1):
                a, b = max(h, page * p.page), min(h + n, (page + 1) * p.page)
                top = x[rows][a - h:b - h].abs().amax((0, 2)) / MOST[p.code]
                if a > page * p.page:
                    top = torch.maximum(top, old[w][s][1][a - 1])
                assert ((p.cache[2 + w][p.ids[s][page]].double() - top).abs() <= 2.0 ** -22 * top).all()
                written[p.ids[s][page], :b - page * p.page] = True
        same = before[w].view(torch.uint8) == p.cache[w].view(torch.uint8)
        assert same.transpose(1, 2)[~written].all()           # free slots and other pages keep their bytes
        others = ~written.any(1)
        assert torch.equal(before[2 + w][others], p.cache[2 + w][others])
    p.held = [h + n for h, n in zip(p.held, new)]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype, page, heads, dim, rotated, q_heads", [
    (BF16, 64, 2, 128, 128, 8), (F16, 16, 3, 80, 40, 9), (F32, 32, 2, 64, 48, 4), (BF16, 128, 2, 48, 44, 3),
    (F16, 64, 1, 48, 46, 1), (F32, 16, 5, 96, 0, 0), (BF16, 32, 1, 256, 254, 40), (F32, 64, 4, 16, 6, 17),
    (F16, 128, 9, 32, 32, 64),
])
@pytest.mark.parametrize("given", [False, True])
def test_append_of_long_runs(code, layout, dtype, page, heads, dim, rotated, q_heads, given):
    held, new = [0, 5, page + 3, 2 * page - 1], [700, 3, 200, 4 * page + 1]
    p = Pages(dim + page, held, new, code=code, page=page, heads=heads, dim=dim)
    append_and_check(p, new, dtype=dtype, layout=layout, rotated=rotated, q_heads=q_heads, given=given)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_of_long_runs_makes_scales_grow(code):
    p = Pages(50, [10, 77], [3000, 3000], code=code, page=64, heads=2, dim=64)
    append_and_check(p, [300, 400], rotated=64, q_heads=4)
    append_and_check(p, [500, 150], rotated=64, q_heads=4, factor=8.0)   # pages begun by the call before get larger rows
    append_and_check(p, [120, 333], rotated=64, q_heads=4, factor=0.125)

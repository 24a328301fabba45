"""Rotation by position and the paged 8-bit cache against plain float64 forms.

Tolerances come from the roundings that each result goes through: a product or a
sum in 32 bits is off by 2^-24 of its size, a value rounded to float16 / bfloat16
by 2^-11 / 2^-8 at most of half a unit (2^-12, 2^-9 would hold for the middle of a
binade), an int8 code by half the block's scale, an e4m3 code by 2^-4 of the value
or, below its smallest normal, by 2^-10 of the scale.
"""
import math

import pytest
import torch

import bfft
from bfft import _lib

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF_UNIT = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
MOST = {"int8": 127.0, "e4m3": 448.0}


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=F32):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def rotate64(x, positions, table, layout, sign=1.0):
    """x (..., tokens, heads, dim) and a bound of each value's size |a c| + |b s|, both float64."""
    x, t = x.double(), table.double()[positions.long()]
    c, s = t[..., None, :, 0], sign * t[..., None, :, 1]
    r = 2 * table.shape[1]
    part = x[..., :r]
    a, b = (part[..., :r // 2], part[..., r // 2:]) if layout == "half" else (part[..., 0::2], part[..., 1::2])
    out, size = [], []
    for u, v in ((a * c - b * s, (a * c).abs() + (b * s).abs()), (a * s + b * c, (a * s).abs() + (b * c).abs())):
        out.append(u)
        size.append(v)

    def join(p):
        return torch.cat(p, -1) if layout == "half" else torch.stack(p, -1).flatten(-2)

    rest = x[..., r:]
    return torch.cat((join(out), rest), -1), torch.cat((join(size), torch.zeros_like(rest)), -1)


def check_rotated(got, x, positions, table, layout, sign=1.0):
    want, size = rotate64(x, positions, table, layout, sign)
    tol = 3 * 2.0 ** -24 * size + (HALF_UNIT[got.dtype] * want.abs() + 2.0 ** -25 if got.dtype != F32 else 0.0)
    assert got.shape == x.shape and got.dtype == x.dtype
    assert ((got.double() - want).abs() <= tol).all()


# ------------------------------------------------------------------------------- rotation

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens, heads, dim, rotated", [
    (1, 1, 2, 2), (1, 32, 128, 128), (5, 3, 80, 40), (17, 7, 96, 64), (3, 2, 130, 126), (33, 5, 512, 512),
    (1000, 9, 64, 32), (2, 1, 14, 6),
])
def test_rotate(dtype, layout, tokens, heads, dim, rotated):
    g = generator(tokens * heads + dim)
    table = bfft.rotary_table(5000, rotated)
    x = normal(g, tokens, heads, dim, dtype=dtype)
    positions = torch.randint(0, 5000, (tokens,), device="cuda", generator=g)
    check_rotated(bfft.rotate_positions(x, positions, table, layout=layout), x, positions, table, layout)
    back = bfft.rotate_positions(x, positions.int(), table, layout=layout, transform_direction="inverse")
    check_rotated(back, x, positions, table, layout, -1.0)
    if rotated < dim:
        assert torch.equal(back[..., rotated:], x[..., rotated:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotate_batches_views_and_in_place(layout):
    g = generator(3)
    table = bfft.rotary_table(300, 64, amplitude=1.3)
    wide = normal(g, 2, 5, 11, 3 * 64, dtype=BF16)           # (batch, heads, tokens, packed q k v)
    x = wide[..., 64:128].transpose(1, 2)                     # heads before tokens, rows 192 apart
    rows = torch.randint(0, 300, (2, 11), device="cuda", generator=g)
    y = bfft.rotate_positions(x, rows, table, layout=layout)
    check_rotated(y, x, rows, table, layout)
    one = torch.arange(11, device="cuda")
    check_rotated(bfft.rotate_positions(x, one, table, layout=layout), x, one.expand(2, 11), table, layout)
    odd = normal(g, 7, 3, 65, dtype=BF16)[..., 1:]            # element-aligned rows only
    check_rotated(bfft.rotate_positions(odd, one[:7], table, layout=layout), odd, one[:7], table, layout)
    want = bfft.rotate_positions(x, rows, table, layout=layout)
    other = wide.clone()
    assert bfft.rotate_positions(x, rows, table, layout=layout, out=x) is x
    assert torch.equal(x, want)
    assert torch.equal(wide[..., :64], other[..., :64]) and torch.equal(wide[..., 128:], other[..., 128:])
    none = x[:, :0]
    assert bfft.rotate_positions(none, rows[:, :0], table, layout=layout).shape == none.shape


def test_rotate_positions_outside_the_table_are_nan():
    table = bfft.rotary_table(10, 16)
    x = normal(generator(1), 4, 2, 20)
    y = bfft.rotate_positions(x, torch.tensor([-1, 10, 2**40, 3], device="cuda"), table)
    assert y[:3, :, :16].isnan().all() and torch.equal(y[:, :, 16:], x[:, :, 16:]) and y[3].isfinite().all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotate_gradient(layout):
    g = generator(11)
    table = bfft.rotary_table(100, 24, amplitude=0.9)
    positions = torch.randint(0, 100, (13,), device="cuda", generator=g)
    x = normal(g, 13, 3, 32).requires_grad_(True)
    w = normal(g, 13, 3, 32)
    y = bfft.rotate_positions(x, positions, table, layout=layout)
    dx, = torch.autograd.grad(y, x, w)
    check_rotated(dx, w, positions, table, layout, -1.0)
    # differences: y is linear in x, so a step of any size gives the derivative but for roundings
    u = normal(g, 13, 3, 32)
    with torch.no_grad():
        ahead = bfft.rotate_positions(x + u, positions, table, layout=layout).double()
        behind = bfft.rotate_positions(x - u, positions, table, layout=layout).double()
    slope = ((ahead - behind) * w.double()).sum() / 2
    size = (w.double().abs() * (x.double().abs() + u.double().abs()).amax()).sum()
    assert abs(slope - (dx.double() * u.double()).sum()) <= 8 * 2.0 ** -24 * 2 * size
    # a broadcast input collects the heads' gradients; an expanded gradient (sum) has no adjacent elements
    base = normal(g, 13, 1, 32).requires_grad_(True)
    got, = torch.autograd.grad(bfft.rotate_positions(base.expand(13, 3, 32), positions, table, layout=layout).sum(), base)
    want, size = rotate64(torch.ones(13, 3, 32, device="cuda"), positions, table, layout, -1.0)
    assert ((got.double() - want.sum(1, keepdim=True)).abs() <= 8 * 2.0 ** -24 * (size.sum(1, keepdim=True) + 3)).all()


def test_rotate_twice_differentiable():
    table = bfft.rotary_table(8, 8)
    x = normal(generator(5), 4, 1, 8).requires_grad_(True)
    y = bfft.rotate_positions(x, torch.arange(4, device="cuda"), table)
    dx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    ddx, = torch.autograd.grad(dx.sum(), x)
    assert torch.allclose(dx, 2 * x, atol=1e-5) and torch.allclose(ddx, torch.full_like(x, 2.0), atol=1e-5)


# ------------------------------------------------------------------------------- cache

class Pages:
    """A cache whose sequences hold `held` tokens of known values, on scattered pages."""

    def __init__(self, seed, held, room, *, code, page, heads, dim, spare=2):
        g = self.g = generator(seed)
        self.code, self.page, self.heads, self.dim, self.held = code, page, heads, dim, held
        need = [max(1, -(-(h + r) // page)) for h, r in zip(held, room)]
        total = sum(need) + spare
        self.cache = bfft.paged_cache(total, heads, page, dim, code=code)
        for codes, scale in zip(self.cache[:2], self.cache[2:]):
            fill = torch.randn(codes.shape, device="cuda", generator=g) * MOST[code] / 3
            fill = (fill.round() if code == "int8" else fill).clamp(-MOST[code], MOST[code])
            codes.copy_(fill.to(codes.dtype))
            scale.copy_((1 + torch.rand(scale.shape, device="cuda", generator=g)) * 3 / MOST[code])
        ids = torch.randperm(total, device="cuda", generator=g).tolist()
        table, at = [], 0
        for n in need:
            table.append(ids[at:at + n] + [-1] * (max(need) - n))  # entries behind a sequence's pages are no pages
            at += n
        self.ids, self.table = table, ints(table)

    def values(self, which, s, first, count):
        """(count, heads, dim) float64 values of sequence s, and their blocks' scales."""
        codes, scale = self.cache[which], self.cache[2 + which]
        at = torch.arange(first, first + count)
        page = torch.tensor(self.ids[s], dtype=torch.long)[at // self.page].cuda()
        slot = (at % self.page).cuda()
        sc = scale.double()[page]
        return codes.view(torch.uint8)[page, :, slot].view(codes.dtype).double() * sc[..., None], sc


def code_error(code, value, scale):
    """Largest error of a value held as a code of its block."""
    half = 0.5 * scale if code == "int8" else torch.maximum(2.0 ** -4 * value.abs(), 2.0 ** -10 * scale)
    return half * (1 + 2.0 ** -18)


def cumulative(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def appended(p, new, *, dtype=BF16, layout="half", rotated=None, q_heads=0, positions=None, strided=False, scale=1.0):
    """Appends random rows and checks codes, scales and what else the pages held."""
    g, dim, heads = p.g, p.dim, p.heads
    table = bfft.rotary_table(4096, rotated) if rotated else None
    tokens = sum(new)
    if strided:
        packed = normal(g, tokens, q_heads + 2 * heads, dim + 16, dtype=dtype)[..., :dim]
        q, k, v = packed.split([q_heads, heads, heads], 1)
    else:
        q, k, v = (normal(g, tokens, n, dim, dtype=dtype) for n in (q_heads, heads, heads))
    k, v = k * scale if scale != 1.0 else k, v
    starts = cumulative(new)
    at = torch.cat([torch.arange(h, h + n) for h, n in zip(p.held, new)]).cuda() if tokens else ints([]).long()
    at = at if positions is None else positions
    before = [t.clone() for t in p.cache]
    old = [[p.values(w, s, 0, h) for s, h in enumerate(p.held)] for w in (0, 1)]
    q_out = bfft.append_rotated(p.cache, k, v, p.table, ints(p.held), ints(starts), table, layout=layout,
                                positions=positions, q=q if q_heads else None)
    if q_heads:
        check_rotated(q_out, q, at, table, layout) if rotated else None
    want = [rotate64(k, at, table, layout)[0] if rotated else k.double(), v.double()]
    for w in (0, 1):
        touched = torch.zeros(before[w].shape[:1] + (p.page,), dtype=torch.bool, device="cuda")
        owned = torch.zeros(before[w].shape[0], dtype=torch.bool, device="cuda")
        for s, (h, n) in enumerate(zip(p.held, new)):
            if not n:
                continue
            got, sc = p.values(w, s, h, n)
            x = want[w][starts[s]:starts[s] + n]
            assert ((got - x).abs() <= code_error(p.code, x, sc[..., None]) + 2.0 ** -22 * x.abs()).all()
            first = h - h % p.page
            kept, ksc = p.values(w, s, first, h - first)
            was, wsc = old[w][s][0][first:], old[w][s][1][first:]
            grown = (ksc != wsc)[..., None]
            assert (ksc >= wsc).all()
            assert ((kept - was).abs() <= torch.where(grown, code_error(p.code, was, ksc[..., None]), 0.0)).all()
            if first:
                assert torch.equal(p.values(w, s, 0, first)[0], old[w][s][0][:first])
            for page in range(first // p.page, (h + n - 1) // p.page + 1):
                a, b = max(h, page * p.page), min(h + n, (page + 1) * p.page)
                top = want[w][starts[s] + a - h:starts[s] + b - h].abs().amax((0, 2)) / MOST[p.code]
                if a > page * p.page:
                    top = torch.maximum(top, old[w][s][1][a - 1])
                sc = p.cache[2 + w][p.ids[s][page]].double()
                assert ((sc - top).abs() <= 2.0 ** -22 * top).all()
                touched[p.ids[s][page], :b - page * p.page] = True
                owned[p.ids[s][page]] = True
        same = before[w].view(torch.uint8) == p.cache[w].view(torch.uint8)
        assert same.transpose(1, 2)[~touched].all()          # free slots and other pages keep their bytes
        assert torch.equal(before[2 + w][~owned], p.cache[2 + w][~owned])
    p.held = [h + n for h, n in zip(p.held, new)]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype, layout, page, heads, dim, rotated, q_heads", [
    (BF16, "half", 64, 8, 128, 128, 32), (F16, "interleaved", 32, 3, 96, 48, 9), (F32, "half", 16, 1, 16, 4, 1),
    (BF16, "half", 128, 2, 80, 40, 4), (F32, "interleaved", 16, 5, 256, 256, 0), (F16, "half", 64, 2, 64, 0, 0),
    (BF16, "interleaved", 16, 1, 48, 46, 3),
])
def test_append(code, dtype, layout, page, heads, dim, rotated, q_heads):
    held = [0, 1, page - 1, page, 2 * page + 5, 7, 300]
    new = [1, page - 1, 1, 3 * page + 1, 2, 0, page]
    p = Pages(dim + page, held, [n + 2 for n in new], code=code, page=page, heads=heads, dim=dim)
    appended(p, new, dtype=dtype, layout=layout, rotated=rotated, q_heads=q_heads, strided=True)
    appended(p, [1, 0, 2, 1, 1, 1, 2], dtype=dtype, layout=layout, rotated=rotated, q_heads=q_heads, scale=4.0)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_token_by_token_many_sequences(code):
    p = Pages(9, [0] * 37, [40] * 37, code=code, page=32, heads=2, dim=64)
    rows = []
    for i in range(34):
        k = normal(p.g, 37, 2, 64, dtype=BF16) * (1 + i / 8)
        rows.append(k)
        bfft.append_rotated(p.cache, k, k, p.table, ints([i] * 37), ints(list(range(38))))
    for s in range(0, 37, 9):
        x = torch.stack([r[s] for r in rows]).double()
        for w in (0, 1):
            got, sc = p.values(w, s, 0, 34)
            # each of the times that the scale grew may have rounded a code once more
            growths = sum(bool(x[i].abs().amax() > x[:i].abs().amax()) for i in range(1, 34))
            assert ((got - x).abs() <= (growths + 1) * code_error(code, x, sc[..., None]) * 1.2).all()


def test_append_zero_nan_and_infinite_rows():
    p = Pages(4, [0, 3, 5, 0], [2] * 4, code="int8", page=16, heads=2, dim=32)
    k = normal(p.g, 4, 2, 32)
    k[0] = 0.0
    k[1, 0, 3] = math.nan
    k[2, 1, 0] = -math.inf
    k[3] = 1e-42                                             # below every scale that is kept: zero
    bfft.append_rotated(p.cache, k, k, p.table, ints(p.held), ints([0, 1, 2, 3, 4]))
    got = [p.values(0, s, 0, h + 1)[0] for s, h in enumerate(p.held)]
    assert (got[0] == 0).all() and (got[3] == 0).all()
    assert got[1][:, 0].isnan().all() and got[1][:, 1].isfinite().all()
    assert got[2][:, 1].isnan().all() and got[2][:, 0].isfinite().all()


def test_append_drops_rows_without_a_page():
    p = Pages(6, [0, 10], [40, 6], code="e4m3", page=16, heads=1, dim=16)
    table = p.table.clone()
    table[0, 1] = 10 ** 6                                    # no such page
    before = [t.clone() for t in p.cache]
    k = normal(p.g, 60, 1, 16)
    bfft.append_rotated(p.cache, k, k, table, ints([0, 10]), ints([0, 40, 60]))
    keep = torch.ones(before[0].shape[0], dtype=torch.bool, device="cuda")
    keep[[p.ids[0][0], p.ids[0][2], p.ids[1][0]]] = False
    for a, b in zip(before, p.cache):
        assert torch.equal(a[keep].view(torch.uint8) if a.dim() == 4 else a[keep],
                           b[keep].view(torch.uint8) if b.dim() == 4 else b[keep])
    assert p.values(0, 0, 0, 16)[0].isfinite().all()


def test_append_at_given_positions():
    p = Pages(8, [4, 0], [3, 20], code="int8", page=16, heads=2, dim=64)
    positions = torch.randint(0, 4096, (23,), device="cuda", generator=p.g)
    appended(p, [3, 20], rotated=64, q_heads=4, positions=positions)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_read(code, dtype):
    p = Pages(12, [70, 1, 33, 200], [0] * 4, code=code, page=32, heads=3, dim=48)
    first, count = [0, 0, 31, 7], [70, 0, 2, 193]
    k, v = bfft.read_cache(p.cache, p.table, ints(first), ints(cumulative(count)), sum(count), dtype=dtype)
    for w, got in enumerate((k, v)):
        want = torch.cat([p.values(w, s, f, n)[0] for s, (f, n) in enumerate(zip(first, count))])
        # code * scale is rounded to 32 bits, then once more to dtype
        assert ((got.double() - want).abs() <= (2.0 ** -24 + HALF_UNIT[dtype]) * want.abs() + 2.0 ** -25).all()
    k, v = bfft.read_cache(p.cache, p.table, ints([60, 0, 0, 0]), ints([0, 50, 50, 50, 50]), 50, dtype=dtype)
    assert k[:36].isfinite().all() and k[36:].isnan().all() and v[36:].isnan().all()


# ------------------------------------------------------------------------------- attention

def attention64(p, q, lens, starts, *, scale, causal, window):
    """out, lse, sum p |v| of each value, and a bound of the scores' rounding, all float64."""
    tokens, q_heads, dim = q.shape
    out = torch.zeros(tokens, q_heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((tokens, q_heads), -math.inf, dtype=torch.float64, device="cuda")
    size, slack = torch.zeros_like(out), torch.zeros_like(lse)
    for s, n in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        if b == a or n <= 0:
            continue
        k, v = p.values(0, s, 0, n)[0], p.values(1, s, 0, n)[0]
        group = q_heads // p.heads
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        x = q[a:b].double()
        z = torch.einsum("qhd,khd->hqk", x, k) * scale
        rough = torch.einsum("qhd,khd->hqk", x.abs(), k.abs()) * abs(scale)
        pos = torch.arange(n - (b - a), n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        seen = key <= pos if causal else torch.ones(b - a, n, dtype=torch.bool, device="cuda")
        if window:
            seen = seen & (key > pos - window)
        z = z.masked_fill(~seen, -math.inf)
        l = torch.logsumexp(z, -1)
        w = torch.exp(z - l[..., None]).masked_fill(~seen, 0.0).nan_to_num(0.0)
        out[a:b] = torch.einsum("hqk,khd->qhd", w, v)
        size[a:b] = torch.einsum("hqk,khd->qhd", w, v.abs())
        lse[a:b] = l.T
        slack[a:b] = rough.masked_fill(~seen, 0.0).amax(-1).T
    return out, lse, size, slack


def check_attention(p, q, lens, new, *, scale=None, causal=True, window=0, table=None):
    starts = cumulative(new)
    got, lse = bfft.cache_attention(q, p.cache, p.table if table is None else table, ints(lens), ints(starts),
                                    softmax_scale=scale, causal=causal, window=window, return_lse=True)
    factor = p.dim ** -0.5 if scale is None else scale
    want, want_lse, size, slack = attention64(p, q, lens, starts, scale=factor, causal=causal, window=window)
    empty = want_lse == -math.inf
    assert (got[empty] == 0).all() and (lse[empty] == -math.inf).all()
    # a score is off by some 2^-22 of sum |q||k| (32-bit sums, rounded factors), a weight by e^that, by the
    # exponential's 2^-22 and, where matrix products take it, by 2^-11 (float16); then the output's own rounding
    delta = 2.0 ** -21 * (1 + slack)
    tol = HALF_UNIT[q.dtype] * want.abs() + (2.0 ** -10 + 2 * delta[..., None]) * size + 2.0 ** -24
    assert ((got.double() - want).abs() <= tol).all()
    off = (lse.double() - want_lse).abs()[~empty]
    assert (off <= delta[~empty] + 2.0 ** -20 * (1 + want_lse[~empty].abs())).all()
    return got, lse


SHAPES = [  # page, kv heads, group, dim
    (64, 2, 4, 128), (16, 1, 1, 16), (32, 3, 5, 80), (128, 1, 8, 64), (16, 2, 16, 256), (64, 1, 33, 96), (32, 2, 2, 128),
]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("page, heads, group, dim", SHAPES)
def test_attention_single_tokens(code, dtype, page, heads, group, dim):
    lens = [1, 2, page - 1, page, page + 1, 0, 777, 2049]
    p = Pages(dim + group, lens, [0] * 8, code=code, page=page, heads=heads, dim=dim)
    q = normal(p.g, 8, heads * group, dim, dtype=dtype) * 1.5
    first = check_attention(p, q, lens, [1] * 8)
    again = check_attention(p, q, lens, [1] * 8)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    check_attention(p, q, lens, [1] * 8, window=100)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page, heads, group, dim", SHAPES)
@pytest.mark.parametrize("causal, window", [(True, 0), (True, 70), (False, 0), (False, 33)])
def test_attention_ragged_rows(code, page, heads, group, dim, causal, window):
    lens = [300, 5, 131, 0, 64, 1, 513]
    new = [3, 5, 131, 2, 0, 4, 150]                          # the sequence of one token gets four rows: three see nothing
    p = Pages(dim * 3 + group, lens, [0] * 7, code=code, page=page, heads=heads, dim=dim)
    q = normal(p.g, sum(new), heads * group, dim, dtype=BF16)
    check_attention(p, q, lens, new, causal=causal, window=window)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group, new, lens", [
    (4, [257, 1, 64], [1500, 800, 64]), (1, [300], [300]), (8, [129, 130], [129, 1025]), (3, [500], [4000]),
])
def test_attention_prompts(code, dim, group, new, lens):
    p = Pages(dim + len(new), lens, [0] * len(lens), code=code, page=64, heads=2, dim=dim)
    q = normal(p.g, sum(new), 2 * group, dim, dtype=BF16)
    check_attention(p, q, lens, new)
    check_attention(p, q.to(F16), lens, new, window=200)
    check_attention(p, q, lens, new, causal=False)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0, 1e-4])
def test_attention_scales_and_sizes(rows, scale):
    p = Pages(77, [900], [0], code="int8", page=32, heads=2, dim=128)
    p.cache.v_scale.mul_(torch.logspace(-6, 6, p.cache.v_scale.numel(), device="cuda").view_as(p.cache.v_scale))
    p.cache.v_scale[p.ids[0][3]] = 0.0                       # a block of zero values still counts in the sum
    q = normal(p.g, rows, 8, 128, dtype=BF16)
    check_attention(p, q, [900], [rows], scale=scale)
    q[:, 1] *= 2.0 ** 60                                     # one head's queries far outside float16
    q[:, 2] *= 2.0 ** -60
    p.cache.k_scale.mul_(2.0 ** -20)
    check_attention(p, q[:, 2:4].repeat(1, 2, 1), [900], [rows], scale=scale)
    check_attention(p, q[:, 1:2].repeat(1, 2, 1), [900], [rows], scale=scale * 2.0 ** -50)


@pytest.mark.parametrize("rows", [1, 3, 200])
@pytest.mark.parametrize("dim", [48, 128])
def test_attention_ignores_what_no_row_sees(rows, dim):
    lens = [331, 260]
    p = Pages(55 + rows, lens, [0, 0], code="e4m3", page=32, heads=2, dim=dim)
    q = normal(p.g, 2 * rows, 4, dim, dtype=BF16)
    want = check_attention(p, q, lens, [rows] * 2, window=64)
    # NaN codes behind the sequences' ends, NaN scales of pages that no row sees
    for codes, scale in zip(p.cache[:2], p.cache[2:]):
        for s, n in enumerate(lens):
            codes.view(torch.uint8)[p.ids[s][n // 32], :, n % 32:] = 0x7f
        used = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda")
        for s, n in enumerate(lens):
            for page in range(max(0, n - rows + 1 - 64) // 32, (n - 1) // 32 + 1):
                used[p.ids[s][page]] = True
        scale[~used] = math.nan
    starts = ints([0, rows, 2 * rows])
    got = bfft.cache_attention(q, p.cache, p.table, ints(lens), starts, window=64, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("rows", [1, 150])
def test_attention_nan_reaches_the_rows_that_see_it(rows):
    p = Pages(31, [400, 400], [0, 0], code="int8", page=64, heads=2, dim=64)
    p.cache.k_scale[p.ids[0][2], 1] = math.nan
    p.cache.v_scale[p.ids[1][1], 0] = math.nan
    q = normal(p.g, 2 * rows, 4, 64, dtype=BF16)
    out, lse = bfft.cache_attention(q, p.cache, p.table, ints([400, 400]), ints([0, rows, 2 * rows]), return_lse=True)
    assert out[:rows, 2:].isnan().all() and lse[:rows, 2:].isnan().all() and out[:rows, :2].isfinite().all()
    assert out[rows:, :2].isnan().all() and out[rows:, 2:].isfinite().all()


@pytest.mark.parametrize("rows", [1, 140])
def test_attention_pages_outside_the_cache_are_not_seen(rows):
    p = Pages(21, [256], [0], code="int8", page=64, heads=1, dim=128)
    q = normal(p.g, rows, 4, 128, dtype=BF16)
    table = p.table.clone()
    table[0, 1] = -7
    out, lse = bfft.cache_attention(q, p.cache, table, ints([256]), ints([0, rows]), causal=False, return_lse=True)
    k, v = (p.values(w, 0, 0, 256)[0][:, 0] for w in (0, 1))
    keep = torch.ones(256, dtype=torch.bool, device="cuda")
    keep[64:128] = False
    z = torch.einsum("qhd,kd->qhk", q.double(), k[keep]) * 128 ** -0.5
    assert (lse.double() - torch.logsumexp(z, -1)).abs().max() < 1e-5
    assert (out.double() - torch.softmax(z, -1) @ v[keep]).abs().max() < 2.0 ** -7 * float(v.abs().max())
    # a length beyond the table sees what the table has
    more = bfft.cache_attention(q, p.cache, table, ints([1000]), ints([0, rows]), causal=False)
    assert torch.equal(more, out)


@pytest.mark.parametrize("rows", [1, 70])
def test_attention_strides_streams_and_out(rows):
    p = Pages(41, [500, 90], [0, 0], code="int8", page=16, heads=2, dim=64)
    wide = normal(p.g, 2 * rows, 12, 80, dtype=F16)
    q = wide[:, 2:10, 8:72]
    want, _ = check_attention(p, q, [500, 90], [rows] * 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    buffer = torch.full((8, 2 * rows, 64), 7.0, dtype=F16, device="cuda")
    with torch.cuda.stream(side):
        got = bfft.cache_attention(q, p.cache, p.table, ints([500, 90]), ints([0, rows, 2 * rows]),
                                   out=buffer.transpose(0, 1))
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(buffer.transpose(0, 1), want)
    odd = torch.zeros(2 * rows, 8, 65, dtype=F16, device="cuda")[..., 1:]  # rows on odd elements
    odd.copy_(q)
    assert torch.equal(bfft.cache_attention(odd, p.cache, p.table, ints([500, 90]), ints([0, rows, 2 * rows])), want)


def test_attention_long_cache_offsets():
    """Codes behind 2^31 bytes, split over a long axis, against a cut of it."""
    pages, page, dim = 34000, 128, 256
    cache = bfft.paged_cache(pages, 2, page, dim, code="int8")   # 2.2 GB of codes each
    g = generator(2)
    ids = torch.arange(pages - 1, pages - 1 - 1100, -1, device="cuda")
    for codes, scale in zip(cache[:2], cache[2:]):
        codes[ids] = torch.randint(-127, 128, (1100, 2, page, dim), device="cuda", generator=g, dtype=torch.int8)
        scale[ids] = 0.02
    q = normal(g, 1, 4, dim, dtype=BF16)
    n = 1100 * page - 5
    out, lse = bfft.cache_attention(q, cache, ids.int()[None], ints([n]), ints([0, 1]), return_lse=True)
    for h in range(4):
        k, v = ((codes[ids, h // 2].reshape(-1, dim)[:n].double() * 0.02) for codes in cache[:2])
        z = k @ q[0, h].double() * dim ** -0.5
        assert abs(lse[0, h].double() - torch.logsumexp(z, 0)) < 1e-4
        assert (out[0, h].double() - torch.softmax(z, 0) @ v).abs().max() < 2e-3


# ------------------------------------------------------------------------------- together

@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_prompt_then_tokens_agree_with_full_precision_attention(code):
    """A prompt and single tokens appended and attended to, against attention over the unquantised rows."""
    g = generator(17)
    heads, group, dim, page, total = 2, 4, 64, 16, 90
    table = bfft.rotary_table(256, dim)
    cache = bfft.paged_cache(8, heads, page, dim, code=code)
    pages = ints([[5, 2, 7, 0, 1, 3]])
    q, k, v = (normal(g, total, n, dim, dtype=BF16) for n in (heads * group, heads, heads))
    outs, at = [], 0
    for n in [70] + [1] * 20:
        starts = ints([0, n])
        rq = bfft.append_rotated(cache, k[at:at + n], v[at:at + n], pages, ints([at]), starts, table, q=q[at:at + n])
        outs.append(bfft.cache_attention(rq, cache, pages, ints([at + n]), starts))
        at += n
    where = torch.arange(total, device="cuda")
    rq, rk = (rotate64(x, where, table, "half")[0] for x in (q, k))
    z = torch.einsum("qhd,khd->hqk", rq, rk.repeat_interleave(group, 1)) * dim ** -0.5
    z = z.masked_fill(where > where[:, None], -math.inf)
    want = torch.einsum("hqk,khd->qhd", torch.softmax(z, -1), v.double().repeat_interleave(group, 1))
    err = (torch.cat(outs).double() - want).norm() / want.norm()
    # values off by up to scale / 2 (2^-7.6 of the block's largest, some 3.5 deviations) or 2^-4, in the mean 1 / sqrt 3 of it
    assert err < (0.02 if code == "int8" else 0.05)


def test_calls_can_be_captured():
    p = Pages(61, [100, 33], [4, 4], code="int8", page=32, heads=2, dim=64)
    table = bfft.rotary_table(256, 64)
    q, k, v = (normal(p.g, 2, n, 64, dtype=BF16) for n in (8, 2, 2))
    held, lens, starts = ints([100, 33]), ints([101, 34]), ints([0, 1, 2])

    def step():
        r = bfft.append_rotated(p.cache, k, v, p.table, held, starts, table, q=q)
        return bfft.cache_attention(r, p.cache, p.table, lens, starts)

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------- refusals

def test_refusals_come_before_any_launch():
    p = Pages(1, [20, 3], [4, 4], code="int8", page=16, heads=2, dim=32)
    table, one = bfft.rotary_table(64, 32), ints([0, 1, 2])
    x = normal(p.g, 2, 2, 32, dtype=BF16)
    q = normal(p.g, 2, 4, 32, dtype=BF16)
    held = ints([20, 3])
    count = _lib.launch_counter()

    def refuses(exc, fn, *args, **kw):
        with pytest.raises(exc):
            fn(*args, **kw)

    rot, app, att, read = bfft.rotate_positions, bfft.append_rotated, bfft.cache_attention, bfft.read_cache
    pos = held
    refuses(TypeError, rot, [1.0], pos, table)
    refuses(TypeError, rot, x.double(), pos, table)
    refuses(TypeError, rot, x, pos.float(), table)
    refuses(TypeError, rot, x, pos, table.half())
    refuses(ValueError, rot, x.cpu(), pos, table)
    refuses(ValueError, rot, x[0], pos, table)
    refuses(ValueError, rot, x, pos[:1], table)
    refuses(ValueError, rot, x[..., ::2], pos, table)
    refuses(ValueError, rot, x[..., :30], pos, table)            # table wider than the heads
    refuses(ValueError, rot, x, pos, table, layout="thirds")
    refuses(ValueError, rot, x, pos, table, transform_direction="sideways")
    refuses(ValueError, rot, x, pos, table, out=x[:1])
    refuses(ValueError, rot, x.float().requires_grad_(True), pos, table, out=x.float())
    refuses(ValueError, rot, normal(p.g, 2, 2, 514, dtype=BF16), pos, table)
    refuses(TypeError, app, "cache", x, x, p.table, held, one)
    refuses(TypeError, app, (x, x, x, x), x, x, p.table, held, one)
    refuses(TypeError, app, p.cache, x, x.float(), p.table, held, one)
    refuses(ValueError, app, p.cache, x[:, :1], x[:, :1], p.table, held, one)
    refuses(ValueError, app, p.cache, x[..., :16], x, p.table, held, one)
    refuses(TypeError, app, p.cache, x, x, p.table.long(), held, one)
    refuses(ValueError, app, p.cache, x, x, p.table[0], held, one)
    refuses(ValueError, app, p.cache, x, x, p.table, held[:1], one)
    refuses(ValueError, app, p.cache, x, x, p.table, held, one[:2])
    refuses(ValueError, app, p.cache, x, x, p.table, held, one, table, positions=pos[:1])
    refuses(ValueError, app, p.cache, x, x, p.table, held, one, table, q=q[:1])
    refuses(ValueError, app, p.cache, x, x, p.table, held, one, bfft.rotary_table(8, 34))
    refuses(ValueError, app, (*p.cache[:3], p.cache[3][:1]), x, x, p.table, held, one)
    refuses(ValueError, app, (p.cache[0][:, :, :9], p.cache[1][:, :, :9], *p.cache[2:]), x, x, p.table, held, one)
    refuses(TypeError, read, p.cache, p.table, held, one, 2, dtype=torch.float64)
    refuses(ValueError, read, p.cache, p.table, held, one, -1)
    refuses(TypeError, att, q.float(), p.cache, p.table, held, one)
    refuses(ValueError, att, q[:, :3], p.cache, p.table, held, one)
    refuses(ValueError, att, q, p.cache, p.table, held, one, window=-1)
    refuses(ValueError, att, q, p.cache, p.table, held, one, softmax_scale=math.nan)
    refuses(ValueError, att, q, p.cache, p.table, held, one, out=q[:1])
    refuses(TypeError, att, q, p.cache, p.table, held, one, out=q.half())
    assert _lib.launch_counter() == count
    assert app(p.cache, x[:0], x[:0], p.table, held, ints([0, 0, 0])) is None
    assert att(q[:0], p.cache, p.table, held, ints([0, 0, 0])).shape == (0, 4, 32)


def test_no_bounded_wait_expired_here():
    assert _lib.device_status(0) == 0


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_decode_example(code):
    from bfft import decode_example

    got = decode_example.run(prompt=150, steps=5, code=code)
    # a value is off by up to scale / 2 (2^-7.6 of the block's largest, some 3.5 deviations) or 2^-4 of itself, in the
    # mean 1 / sqrt 3 of it; keys the same, and rounding again as blocks fill
    assert got["value_rel_error"] < (0.02 if code == "int8" else 0.045)
    assert got["attention_rel_error"] < (0.03 if code == "int8" else 0.06)
    assert got["gradient_is_adjoint"]


# ------------------------------------------------------------------------------- many rows, long axes

def long_pages(seed, *, code="int8", page=64, dim=128, lens=(4100, 333), heads=2):
    return Pages(seed, list(lens), [0] * len(lens), code=code, page=page, heads=heads, dim=dim)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page, dim, group", [
    (16, 48, 4), (32, 80, 4), (128, 112, 4), (16, 64, 4), (64, 96, 7), (128, 128, 4), (32, 16, 32),
])
@pytest.mark.parametrize("causal, window", [(True, 0), (True, 517), (False, 0)])
def test_attention_many_rows(code, page, dim, group, causal, window):
    p = long_pages(dim + page, code=code, page=page, dim=dim)
    q = normal(p.g, 333, 2 * group, dim, dtype=BF16) * 1.5
    check_attention(p, q, [4100, 333], [300, 33], causal=causal, window=window)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 64])
def test_attention_many_rows_ignore_what_none_sees(code, page):
    p = long_pages(5, code=code, page=page)
    q = normal(p.g, 400, 8, 128, dtype=F16)
    lens, new = [4100, 333], [300, 100]
    p.cache.v_scale[p.ids[0][40]] = 0.0                      # a block of zero values counts in the sum
    want = check_attention(p, q, lens, new, window=1000)
    for codes, scale in zip(p.cache[:2], p.cache[2:]):
        for s, n in enumerate(lens):
            codes.view(torch.uint8)[p.ids[s][n // page], :, n % page:] = 0x7f
        used = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda")
        for s, n in enumerate(lens):
            for i in range(max(0, n - new[s] + 1 - 1000) // page, (n - 1) // page + 1):
                used[p.ids[s][i]] = True
        scale[~used] = math.nan
    got = bfft.cache_attention(q, p.cache, p.table, ints(lens), ints([0, 300, 400]), window=1000, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    again = bfft.cache_attention(q, p.cache, p.table, ints(lens), ints([0, 300, 400]), window=1000, return_lse=True)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_attention_many_rows_nan_and_missing_pages():
    p = long_pages(6)
    q = normal(p.g, 300, 8, 128, dtype=BF16)
    starts, lens = ints([0, 300, 300]), ints([4100, 333])
    clean = bfft.cache_attention(q, p.cache, p.table, lens, starts, return_lse=True)
    last = 4100 - 20                                          # seen by the last 20 rows only
    p.cache.v_scale[p.ids[0][last // 64], 1] = math.nan
    out, lse = bfft.cache_attention(q, p.cache, p.table, lens, starts, return_lse=True)
    first = 300 - (4100 - last // 64 * 64)                    # the first row that sees the block
    assert out[first:, 4:].isnan().all() and out[:first].isfinite().all() and out[:, :4].isfinite().all()
    assert torch.equal(out[:, :4], clean[0][:, :4]) and lse.isfinite().all()
    p.cache.v_scale[p.ids[0][last // 64], 1] = 0.02
    p.cache.k_scale[p.ids[0][3], 0] = math.nan
    out, lse = bfft.cache_attention(q, p.cache, p.table, lens, starts, return_lse=True)
    assert out[:, :4].isnan().all() and lse[:, :4].isnan().all() and out[:, 4:].isfinite().all()
    table = p.table.clone()
    table[0, 3] = p.cache.k.shape[0]                          # no such page: as if its tokens were not there
    got = bfft.cache_attention(q, p.cache, table, lens, starts, causal=False)
    k, v = (p.values(w, 0, 0, 4100)[0][:, 0] for w in (0, 1))
    keep = torch.ones(4100, dtype=torch.bool, device="cuda")
    keep[192:256] = False
    z = torch.einsum("qhd,kd->qhk", q[:, :4].double(), k[keep]) * 128 ** -0.5
    assert (got[:, :4].double() - torch.softmax(z, -1) @ v[keep]).abs().max() < 2.0 ** -7 * float(v.abs().max())


def test_attention_many_rows_strides_and_sizes():
    p = long_pages(7)
    wide = normal(p.g, 333, 9, 130, dtype=BF16)
    odd = wide[:, 1:, 1:129]                                  # rows on odd elements
    want, _ = check_attention(p, odd, [4100, 333], [300, 33])
    buffer = torch.zeros(8, 333, 136, dtype=BF16, device="cuda")
    out = buffer[:, :, 8:].transpose(0, 1)
    assert bfft.cache_attention(odd.contiguous(), p.cache, p.table, ints([4100, 333]), ints([0, 300, 333]), out=out) is not None
    assert torch.equal(out, want) and (buffer[:, :, :8] == 0).all()
    big = odd * 2.0 ** 50                                     # outside float16
    p.cache.k_scale.mul_(2.0 ** -30)
    check_attention(p, big, [4100, 333], [300, 33], scale=2.0 ** -20)


@pytest.mark.parametrize("dim", [144, 176, 240])
def test_attention_wide_heads(dim):
    lens, new = [700, 33, 0], [1, 20, 2]
    p = Pages(dim, lens, [0] * 3, code="int8", page=32, heads=2, dim=dim)
    q = normal(p.g, 23, 6, dim, dtype=BF16)
    check_attention(p, q, lens, new)
    check_attention(p, q, lens, new, causal=False, window=50)

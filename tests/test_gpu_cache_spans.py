"""Attention over the paged 8-bit cache with first tokens that stay visible and with shared prefixes, against plain
float64 forms.

Tolerances are those of the other tests of the attention: 32-bit sums, float16 weights (2^-11 each, of what a part of
the axis holds: parts are joined in 32 bits), one rounding of the output.  Each test says by the plan's own rule that
it gets to the path it names.
"""
import math

import pytest
import torch

import bfft
from bfft import _lib
from test_gpu_cache import BF16, F16, HALF_UNIT, SHAPES, Pages, cumulative, ints, normal
from test_gpu_cache_edges import lost_under

pytestmark = pytest.mark.gpu


def spans64(p, q, lens, starts, *, scale, causal, window, sinks):
    """out, lse, sum p |v| of each value, and a bound of the scores' rounding, all float64, a sequence at a time."""
    tokens, q_heads, dim = q.shape
    out = torch.zeros(tokens, q_heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((tokens, q_heads), -math.inf, dtype=torch.float64, device="cuda")
    size, slack = torch.zeros_like(out), torch.zeros_like(lse)
    group = q_heads // p.heads
    for s, n in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        if b == a or n <= 0:
            continue
        k, v = (p.values(w, s, 0, n)[0].repeat_interleave(group, 1) for w in (0, 1))
        z = torch.einsum("qhd,khd->hqk", q[a:b].double(), k) * scale
        rough = torch.einsum("qhd,khd->hqk", q[a:b].double().abs(), k.abs()) * abs(scale)
        pos = torch.arange(n - (b - a), n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        seen = (key <= pos) if causal else torch.ones(b - a, n, dtype=torch.bool, device="cuda")
        if window:
            seen = seen & ((key > pos - window) | (key < sinks))
        l = torch.logsumexp(z.masked_fill(~seen, -math.inf), -1)
        w = torch.exp(z - l[..., None]).masked_fill(~seen, 0.0).nan_to_num(0.0)
        out[a:b] = torch.einsum("hqk,khd->qhd", w, v)
        size[a:b] = torch.einsum("hqk,khd->qhd", w, v.abs())
        lse[a:b] = l.T
        slack[a:b] = rough.masked_fill(~seen, 0.0).amax(-1).T
    return out, lse, size, slack


def check_spans(p, q, lens, new, *, scale=None, causal=True, window=0, sinks=0, shared=None, groups=None, table=None, **kw):
    starts = cumulative(new)
    got, lse = bfft.cache_attention(q, p.cache, p.table if table is None else table, ints(lens), ints(starts),
                                    softmax_scale=scale, causal=causal, window=window, sinks=sinks,
                                    shared=None if shared is None else ints(shared),
                                    groups=None if groups is None else ints(groups), return_lse=True, **kw)
    factor = p.dim ** -0.5 if scale is None else scale
    want, want_lse, size, slack = spans64(p, q, lens, starts, scale=factor, causal=causal, window=window, sinks=sinks)
    empty = want_lse == -math.inf
    assert (got[empty] == 0).all() and (lse[empty] == -math.inf).all()
    delta = 2.0 ** -21 * (1 + slack)
    tol = HALF_UNIT[q.dtype] * want.abs() + (2.0 ** -10 + 2 * delta[..., None]) * size + 2.0 ** -24
    assert ((got.double() - want).abs() <= tol).all()
    off = (lse.double() - want_lse).abs()[~empty]
    assert (off <= delta[~empty] + 2.0 ** -20 * (1 + want_lse[~empty].abs())).all()
    return got, lse


def cover(p, table, causal, window, sinks):
    """Tokens that a row sees at most, by what the host knows."""
    width = (p.table if table is None else table).shape[1] * p.page
    return min(width, window + -(-sinks // 16) * 16) if causal and window else width


def takes_tiles(p, q, rows, *, causal=True, window=0, sinks=0, table=None):
    """Row tiles on the tensor cores: from 48 rows of a sequence (of a group) and 3 million pairs of 128 dimensions on."""
    group = q.shape[1] // p.heads
    return (p.dim <= 128 and group <= 128 and rows * group >= 48
            and q.shape[0] * q.shape[1] * cover(p, table, causal, window, sinks) * p.dim >= 3e6 * 128)


def shares(p, q, seqs, groups, *, causal=True, window=0, sinks=0):
    """Groups are told apart from 24 MB of re-read prefix (of the table's width) on, up to 128 rows a kv head."""
    saved = (seqs - groups) * cover(p, None, causal, window, sinks) * p.heads * p.dim * 2
    return q.shape[0] // seqs * (q.shape[1] // p.heads) <= 128 and saved >= 24e6


def widen(p, seqs, groups):
    """Entries behind the sequences' pages, as of tables made for longer ones, so that sharing is worth it."""
    pages = -(-int(24e6) // ((seqs - groups) * p.heads * p.dim * 2 * p.page)) + 1
    if pages > p.table.shape[1]:
        table = torch.full((seqs, pages), -1, dtype=torch.int32, device="cuda")
        table[:, :p.table.shape[1]] = p.table
        p.table = table


def share(p, shared, groups):
    """Makes the sequences of each group name the pages of its first for the whole pages among the shared tokens."""
    for g, n in enumerate(shared):
        k = max(0, n) // p.page
        for s in range(groups[g] + 1, groups[g + 1]):
            p.table[s, :k] = p.table[groups[g], :k]
            p.ids[s][:k] = p.ids[groups[g]][:k]


# ------------------------------------------------------------------------------- visible first tokens

@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("page, heads, group, dim", SHAPES)
@pytest.mark.parametrize("window, sinks", [(1, 1), (33, 4), (100, 16), (100, 17), (700, 200), (64, 5000)])
def test_sinks_single_tokens(code, dtype, page, heads, group, dim, window, sinks):
    lens = [1, 2, page - 1, page, page + 1, 0, 777, 2049]
    p = Pages(dim + group, lens, [0] * 8, code=code, page=page, heads=heads, dim=dim)
    q = normal(p.g, 8, heads * group, dim, dtype=dtype) * 1.5
    first = check_spans(p, q, lens, [1] * 8, window=window, sinks=sinks)
    again = check_spans(p, q, lens, [1] * 8, window=window, sinks=sinks)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page, heads, group, dim", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window, sinks", [(70, 3), (1, 32), (33, 48), (200, 129)])
def test_sinks_ragged_rows(code, page, heads, group, dim, causal, window, sinks):
    lens = [300, 5, 131, 0, 64, 1, 513]
    new = [3, 5, 131, 2, 0, 4, 150]                          # the sequence of one token gets four rows: three see nothing
    p = Pages(dim * 3 + group, lens, [0] * 7, code=code, page=page, heads=heads, dim=dim)
    q = normal(p.g, sum(new), heads * group, dim, dtype=BF16)
    check_spans(p, q, lens, new, causal=causal, window=window, sinks=sinks)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype, page, dim, group, window, sinks", [
    (BF16, 16, 64, 8, 129, 1), (F16, 64, 128, 4, 517, 4), (BF16, 128, 96, 4, 1000, 100), (BF16, 32, 48, 16, 200, 16),
    (F16, 16, 128, 8, 64, 333), (BF16, 64, 80, 5, 2999, 7), (BF16, 128, 128, 1, 400, 129),
])
@pytest.mark.parametrize("causal", [True, False])
def test_sinks_many_rows(code, dtype, page, dim, group, window, sinks, causal):
    lens, new = [4100, 0, 1333, 77], [2000, 60, 1000, 77]
    p = Pages(dim + page, lens, [0] * 4, code=code, page=page, heads=2, dim=dim)
    q = normal(p.g, sum(new), 2 * group, dim, dtype=dtype) * 1.5
    assert takes_tiles(p, q, sum(new) // 4, causal=causal, window=window, sinks=sinks)
    check_spans(p, q, lens, new, causal=causal, window=window, sinks=sinks)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("new, lens, window, sinks", [
    ([30], [9000], 5000, 20), ([64, 70], [20000, 100], 12000, 4), ([1], [40000], 30000, 1000),
])
def test_sinks_whose_axis_is_cut(code, new, lens, window, sinks):
    """Few rows over a long window: parts of the axis, the first tokens in one with the window's, are joined."""
    p = Pages(4, lens, [0] * len(lens), code=code, page=32, heads=2, dim=128)
    q = normal(p.g, sum(new), 8, 128, dtype=BF16)
    check_spans(p, q, lens, new, window=window, sinks=sinks)


@pytest.mark.parametrize("rows, window, lens, tiles", [
    (1, 64, [971, 260], False), (3, 64, [971, 260], False), (200, 64, [971, 260], False), (1000, 700, [2971, 1760], True),
])
@pytest.mark.parametrize("dim", [48, 128])
def test_sinks_ignore_what_no_row_sees(rows, window, lens, tiles, dim):
    sinks = 5
    p = Pages(55 + rows, lens, [0, 0], code="e4m3", page=16, heads=2, dim=dim)
    q = normal(p.g, 2 * rows, 8, dim, dtype=BF16)
    assert takes_tiles(p, q, rows, window=window, sinks=sinks) == tiles
    want = check_spans(p, q, lens, [rows] * 2, window=window, sinks=sinks)
    # NaN codes behind the first tokens, before the windows and behind the ends; NaN scales and no pages between
    table = p.table.clone()
    for s, n in enumerate(lens):
        low = max(0, n - rows + 1 - window)
        for w in (0, 1):
            codes = p.cache[w].view(torch.uint8)
            hidden = torch.tensor([*range(sinks, low), *range(n, -(-n // 16) * 16)], dtype=torch.long)
            codes[torch.tensor(p.ids[s])[hidden // 16].cuda(), :, (hidden % 16).cuda()] = 0x7f
            for page in range(1, low // 16):
                p.cache[2 + w][p.ids[s][page]] = math.nan
        table[s, 1:max(1, low // 16 - 1)] = 10 ** 8
    got = bfft.cache_attention(q, p.cache, table, ints(lens), ints([0, rows, 2 * rows]), window=window, sinks=sinks,
                               return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("rows", [1, 150])
def test_nan_in_the_first_tokens(rows):
    p = Pages(31, [900, 900], [0, 0], code="int8", page=64, heads=2, dim=64)
    p.cache.k_scale[p.ids[0][0], 1] = math.nan
    p.cache.v_scale[p.ids[1][0], 0] = math.nan
    q = normal(p.g, 2 * rows, 4, 64, dtype=BF16)

    def call(sinks):
        return bfft.cache_attention(q, p.cache, p.table, ints([900, 900]), ints([0, rows, 2 * rows]), window=100, sinks=sinks)

    assert call(0).isfinite().all()
    out = call(2)
    assert out[:rows, 2:].isnan().all() and out[:rows, :2].isfinite().all()
    assert out[rows:, :2].isnan().all() and out[rows:, 2:].isfinite().all()


@pytest.mark.parametrize("rows", [2, 300])
def test_sinks_without_a_window_change_nothing(rows):
    p = Pages(3, [2500, 1111], [0, 0], code="int8", page=64, heads=2, dim=128)
    q = normal(p.g, 2 * rows, 8, 128, dtype=BF16)
    args = (q, p.cache, p.table, ints([2500, 1111]), ints([0, rows, 2 * rows]))
    assert torch.equal(bfft.cache_attention(*args, sinks=7), bfft.cache_attention(*args))
    check_spans(p, q, [2500, 1111], [rows] * 2, window=1000, sinks=3000)  # everything is seen


@pytest.mark.parametrize("where", [{0}, {3}, {4}])
@pytest.mark.parametrize("new", [[1, 1], [300, 33]])
def test_sinks_over_a_tiny_page_among_ordinary_ones(where, new):
    lens = [4100, 133]
    p = Pages(130, lens, [0, 0], code="int8", page=32, heads=2, dim=128)
    for ids in p.ids:
        p.cache.v_scale[[i for j, i in enumerate(x for x in ids if x >= 0) if j in where]] = 1e-36
    q = normal(p.g, sum(new), 8, 128, dtype=BF16)
    check_spans(p, q, lens, new, window=90, sinks=60)


def test_sinks_of_a_long_cache():
    """Codes behind 2^31 bytes: the first tokens at the cache's end, the window at its start, and the other way round."""
    pages, page, dim = 34000, 128, 256
    cache = bfft.paged_cache(pages, 2, page, dim, code="int8")   # 2.2 GB of codes each
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    for ids in (torch.arange(1100, device="cuda"), torch.arange(pages - 1100, pages, device="cuda")):
        for codes, scale in zip(cache[:2], cache[2:]):
            codes[ids] = torch.randint(-127, 128, (1100, 2, page, dim), device="cuda", generator=g, dtype=torch.int8)
            scale[ids] = 0.02
    q = normal(g, 2, 4, dim, dtype=BF16)
    low, high = torch.arange(1100, device="cuda"), torch.arange(pages - 1100, pages, device="cuda")
    table = torch.stack((torch.cat((low, high)), torch.cat((high, low))))
    n, window, sinks = 2200 * page - 5, 9000, 300
    out = bfft.cache_attention(q, cache, table.int(), ints([n, n]), ints([0, 1, 2]), window=window, sinks=sinks)
    at = torch.cat((torch.arange(sinks), torch.arange(n - window, n))).cuda()
    for s in range(2):
        for h in range(4):
            k, v = (codes[table[s][at // page], h // 2, at % page].double() * 0.02 for codes in cache[:2])
            z = k @ q[s, h].double() * dim ** -0.5
            assert (out[s, h].double() - torch.softmax(z, 0) @ v).abs().max() < 2e-3


# ------------------------------------------------------------------------------- shared prefixes

def grouped(seed, *, code, page, heads, dim, group, dtype=BF16, new=None):
    """Ten sequences: one in no group, a group of five that share some 600 tokens (one without tokens, one whose tokens
    end within the prefix), a group that shares nothing, a group of one, and one in no group."""
    shared, groups = [600 + page // 2, 0, 333], [1, 6, 8, 9]
    lens = [55, 640, 601 + page, 0, 300, 1100, 17, 900, 700, 1]
    new = new or [1] * 10
    p = Pages(seed, lens, [max(0, 620 + page - n) for n in lens], code=code, page=page, heads=heads, dim=dim)
    share(p, shared, groups)
    widen(p, 10, 3)
    q = normal(p.g, sum(new), heads * group, dim, dtype=dtype) * 1.5
    assert shares(p, q, 10, 3)
    return p, q, lens, new, shared, groups


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("page, heads, group, dim", SHAPES)
def test_shared_single_tokens(code, dtype, page, heads, group, dim):
    p, q, lens, new, shared, groups = grouped(dim + group, code=code, page=page, heads=heads, dim=dim, group=group,
                                              dtype=dtype)
    first = check_spans(p, q, lens, new, shared=shared, groups=groups)
    again = check_spans(p, q, lens, new, shared=shared, groups=groups)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page, heads, group, dim", SHAPES)
@pytest.mark.parametrize("causal, window, sinks", [(True, 0, 0), (False, 0, 0), (False, 433, 17)])
def test_shared_ragged_rows(code, page, heads, group, dim, causal, window, sinks):
    new = [3, 5, 1, 2, 7, 0, 4, 9, 2, 4]
    p, q, lens, new, shared, groups = grouped(dim * 3 + group, code=code, page=page, heads=heads, dim=dim, group=group,
                                              new=new)
    check_spans(p, q, lens, new, causal=causal, window=window, sinks=sinks, shared=shared, groups=groups)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page, heads, group, dim", [(64, 2, 4, 128), (16, 4, 1, 80), (32, 2, 12, 256), (128, 3, 2, 64)])
@pytest.mark.parametrize("window, sinks", [(250, 0), (40, 620), (333, 5), (70, 100)])
@pytest.mark.parametrize("new", [[1], [1, 3, 1, 2, 4, 0, 2]])
def test_shared_windows(code, page, heads, group, dim, window, sinks, new):
    """Windows that end within the prefix, reach into it or leave only its first tokens: 450 sequences in 75 groups, by
    the kernel of few rows."""
    seqs, groups = 450, list(range(0, 451, 6))
    shared = [620 if g % 3 else 160 for g in range(75)]
    lens = [max(0, shared[s // 6] + (37 * s % 400 if s % 5 else -40)) + 4 for s in range(seqs)]
    new = (new * seqs)[:seqs]
    p = Pages(dim, lens, [max(0, 640 - n) for n in lens], code=code, page=page, heads=heads, dim=dim)
    share(p, shared, groups)
    q = normal(p.g, sum(new), heads * group, dim, dtype=BF16) * 1.5
    how = {"window": window, "sinks": sinks}
    assert shares(p, q, seqs, 75, **how) == (375 * (window + -(-sinks // 16) * 16) * heads * dim * 2 >= 24e6)
    assert not takes_tiles(p, q, sum(new) // 75, **how)
    check_spans(p, q, lens, new, shared=shared, groups=groups, **how)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype, page, heads, group, dim, each", [
    (BF16, 64, 2, 4, 128, 1), (F16, 16, 1, 8, 64, 3), (BF16, 128, 2, 1, 96, 10), (BF16, 32, 3, 5, 80, 4),
    (F16, 64, 1, 33, 48, 1), (BF16, 16, 2, 16, 112, 4),
])
@pytest.mark.parametrize("causal, window, sinks", [(True, 0, 0), (True, 1900, 5), (False, 700, 0)])
def test_shared_many_rows(code, dtype, page, heads, group, dim, each, causal, window, sinks):
    """Prefixes on the tensor-core tiles, the sequences' own tokens by the kernel of few rows."""
    seqs, prefix = 210, [2011, 777]
    groups = [0, 90, 209]                                    # the last sequence is in none
    of = [0] * 90 + [1] * 119
    lens = [prefix[g] + 1 + 37 * i % 260 for i, g in enumerate(of)] + [400]
    lens[5] = lens[100] = 0
    lens[7] = 1000                                           # within the prefix
    new = [1 + i % each for i in range(seqs)]
    p = Pages(dim + each, lens, [max(0, 2100 - n) for n in lens], code=code, page=page, heads=heads, dim=dim)
    share(p, prefix, groups)
    q = normal(p.g, sum(new), heads * group, dim, dtype=dtype) * 1.5
    rows = sum(new) // 2
    assert shares(p, q, seqs, 2, causal=causal, window=window, sinks=sinks)
    assert takes_tiles(p, q, rows, causal=causal, window=window, sinks=sinks)
    assert not takes_tiles(p, q, sum(new) // seqs, causal=causal, window=window, sinks=sinks)
    first = check_spans(p, q, lens, new, causal=causal, window=window, sinks=sinks, shared=prefix, groups=groups)
    again = check_spans(p, q, lens, new, causal=causal, window=window, sinks=sinks, shared=prefix, groups=groups)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page, dim", [(64, 128), (16, 64), (128, 80)])
@pytest.mark.parametrize("causal, window, sinks", [(True, 0, 0), (True, 3100, 9), (False, 0, 0)])
@pytest.mark.parametrize("groups", [None, [1, 7]])
def test_shared_prompts(code, page, dim, causal, window, sinks, groups):
    """Questions of some tens of rows behind one text: prefixes and own tokens both on the tensor-core tiles."""
    prefix, seqs = [3500], 24
    groups = groups and [1, seqs - 1]
    new = [31, 40, 17, 28, 50, 21, 24, 33] * 3
    lens = [3500 + n + 150 * (i % 3) for i, n in enumerate(new)]
    lens[2] = 11                                             # six of whose rows see nothing
    p = Pages(dim + page, lens, [max(0, 3520 - n) for n in lens], code=code, page=page, heads=4, dim=dim)
    share(p, prefix, [0, seqs])
    q = normal(p.g, sum(new), 16, dim, dtype=BF16) * 1.5
    assert shares(p, q, seqs, 1, causal=causal, window=window, sinks=sinks)
    assert takes_tiles(p, q, sum(new) // seqs, causal=causal, window=window, sinks=sinks)
    check_spans(p, q, lens, new, causal=causal, window=window, sinks=sinks, shared=prefix, groups=groups)


@pytest.mark.parametrize("form", ["plain", "sinks", "shared"])
@pytest.mark.parametrize("dim", [64, 112])
def test_row_tiles_of_odd_queries(form, dim):
    """Queries that the copy engine cannot take: rows on odd elements, and one row that stands for many."""
    seqs, each = 210, 2
    kw = {"plain": {}, "sinks": {"window": 1900, "sinks": 3}, "shared": {"shared": [1984]}}[form]
    lens = [2000 + i % 50 for i in range(seqs)] if form == "shared" else [4100, 3000]
    new = [each] * seqs if form == "shared" else [200, 220]
    p = Pages(dim, lens, [0] * len(lens), code="int8", page=64, heads=2, dim=dim)
    if form == "shared":
        share(p, [1984], [0, seqs])
        assert shares(p, torch.empty(420, 8, dim), seqs, 1)
    q = normal(p.g, 420, 8, dim + 1, dtype=BF16)[..., 1:]
    assert takes_tiles(p, q, 420 if form == "shared" else 210, **({} if form == "shared" else kw))
    check_spans(p, q, lens, new, **kw)
    same = normal(p.g, 1, 8, dim, dtype=BF16)
    want = check_spans(p, same.expand(420, 8, dim).contiguous(), lens, new, **kw)
    got = check_spans(p, same.expand(420, 8, dim), lens, new, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    head = normal(p.g, 420, 1, dim, dtype=F16)
    assert torch.equal(check_spans(p, head.expand(420, 8, dim), lens, new, **kw)[0],
                       check_spans(p, head.expand(420, 8, dim).contiguous(), lens, new, **kw)[0])


@pytest.mark.parametrize("new, lens, window", [
    ([1], [30000], 9000), ([1, 1], [700, 90], 500), ([40], [9000], 5000), ([600, 70], [4100, 800], 2000),
])
def test_rows_behind_the_last_sequence_stay(new, lens, window):
    """Direct, by a cluster, by chunks that a second kernel joins, and by row tiles."""
    p = Pages(9, lens, [0] * len(lens), code="int8", page=64, heads=2, dim=128)
    q = normal(p.g, sum(new) + 3, 8, 128, dtype=BF16)
    for kw in ({"window": window, "sinks": 4}, {"window": window}, {}):
        left = torch.full_like(q, 7.0)
        bfft.cache_attention(q, p.cache, p.table, ints(lens), ints(cumulative(new)), out=left, **kw)
        assert (left[sum(new):] == 7.0).all() and left[:sum(new)].isfinite().all()


def test_sharing_is_left_out_where_sequences_have_many_rows():
    lens, new = [2000, 1500], [300, 200]
    p = Pages(5, lens, [0, 0], code="int8", page=64, heads=2, dim=128)
    share(p, [1024], [0, 2])
    q = normal(p.g, 500, 8, 128, dtype=BF16)
    got = check_spans(p, q, lens, new, shared=[1024])
    plain = bfft.cache_attention(q, p.cache, p.table, ints(lens), ints([0, 300, 500]))
    assert torch.equal(got[0], plain) and not shares(p, q, 2, 1)
    few = check_spans(p, q[:2], lens, [1, 1], shared=[1024])              # and where it saves a few bytes only
    assert torch.equal(few[0], bfft.cache_attention(q[:2], p.cache, p.table, ints(lens), ints([0, 1, 2])))


@pytest.mark.parametrize("dim, heads", [(16, 64), (32, 64)])
def test_pieces_longer_than_the_table_of_pages(dim, heads):
    """Items of over 380 pages of 16: the kernel of few rows takes them in segments."""
    lens = [14000 + 500 * i for i in range(9)]
    p = Pages(dim, lens, [0] * 9, code="e4m3", page=16, heads=heads, dim=dim)
    q = normal(p.g, 9, heads, dim, dtype=BF16)
    shared = [0, 8000]
    groups = [0, 3, 9]
    share(p, shared, groups)
    assert shares(p, q, 9, 2) and shares(p, q, 9, 2, window=8500, sinks=100)
    total = sum(lens[:3]) + sum(n - 8000 for n in lens[3:]) + 8000
    assert total / (2 * 3 * 148 // heads) > 380 * 16
    check_spans(p, q, lens, [1] * 9, shared=shared, groups=groups)
    check_spans(p, q, lens, [1] * 9, shared=shared, groups=groups, window=8500, sinks=100)
    for ids in p.ids[:3]:                                    # a small value scale in one segment only
        p.cache.v_scale[ids[450]] = 1e-36
    check_spans(p, q, lens, [1] * 9, shared=shared, groups=groups)
    for s in (1, 2):
        p.cache.v_scale[p.ids[s][3]] = 1e-36
    check_spans(p, q, lens, [1] * 9, shared=shared, groups=groups)


def check_relative(p, q, lens, new, shared):
    """Every row against its own size: nothing absolute but the last bit of bfloat16's smallest values.  What weights
    lose in float16 is that of a row's largest, and a part of the axis has a largest of its own, no greater."""
    starts, scale = cumulative(new), p.dim ** -0.5
    got, lse = bfft.cache_attention(q, p.cache, p.table, ints(lens), ints(starts), shared=ints(shared), return_lse=True)
    want, want_lse, size, slack = spans64(p, q, lens, starts, scale=scale, causal=True, window=0, sinks=0)
    delta = 2.0 ** -21 * (1 + slack)
    tol = HALF_UNIT[q.dtype] * want.abs() + (2.0 ** -10 + 2 * delta[..., None]) * size + 2.0 ** -133
    tol = tol + lost_under(p, q, lens, starts, 10, scale=scale, causal=True, window=0)
    assert ((got.double() - want).abs() <= tol).all()
    assert ((lse.double() - want_lse).abs() <= delta + 2.0 ** -20 * (1 + want_lse.abs())).all()
    return got, lse


@pytest.mark.parametrize("each, tiles", [(1, False), (1, True), (3, True)])
def test_shared_over_tiny_values(each, tiles):
    seqs = 200 if tiles else 4
    lens = [2000 + each + i % 90 for i in range(seqs)]
    p = Pages(each, lens, [0] * seqs, code="int8", page=32, heads=2, dim=128)
    share(p, [2000], [0, seqs])
    widen(p, seqs, 1)
    q = normal(p.g, seqs * each, 8, 128, dtype=BF16)
    assert shares(p, q, seqs, 1) and takes_tiles(p, q, seqs * each) == tiles
    for where in ([3], range(62)):                           # one page of the prefix, then all of it
        p.cache.v_scale[[p.ids[0][i] for i in where]] = 1e-36
        check_relative(p, q, lens, [each] * seqs, [2000])
    for s in range(seqs):                                    # and the sequences' own
        p.cache.v_scale[[i for i in p.ids[s] if i >= 0]] = 1e-36
    out, lse = check_relative(p, q, lens, [each] * seqs, [2000])
    assert lse.isfinite().all() and out.isfinite().all() and out.abs().amax() > 1e-37


@pytest.mark.parametrize("each", [1, 30])
def test_shared_ignores_what_no_row_sees(each):
    seqs = 60
    lens = [1024 + each + i % 50 for i in range(seqs)]
    p = Pages(17, lens, [0] * seqs, code="e4m3", page=64, heads=8, dim=64)
    share(p, [1024], [0, seqs])
    q = normal(p.g, seqs * each, 16, 64, dtype=F16)
    assert shares(p, q, seqs, 1, window=500, sinks=3)
    assert takes_tiles(p, q, seqs * each, window=500, sinks=3) == (each > 1)
    want = check_spans(p, q, lens, [each] * seqs, shared=[1030], window=500, sinks=3)
    low = 1024 + 1 + min(i % 50 for i in range(seqs)) - 500
    for w in (0, 1):
        codes = p.cache[w].view(torch.uint8)
        hidden = torch.arange(3, low)
        codes[torch.tensor(p.ids[0])[hidden // 64].cuda(), :, (hidden % 64).cuda()] = 0x7f
        for page in range(1, low // 64):
            p.cache[2 + w][p.ids[0][page]] = math.nan
        for s, n in enumerate(lens):
            if n % 64:
                codes[p.ids[s][n // 64], :, n % 64:] = 0x7f
    got = bfft.cache_attention(q, p.cache, p.table, ints(lens), ints(cumulative([each] * seqs)), shared=ints([1030]),
                               window=500, sinks=3, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("each", [1, 20])
def test_nan_and_missing_pages_of_a_prefix(each):
    seqs = 50
    lens = [1200 + each] * 25 + [640] + [1200 + each] * 24
    p = Pages(23, lens, [600] * seqs, code="int8", page=64, heads=2, dim=64)
    share(p, [1152], [0, seqs])
    widen(p, seqs, 1)
    q = normal(p.g, seqs * each, 4, 64, dtype=BF16)
    assert shares(p, q, seqs, 1)
    args = (ints(lens), ints(cumulative([each] * seqs)))
    p.cache.v_scale[p.ids[0][12], 0] = math.nan              # tokens 768..: the sequence of 640 does not see them
    out = bfft.cache_attention(q, p.cache, p.table, *args, shared=ints([1152]))
    short = torch.zeros(seqs, dtype=torch.bool, device="cuda")
    short[25] = True
    short = short.repeat_interleave(each)
    assert out[~short][:, :2].isnan().all() and out[~short][:, 2:].isfinite().all() and out[short].isfinite().all()
    # a prefix's page that is not in the cache is not seen
    table = p.table.clone()
    table[:, 12] = -1
    got, lse = bfft.cache_attention(q, p.cache, table, *args, shared=ints([1152]), return_lse=True)
    want, plain = bfft.cache_attention(q, p.cache, table, *args, return_lse=True)
    assert got.isfinite().all() and (lse - plain).abs().max() < 1e-5
    assert (got.float() - want.float()).abs().max() <= 2.0 ** -6 * want.float().abs().max()


@pytest.mark.parametrize("each, seqs", [(1, 6), (1, 200), (24, 12)])
def test_shared_strides_streams_graphs_and_out(each, seqs):
    """Odd strides, another stream, q as its own output, rows behind the last sequence, and a captured call whose
    tables change between replays."""
    lens = [900 + each + i % 70 for i in range(seqs)]
    p = Pages(41, lens, [100] * seqs, code="int8", page=16, heads=2, dim=64)
    share(p, [896], [0, seqs])
    widen(p, seqs, 1)
    wide = normal(p.g, seqs * each, 12, 80, dtype=F16)
    q = wide[:, 2:10, 8:72]
    assert shares(p, q, seqs, 1)
    new, starts = [each] * seqs, ints(cumulative([each] * seqs))
    want, want_lse = check_spans(p, q, lens, new, shared=[896])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    buffer = torch.full((8, seqs * each, 64), 7.0, dtype=F16, device="cuda")
    shared = ints([896])
    with torch.cuda.stream(side):
        bfft.cache_attention(q, p.cache, p.table, ints(lens), starts, shared=shared, out=buffer.transpose(0, 1))
    side.synchronize()
    assert torch.equal(buffer.transpose(0, 1), want)
    odd = torch.zeros(seqs * each, 8, 65, dtype=F16, device="cuda")[..., 1:]  # rows on odd elements
    odd.copy_(q)
    assert torch.equal(bfft.cache_attention(odd, p.cache, p.table, ints(lens), starts, shared=shared), want)
    # rows behind the last sequence stay as they are
    more = torch.cat((q, q[:3]))
    left = torch.full_like(more, 5.0)
    bfft.cache_attention(more, p.cache, p.table, ints(lens), starts, shared=shared, out=left)
    assert (left[seqs * each:] == 5.0).all()
    x = q.clone()
    assert bfft.cache_attention(x, p.cache, p.table, ints(lens), starts, shared=shared, out=x) is x
    assert torch.equal(x, want)
    # a captured call reads its tables anew at each replay
    held, groups = ints(lens), ints([0, seqs])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, lse = bfft.cache_attention(q, p.cache, p.table, held, starts, shared=shared, groups=groups, return_lse=True)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    for tokens, longer, last in ((512, 50, seqs), (0, 3, seqs), (896, 60, seqs // 2)):
        shared.fill_(tokens)
        held.copy_(ints([n + longer for n in lens]))
        groups.copy_(ints([0, last]))
        graph.replay()
        torch.cuda.synchronize()
        again = check_spans(p, q, [n + longer for n in lens], new, shared=[tokens], groups=[0, last])
        assert torch.equal(got, again[0]) and torch.equal(lse, again[1])


def test_two_graphs_and_two_streams_at_once():
    """Two captured calls, replayed side by side, each with a workspace of its own."""
    seqs, calls = 250, []
    for seed in (1, 2):
        lens = [1500 + i % 200 for i in range(seqs)]
        p = Pages(seed, lens, [0] * seqs, code="int8", page=64, heads=2, dim=128)
        share(p, [1472], [0, seqs])
        q = normal(p.g, seqs, 8, 128, dtype=BF16)
        assert takes_tiles(p, q, seqs) and shares(p, q, seqs, 1)
        args = (q, p.cache, p.table, ints(lens), ints(list(range(seqs + 1))))
        want = bfft.cache_attention(*args, shared=ints([1472]))
        shared = ints([1472])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = bfft.cache_attention(*args, shared=shared)
        calls.append((graph, got, want, torch.cuda.Stream(), args, shared))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, got, _, stream, _, _ in calls:
            with torch.cuda.stream(stream):
                got.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for _, got, want, _, _, _ in calls:
        assert torch.equal(got, want)


def test_many_sequences_and_groups():
    """More sequences and groups than a block has threads: the items are found in rounds."""
    seqs = 1500
    groups = list(range(0, 1501, 3))
    shared = [16 * (g % 9) for g in range(500)]
    lens = [shared[s // 3] + 1 + s % 40 for s in range(seqs)]
    p = Pages(8, lens, [0] * seqs, code="int8", page=16, heads=1, dim=64)
    share(p, shared, groups)
    widen(p, seqs, 500)
    q = normal(p.g, seqs, 4, 64, dtype=BF16)
    assert shares(p, q, seqs, 500)
    check_spans(p, q, lens, [1] * seqs, shared=shared, groups=groups)
    check_spans(p, q, lens, [1] * seqs, shared=[shared[0]] + [0] * 4, groups=[0, 3, 3, 9, 1500, 1500])


@pytest.mark.parametrize("tokens", [-5, 0, 15, 10 ** 9])
def test_counts_of_shared_tokens_out_of_range(tokens):
    """Less than a page shares nothing; more than the table has shares the table."""
    lens = [200, 208, 150]
    p = Pages(6, lens, [8, 0, 58], code="int8", page=16, heads=2, dim=64)
    if tokens > 0:
        share(p, [min(tokens, 208)], [0, 3])
    widen(p, 3, 1)
    q = normal(p.g, 3, 8, 64, dtype=BF16)
    assert shares(p, q, 3, 1)
    check_spans(p, q, lens, [1] * 3, shared=[tokens])


# ------------------------------------------------------------------------------- refusals

def test_refusals_of_spans_come_before_any_launch():
    p = Pages(1, [20, 3], [4, 4], code="int8", page=16, heads=2, dim=32)
    q, held, one = normal(p.g, 2, 4, 32, dtype=BF16), ints([20, 3]), ints([0, 1, 2])
    count = _lib.launch_counter()

    def refuses(exc, **kw):
        with pytest.raises(exc):
            bfft.cache_attention(q, p.cache, p.table, held, one, **kw)

    refuses(ValueError, window=4, sinks=-1)
    refuses(ValueError, window=4, sinks=1.5)
    refuses(ValueError, window=4, sinks=1 << 31)
    refuses(ValueError, groups=ints([0, 2]))                                  # nothing is shared
    refuses(TypeError, shared=16)
    refuses(TypeError, shared=ints([16]).long())
    refuses(TypeError, shared=ints([16]), groups=ints([0, 2]).float())
    refuses(ValueError, shared=ints([16]).cpu())
    refuses(ValueError, shared=ints([16]), groups=ints([0, 2]).cpu())
    refuses(ValueError, shared=ints([16, 16]))                                # two groups, and nothing says which
    refuses(ValueError, shared=ints([16, 16]), groups=ints([0, 2]))
    refuses(ValueError, shared=ints([[16]]))
    refuses(ValueError, shared=ints([16, 0, 16])[::2], groups=ints([0, 1, 2]))
    refuses(ValueError, shared=ints([16]), groups=ints([0, 9, 2])[::2])
    assert _lib.launch_counter() == count
    none = ints([])
    assert torch.equal(bfft.cache_attention(q, p.cache, p.table, held, one, shared=none, groups=ints([0])),
                       bfft.cache_attention(q, p.cache, p.table, held, one))
    empty = bfft.cache_attention(q[:0], p.cache, p.table, held, ints([0, 0, 0]), shared=ints([16]), window=3, sinks=1)
    assert empty.shape == (0, 4, 32)


def test_no_bounded_wait_expired_here():
    assert _lib.device_status(0) == 0

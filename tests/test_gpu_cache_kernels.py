"""Which kernels a call of the attention launches, read from a captured graph of it: the forms with first tokens and
with groups are there where they should be, and their results are those of the plain float64 form."""
import os
import re
import tempfile
import warnings

import pytest
import torch

import bfft
from bfft import _lib, decode_example
from test_gpu_cache import BF16, F16, Pages, cumulative, ints, normal
from test_gpu_cache_spans import check_spans, grouped, share, widen

pytestmark = pytest.mark.gpu

FORMS = {"0": "", "1": " sinks", "2": " groups"}  # the kernels' last template argument


def kernels(call):
    """The attention kernels that a call launches, in their order."""
    call()                                                    # the first one sets kernel attributes
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    graph.enable_debug_mode()
    with torch.cuda.graph(graph):
        call()
    with tempfile.TemporaryDirectory() as where:
        path = os.path.join(where, "graph.dot")
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")                   # torch says that it writes a file
            graph.debug_dump(path)
        text = open(path).read()
    found = []
    for at, name, rest in re.findall(r"ID \| (\d+) \(topoId: \d+\) \| \w*?k_attention_(join_items|items|join|split|tiles)(\w*)", text):
        form = FORMS[re.findall(r"Li(\d+)E", rest)[-1]] if name in ("split", "tiles") else ""
        found.append((int(at), name + form))
    return [name for _, name in sorted(found)]


def attention(p, q, lens, new, **kw):
    kw = {k: ints(v) if k in ("shared", "groups") else v for k, v in kw.items()}
    args = (q, p.cache, p.table, ints(lens), ints(cumulative(new)))
    return lambda: bfft.cache_attention(*args, **kw)


def check(p, q, lens, new, want, **kw):
    count = _lib.launch_counter()
    check_spans(p, q, lens, new, **kw)
    assert _lib.launch_counter() == count + len(want)
    assert kernels(attention(p, q, lens, new, **kw)) == want


@pytest.mark.parametrize("how, form", [({}, ""), ({"window": 500}, ""), ({"window": 500, "sinks": 5}, " sinks"), ({"sinks": 5}, "")])
@pytest.mark.parametrize("dim", [64, 128])
def test_without_groups(how, form, dim):
    p = Pages(dim, [9000, 8000], [0, 0], code="int8", page=64, heads=2, dim=dim)
    for rows in (1, 3):                                       # a short axis is one cluster's, a long one is joined
        q = normal(p.g, 2 * rows, 8, dim, dtype=BF16)
        check(p, q, [9000, 8000], [rows] * 2, ["split" + form] + ["join"] * ("window" not in how), **how)
    q = normal(p.g, 4000, 8, dim, dtype=BF16)
    check(p, q, [9000, 8000], [2000] * 2, ["tiles" + form], **how)


@pytest.mark.parametrize("page, heads, group, dim", [(64, 2, 4, 128), (16, 4, 1, 80), (32, 2, 12, 256)])
def test_groups_of_few_rows(page, heads, group, dim):
    """One launch of the kernel of few rows for prefixes and own tokens, the items found in it."""
    p, q, lens, new, shared, groups = grouped(dim, code="int8", page=page, heads=heads, dim=dim, group=group)
    check(p, q, lens, new, ["split groups", "join_items"], shared=shared, groups=groups)


@pytest.mark.parametrize("how", [{}, {"window": 250, "sinks": 7}])
def test_many_groups_of_few_rows(how):
    """The items of more than 128 groups and sequences are listed first."""
    seqs, groups = 450, list(range(0, 451, 6))
    shared = [620 if g % 3 else 160 for g in range(75)]
    lens = [shared[s // 6] + 37 * s % 400 + 4 for s in range(seqs)]
    p = Pages(3, lens, [max(0, 640 - n) for n in lens], code="e4m3", page=64, heads=2, dim=128)
    share(p, shared, groups)
    q = normal(p.g, seqs, 8, 128, dtype=BF16)
    check(p, q, lens, [1] * seqs, ["items", "split groups", "join_items"], shared=shared, groups=groups, **how)


@pytest.mark.parametrize("seqs, dtype", [(24, BF16), (200, F16)])
@pytest.mark.parametrize("how", [{}, {"window": 3900, "sinks": 5}])
def test_prefixes_on_row_tiles(seqs, dtype, how):
    """Prefixes on the row tiles, own tokens by the kernel of few rows (its items by a block of the row tiles, where
    there are many)."""
    lens = [4100 + 1 + 37 * i % 260 for i in range(seqs)]
    p = Pages(seqs, lens, [0] * seqs, code="int8", page=64, heads=4, dim=128)
    share(p, [4100], [0, seqs])
    q = normal(p.g, seqs, 32, 128, dtype=dtype)
    check(p, q, lens, [1] * seqs, ["tiles groups", "split groups", "join_items"], shared=[4100], groups=[0, seqs], **how)


def test_prefixes_and_own_tokens_on_row_tiles():
    new = [31, 40, 17, 28, 50, 21, 24, 33] * 3
    lens = [3500 + n + 150 * (i % 3) for i, n in enumerate(new)]
    p = Pages(64, lens, [0] * 24, code="int8", page=64, heads=4, dim=128)
    share(p, [3500], [0, 24])
    q = normal(p.g, sum(new), 16, 128, dtype=BF16)
    check(p, q, lens, new, ["tiles groups", "join_items"], shared=[3500])


def test_more_groups_than_a_block_has_threads():
    seqs, groups = 1800, list(range(0, 1801, 3))
    shared = [16 * (g % 9) for g in range(600)]
    lens = [shared[s // 3] + 1 + s % 40 for s in range(seqs)]
    p = Pages(8, lens, [0] * seqs, code="int8", page=16, heads=1, dim=64)
    share(p, shared, groups)
    widen(p, seqs, 600)
    q = normal(p.g, seqs, 4, 64, dtype=BF16)
    check(p, q, lens, [1] * seqs, ["items", "split groups", "join_items"], shared=shared, groups=groups)


def test_groups_left_out():
    """Sequences of many rows, and prefixes that are soon read again, go as without groups."""
    lens, new = [2000, 1500], [300, 200]
    p = Pages(5, lens, [0, 0], code="int8", page=64, heads=2, dim=128)
    share(p, [1024], [0, 2])
    q = normal(p.g, 500, 8, 128, dtype=BF16)
    for rows, each in ((500, new), (2, [1, 1])):
        alone = kernels(attention(p, q[:rows], lens, each))
        assert not any("groups" in name for name in alone)
        check(p, q[:rows], lens, each, alone, shared=[1024])


def test_two_users_of_the_example_share_a_prefix(monkeypatch):
    """The example with heads wide enough that two users' common tokens are read together while they decode."""
    seen = []

    def record(*args, **kw):
        out = bfft.cache_attention(*args, **kw)
        seen.append(kernels(lambda: bfft.cache_attention(*args, **kw)))
        return out

    monkeypatch.setattr(decode_example, "cache_attention", record)
    r = decode_example.run(prompt=2950, steps=3, q_heads=16, kv_heads=16, dim=256, common=900)
    assert r["attention_rel_error"] < 0.03 and r["gradient_is_adjoint"]
    assert seen[1:] == [["split groups", "join_items"]] * 3


def test_no_bounded_wait_expired_here():
    assert _lib.device_status(0) == 0

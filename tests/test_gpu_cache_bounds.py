"""Attention with first tokens where a chunk of the axis holds as many pages as shared memory does, against the plain
float64 form of the other tests of this attention, with their tolerances."""
import pytest
import torch

from bfft import _lib
from test_gpu_cache import BF16, Pages, normal
from test_gpu_cache_spans import check_spans

pytestmark = pytest.mark.gpu

PARTS = 256 << 20  # bytes that the parts of a call are kept to


@pytest.mark.parametrize("causal, window, sinks", [(True, 80500, 20), (False, 700, 4), (False, 1, 333)])
def test_chunks_of_as_many_pages_as_fit(causal, window, sinks):
    """Heads of 256, pages of 16: the axis of 80 thousand tokens is more than one chunk holds; one sequence is as long,
    the others end far before."""
    lens, new = [600, 512, 900, 1000, 0, 777, 640, 513, 81000], [512] * 8 + [6]
    p = Pages(256, lens, [0] * 9, code="int8", page=16, heads=1, dim=256)
    table = torch.full((9, 5200), -1, dtype=torch.int32, device="cuda")
    table[:, :p.table.shape[1]] = p.table
    q = normal(p.g, sum(new), 32, 256, dtype=BF16)
    assert PARTS // 2 < sum(new) * 32 * 258 * 4 <= PARTS      # one chunk, where it can be
    check_spans(p, q, lens, new, causal=causal, window=window, sinks=sinks, table=table)


@pytest.mark.parametrize("each, kv_heads", [(2, 8), (3, 4)])
def test_chunks_of_as_many_pages_as_fit_for_heads_of_128(each, kv_heads):
    """Row tiles of 8 and of 16 rows."""
    seqs = 8192 // each
    lens = [(37 * s) % 90 for s in range(seqs)]
    p = Pages(each, lens, [0] * seqs, code="e4m3", page=16, heads=kv_heads, dim=128)
    table = torch.full((seqs, 8244), -1, dtype=torch.int32, device="cuda")  # one chunk takes up to 8235
    table[:, :p.table.shape[1]] = p.table
    q = normal(p.g, seqs * each, 32, 128, dtype=BF16)
    assert PARTS // 2 < seqs * each * 32 * 130 * 4 <= PARTS
    check_spans(p, q, lens, [each] * seqs, causal=False, window=9, sinks=5, table=table)


def test_no_bounded_wait_expired_here():
    assert _lib.device_status(0) == 0

"""Row tiles that are half filled or less (up to 128 rows of a kv head) write their rows another way than full ones: as
parts and directly, at odd widths and strides, beside full tiles, against the plain float64 form of the other tests of
this attention, with their tolerances."""
import pytest
import torch

import bfft
from bfft import _lib
from test_gpu_cache import BF16, F16, Pages, cumulative, ints, normal
from test_gpu_cache_kernels import attention, kernels
from test_gpu_cache_spans import check_spans, share

pytestmark = pytest.mark.gpu

FORMS = [({}, ""), ({"window": 700}, ""), ({"window": 700, "sinks": 20}, " sinks")]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype, dim, page", [(BF16, 128, 64), (F16, 64, 16), (BF16, 80, 32), (F16, 48, 128), (BF16, 112, 16)])
@pytest.mark.parametrize("how, form", [({}, ""), ({"window": 6000}, ""), ({"window": 6000, "sinks": 20}, " sinks")])
@pytest.mark.parametrize("causal", [True, False])
def test_parts_of_one_half(code, dtype, dim, page, how, form, causal):
    """Few sequences of 16 to 31 rows of four heads: the axis is cut, its parts are joined."""
    lens, new = [9000, 5000, 24], [16, 31, 24]
    p = Pages(dim, lens, [0] * 3, code=code, page=page, heads=8, dim=dim)
    q = normal(p.g, sum(new), 32, dim, dtype=dtype) * 1.5
    how = {"causal": causal, **how}
    assert kernels(attention(p, q, lens, new, **how)) == ["tiles" + form, "join"]
    first = check_spans(p, q, lens, new, **how)
    again = check_spans(p, q, lens, new, **how)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype, dim, group", [(BF16, 128, 4), (F16, 64, 5), (BF16, 80, 8), (F16, 96, 3)])
@pytest.mark.parametrize("how, form", FORMS)
def test_rows_of_one_half_without_parts(code, dtype, dim, group, how, form):
    """Many sequences: a row tile walks the whole axis.  Beside it full tiles (80 rows of a sequence and more), tiles
    of one row and sequences without tokens."""
    seqs = 90
    new = [20 + i % 12 for i in range(seqs - 3)] + [80, 129, 1]
    lens = [900 + 13 * i % 300 for i in range(seqs)]
    lens[4] = 0
    p = Pages(group, lens, [40] * seqs, code=code, page=32, heads=4, dim=dim)
    q = normal(p.g, sum(new), 4 * group, dim, dtype=dtype) * 1.5
    call = attention(p, q, lens, new, **how)
    assert kernels(call) == ["tiles" + form]
    want, _ = check_spans(p, q, lens, new, **how)
    starts = ints(cumulative(new))
    # odd rows of the output, other strides, the queries themselves, rows behind the last sequence
    odd = torch.full((sum(new), 4 * group, dim + 1), 3.0, dtype=dtype, device="cuda")
    wide = torch.full((4 * group, sum(new), dim + 8), 3.0, dtype=dtype, device="cuda")
    for out in (odd[..., 1:], wide.transpose(0, 1)[..., :dim], q.clone()):
        source = out if out.shape == q.shape and torch.equal(out, q) else q
        bfft.cache_attention(source, p.cache, p.table, ints(lens), starts, out=out, **how)
        assert torch.equal(out, want)
    assert (odd[..., 0] == 3.0).all() and (wide[..., dim:] == 3.0).all()
    more = torch.cat((q, q[:5]))
    left = torch.full_like(more, 5.0)
    bfft.cache_attention(more, p.cache, p.table, ints(lens), starts, out=left, **how)
    assert torch.equal(left[:sum(new)], want) and (left[sum(new):] == 5.0).all()


@pytest.mark.parametrize("dim, group, seqs, each", [(128, 8, 12, 1), (64, 4, 20, 1), (96, 16, 7, 1), (128, 4, 10, 3)])
def test_prefixes_of_one_half(dim, group, seqs, each):
    """A group of up to 128 rows over its prefix."""
    lens = [12000 + each + 31 * i % 200 for i in range(seqs)]
    p = Pages(dim, lens, [0] * seqs, code="int8", page=64, heads=8, dim=dim)
    share(p, [12000], [0, seqs])
    q = normal(p.g, seqs * each, 8 * group, dim, dtype=BF16)
    for how in ({}, {"window": 10000, "sinks": 9}):
        used = kernels(attention(p, q, lens, [each] * seqs, shared=[12000], **how))
        assert used == ["tiles groups", "split groups", "join_items"]
        check_spans(p, q, lens, [each] * seqs, shared=[12000], **how)
    p.cache.v_scale[p.ids[0][3]] = 1e-36                      # a small value scale: the sums are held 2^36 times smaller
    check_spans(p, q, lens, [each] * seqs, shared=[12000])


def test_small_value_scales_in_one_half():
    lens, new = [9000, 5000], [16, 31]
    p = Pages(4, lens, [0] * 2, code="int8", page=64, heads=8, dim=128)
    q = normal(p.g, sum(new), 32, 128, dtype=BF16)
    for ids in p.ids:
        p.cache.v_scale[ids[5]] = 1e-36
    check_spans(p, q, lens, new)
    many = Pages(5, [900] * 90, [0] * 90, code="int8", page=64, heads=4, dim=128)
    for ids in many.ids:
        many.cache.v_scale[ids[5]] = 1e-36
    check_spans(many, normal(many.g, 1800, 16, 128, dtype=BF16), [900] * 90, [20] * 90)


def test_no_bounded_wait_expired_here():
    assert _lib.device_status(0) == 0

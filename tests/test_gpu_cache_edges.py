"""Position and cache calls at the edges of their ranges, against plain float64 forms.

Tolerances are those of the other tests of these calls: 32-bit sums, float16 weights,
one rounding of the output.
"""
import math

import pytest
import torch
from torch.autograd import forward_ad

import bfft
from bfft import _lib
from test_cache_host import pack_append, pack_attention, pack_cache, pack_rotate, pack_sequences
from test_gpu_cache import BF16, F16, HALF_UNIT, Pages, attention64, check_attention, cumulative, ints, normal

pytestmark = pytest.mark.gpu


def takes_tiles(p, q, new, table, *, causal=True, window=0):
    """The rule by which a call goes to the tensor-core tiles: rows of a sequence in the mean, and pairs in all."""
    group, each = q.shape[1] // p.heads, q.shape[0] // len(new)
    cover = table.shape[1] * p.page
    if causal and window:
        cover = min(cover, window)
    return p.dim <= 128 and group <= 128 and each * group >= 48 and q.shape[0] * q.shape[1] * cover * p.dim >= 3e6 * 128


def lost_under(p, q, lens, starts, top, *, scale, causal, window, zero_as=0.0):
    """What float16 weights lose of each output: a weight times its value scale is rounded to float16 with the row's
    largest at 2^top or over, so to within half of 2^-24, which then meets the tokens' codes.  A zero value scale
    takes part in that largest as `zero_as`."""
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    group = q.shape[1] // p.heads
    for s, n in enumerate(lens):
        rows = slice(starts[s], starts[s + 1])
        k, (v, vs) = p.values(0, s, 0, n)[0], p.values(1, s, 0, n)
        codes = torch.where(vs[..., None] > 0, v / vs[..., None], 0.0).abs()
        pos = torch.arange(n - (starts[s + 1] - starts[s]), n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        seen = (key <= pos if causal else key >= 0) & ((key > pos - window) if window else key >= 0)
        for h in range(q.shape[1]):
            j = h // group
            z = (q[rows, h].double() @ k[:, j].T * scale).masked_fill(~seen, -math.inf)
            largest = (torch.softmax(z, -1) * torch.where(vs == 0, zero_as, vs)[:, j]).amax(-1, keepdim=True)
            out[rows, h] = 2.0 ** -(25 + top) * largest * (seen.double() @ codes[:, j])
    return out


def check_relative(p, q, lens, new, *, tiles, scale=None, causal=True, window=0, zero_as=0.0):
    """Every row against its own size: nothing absolute but the last bit of bfloat16's (float16's) smallest values."""
    assert takes_tiles(p, q, new, p.table, causal=causal, window=window) == tiles
    starts = cumulative(new)
    got, lse = bfft.cache_attention(q, p.cache, p.table, ints(lens), ints(starts), softmax_scale=scale, causal=causal,
                                    window=window, return_lse=True)
    factor = p.dim ** -0.5 if scale is None else scale
    want, want_lse, size, slack = attention64(p, q, lens, starts, scale=factor, causal=causal, window=window)
    assert lse.isfinite().all() and got.isfinite().all()
    delta = 2.0 ** -21 * (1 + slack)
    tol = HALF_UNIT[q.dtype] * want.abs() + (2.0 ** -10 + 2 * delta[..., None]) * size
    tol = tol + lost_under(p, q, lens, starts, 10 if tiles else 14, scale=factor, causal=causal, window=window,
                           zero_as=zero_as)
    tol = tol + (2.0 ** -133 if q.dtype == BF16 else 2.0 ** -24)
    assert ((got.double() - want).abs() <= tol).all()
    assert ((lse.double() - want_lse).abs() <= delta + 2.0 ** -20 * (1 + want_lse.abs())).all()
    return got, lse


# ------------------------------------------------------------------------------- small value scales

def small_pages(code, where, lens, *, page=32, dim=128):
    """Pages whose values are ordinary, but for those of `where` in each sequence: about 1e-36."""
    p = Pages(dim + len(lens), lens, [0] * len(lens), code=code, page=page, heads=2, dim=dim)
    for ids in p.ids:
        kept = [i for i in ids if i >= 0]
        p.cache.v_scale[kept if where is None else [i for j, i in enumerate(kept) if j in where]] = 1e-36
    return p


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens, new, tiles", [
    ([700], [1], False),             # one cluster
    ([6000, 41], [1, 1], False),     # chunks and a joining kernel
    ([900], [40], False),            # several rows, and rows that see one page only
    ([4100], [4100], True),          # row tiles, no joining: the first rows see the first page only
    ([4100, 333], [300, 33], True),  # row tiles, chunks joined
])
def test_attention_over_tiny_values(code, dtype, lens, new, tiles):
    """The weights' sum holds 1 / value scale: it may not overflow however small the scales are."""
    p = small_pages(code, None, lens)
    q = normal(p.g, sum(new), 8, 128, dtype=dtype)
    out, _ = check_relative(p, q, lens, new, tiles=tiles)
    if dtype == BF16:
        assert out.abs().amax() > 1e-36


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("where", [{0}, {3}, {0, 1, 2, 3, 4, 5, 6, 7}])
@pytest.mark.parametrize("lens, new, tiles", [
    ([700], [1], False), ([6000, 41], [1, 1], False), ([300], [300], False), ([4100], [4100], True),
    ([4100, 333], [300, 33], True),
])
def test_attention_over_a_tiny_page_among_ordinary_ones(code, where, lens, new, tiles):
    p = small_pages(code, where, lens)
    q = normal(p.g, sum(new), 8, 128, dtype=BF16)
    check_relative(p, q, lens, new, tiles=tiles)


@pytest.mark.parametrize("rows, tiles", [(1, False), (300, True)])
def test_attention_over_scales_without_a_normal_float(rows, tiles):
    """A scale under 2^-126 stands for zeros, as the append has it: its block's tokens count in the sum only."""
    p = small_pages("int8", None, [4100])
    p.cache.v_scale[p.ids[0][1::2]] = 1e-39
    q = normal(p.g, rows, 8, 128, dtype=BF16)
    got = bfft.cache_attention(q, p.cache, p.table, ints([4100]), ints([0, rows]), return_lse=True)
    p.cache.v_scale[p.ids[0][1::2]] = 0.0
    want = bfft.cache_attention(q, p.cache, p.table, ints([4100]), ints([0, rows]), return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[1].isfinite().all()
    check_relative(p, q, [4100], [rows], tiles=tiles)


# ------------------------------------------------------------------------------- what autograd has to know

def step_inputs(rows=2):
    p = Pages(3, [20] * rows, [4] * rows, code="int8", page=16, heads=2, dim=32)
    x = normal(p.g, rows, 2, 32, dtype=BF16)
    return p, x, normal(p.g, rows, 4, 32, dtype=BF16), ints([20] * rows), ints(list(range(rows + 1))), bfft.rotary_table(64, 32)


def test_in_place_rotation_is_seen_by_saved_tensors():
    table = bfft.rotary_table(16, 32)
    x, where = normal(torch.Generator("cuda").manual_seed(1), 4, 2, 32), ints([0, 1, 2, 3])
    w = torch.ones_like(x).requires_grad_(True)
    loss = (w * x).sum()                                     # saves x for w's gradient
    bfft.rotate_positions(x, where, table, out=x)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()


def test_writes_raise_the_versions():
    p, x, q, held, starts, table = step_inputs()
    out = torch.empty_like(q)
    view = torch.empty(2, 4, 64, dtype=BF16, device="cuda")
    before = [t._version for t in (*p.cache, out, view)]
    bfft.append_rotated(p.cache, x, x, p.table, held, starts, table, q=q)
    bfft.cache_attention(q, p.cache, p.table, ints([21, 21]), starts, out=out)
    bfft.rotate_positions(q, held, table, out=view[..., 16:48])
    after = [t._version for t in (*p.cache, out, view)]
    assert all(a > b for a, b in zip(after, before))
    reads = [t._version for t in (x, q, held, starts, table, *p.cache)]
    bfft.rotate_positions(q, held, table)
    bfft.cache_attention(q, p.cache, p.table, ints([21, 21]), starts)
    bfft.read_cache(p.cache, p.table, held, starts, 2)
    assert reads == [t._version for t in (x, q, held, starts, table, *p.cache)]


def test_calls_in_and_on_tensors_of_inference_mode():
    with torch.inference_mode():
        p, x, q, held, starts, table = step_inputs()
        bfft.append_rotated(p.cache, x, x, p.table, held, starts, table, q=q)
        want = bfft.cache_attention(q, p.cache, p.table, ints([21, 21]), starts, out=torch.empty_like(q))
    # tensors made in inference mode have no versions; they still can be written
    bfft.append_rotated(p.cache, x, x, p.table, held, starts, table, q=q)
    got = bfft.cache_attention(q, p.cache, p.table, ints([21, 21]), starts, out=torch.empty_like(q))
    assert torch.equal(got, want)


def test_outputs_that_require_a_gradient_are_refused():
    p, x, q, held, starts, table = step_inputs()
    out = torch.empty_like(q).requires_grad_(True)
    lens = ints([21, 21])
    count = _lib.launch_counter()
    with pytest.raises(ValueError, match="gradient"):
        bfft.rotate_positions(q, held, table, out=out)
    with pytest.raises(ValueError, match="gradient"):
        bfft.cache_attention(q, p.cache, p.table, lens, starts, out=out)
    assert _lib.launch_counter() == count
    with torch.no_grad():                                    # as torch's own out arguments: only the graph forbids it
        assert bfft.rotate_positions(q, held, table, out=out) is out
        assert torch.equal(out, bfft.rotate_positions(q, held, table))
        bfft.cache_attention(q, p.cache, p.table, lens, starts, out=out)
        assert torch.equal(out, bfft.cache_attention(q, p.cache, p.table, lens, starts))


def test_calls_without_a_gradient_refuse_inputs_that_require_one():
    """None of these may return a result that silently has no gradient."""
    p, x, q, held, starts, table = step_inputs()
    lens, k_scale = ints([21, 21]), p.cache.k_scale.clone().requires_grad_(True)
    learned = bfft.PagedCache(p.cache.k, p.cache.v, k_scale, p.cache.v_scale)

    def leaf(t):
        return t.clone().requires_grad_(True)

    rot, app, att, read = bfft.rotate_positions, bfft.append_rotated, bfft.cache_attention, bfft.read_cache
    calls = [
        (rot, (q, held, leaf(table)), {}), (rot, (leaf(q), held, leaf(table)), {}),
        (app, (p.cache, leaf(x), x, p.table, held, starts, table), {}),
        (app, (p.cache, x, leaf(x), p.table, held, starts, table), {}),
        (app, (p.cache, x, x, p.table, held, starts, leaf(table)), {}),
        (app, (p.cache, x, x, p.table, held, starts, table), {"q": leaf(q)}),
        (app, (learned, x, x, p.table, held, starts, table), {}),
        (att, (leaf(q), p.cache, p.table, lens, starts), {}),
        (att, (q, learned, p.table, lens, starts), {}),
        (read, (learned, p.table, held, starts, 2), {}),
    ]
    before = [t.clone() for t in p.cache]
    count = _lib.launch_counter()
    for fn, args, kw in calls:
        with pytest.raises(ValueError, match="gradient"):
            fn(*args, **kw)
    assert _lib.launch_counter() == count
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, p.cache))
    with torch.no_grad():
        for fn, args, kw in calls:
            fn(*args, **kw)


def test_forward_mode_tangents_are_refused():
    p, x, q, held, starts, table = step_inputs()
    lens = ints([21, 21])
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        dual_x = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: bfft.rotate_positions(dual, held, table),
                     lambda: bfft.rotate_positions(q, held, forward_ad.make_dual(table, torch.ones_like(table))),
                     lambda: bfft.append_rotated(p.cache, dual_x, x, p.table, held, starts, table),
                     lambda: bfft.append_rotated(p.cache, x, x, p.table, held, starts, table, q=dual),
                     lambda: bfft.cache_attention(dual, p.cache, p.table, lens, starts),
                     lambda: bfft.rotate_positions(q, held, table, out=forward_ad.make_dual(q.clone(), torch.ones_like(q)))):
            with pytest.raises(ValueError, match="gradient"):
                call()
        assert forward_ad.unpack_dual(bfft.rotate_positions(q, held, table)).tangent is None


# ------------------------------------------------------------------------------- overlapping memory

def test_outputs_that_overlap_are_refused():
    p, x, q, held, starts, table = step_inputs()
    lens, where = ints([21, 21]), held
    wide = normal(p.g, 2, 9, 80, dtype=BF16)
    src = wide[:, 1:5, 8:40]
    flat = normal(p.g, 2000, dtype=BF16)
    outs = [
        wide[:, 2:6, 8:40],                                   # a head on
        wide[:, 1:5, 9:41],                                   # an element on
        wide[:, 0:8:2, 8:40],                                 # other strides over the same memory
        wide.new_zeros(1, 4, 32).expand(2, 4, 32),            # rows written twice
        torch.as_strided(flat, (2, 4, 32), (64, 16, 1)),      # heads that run into each other
    ]
    count = _lib.launch_counter()
    for out in outs:
        with pytest.raises(ValueError, match="overlap"):
            bfft.rotate_positions(src, where, table, out=out)
        with pytest.raises(ValueError, match="overlap"):
            bfft.cache_attention(src, p.cache, p.table, lens, starts, out=out)
    # keys and values in one place: fine to read, not to append to
    one = bfft.PagedCache(p.cache.k, p.cache.k, p.cache.k_scale, p.cache.k_scale)
    for bad in (one, bfft.PagedCache(p.cache.k, p.cache.v, p.cache.k_scale, p.cache.k_scale)):
        with pytest.raises(ValueError, match="overlap"):
            bfft.append_rotated(bad, x, x, p.table, held, starts, table)
    assert _lib.launch_counter() == count
    k, v = bfft.read_cache(one, p.table, ints([0, 0]), starts, 2)
    assert torch.equal(k, v)


def test_outputs_between_the_inputs_rows_are_taken():
    p, x, q, held, starts, table = step_inputs()
    lens = ints([21, 21])
    wide = normal(p.g, 2, 9, 80, dtype=BF16)
    for src, out in ((wide[:, 0:8:2, :32], wide[:, 1:9:2, :32]),          # heads in turn
                     (wide[:, 1:5, :32], wide[:, 1:5, 32:64]),            # halves of the rows
                     (wide[:1].expand(2, 9, 80)[:, 2:6, :32], wide.new_zeros(2, 4, 32)),
                     (wide[:, 3:7, 8:40], wide[:, 3:7, 8:40])):           # in place
        want = bfft.rotate_positions(src, held, table)
        want_y = bfft.cache_attention(src, p.cache, p.table, lens, starts)
        kept = src.clone()
        assert torch.equal(bfft.cache_attention(src, p.cache, p.table, lens, starts, out=out), want_y)
        src.copy_(kept) if src.data_ptr() == out.data_ptr() else None
        assert torch.equal(bfft.rotate_positions(src, held, table, out=out), want)


# ------------------------------------------------------------------------------- tables wider than the lengths

@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attention_of_many_rows_over_a_wide_table(page, code):
    """Parts of 512 sequences over 131072 tokens would take more than the workspace's limit: chunks of over 8000 tokens."""
    lens = [70001] + [5 + 31 * i % 300 for i in range(511)]
    p = Pages(page, lens, [0] * 512, code=code, page=page, heads=2, dim=128)
    table = torch.full((512, 131072 // page), -1, dtype=torch.int32, device="cuda")
    table[:, :p.table.shape[1]] = p.table
    q = normal(p.g, 2048, 16, 128, dtype=BF16) * 1.5
    assert not takes_tiles(p, q, [4] * 512, table)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    bfft.cache_attention(q, p.cache, table, ints(lens), ints(cumulative([4] * 512)))
    assert torch.cuda.max_memory_allocated() - held < (256 << 20) + 2 * q.numel() * 2
    check_attention(p, q, lens, [4] * 512, table=table)
    check_attention(p, q, lens, [4] * 512, table=table, causal=False, window=30000)


# ------------------------------------------------------------------------------- the C entries' status

def test_a_device_that_is_not_there_fails_its_own_call_only():
    """The failed call's error does not stay behind for the next one to report."""
    lib = _lib.load()
    p, x, q, held, starts, table = step_inputs()
    out, lens = torch.empty_like(q), ints([21, 21])
    k, v = torch.empty_like(x), torch.empty_like(x)
    stream = torch.cuda.current_stream().cuda_stream
    cache = pack_cache(*(t.data_ptr() for t in p.cache), p.cache.k.shape[0], 2, 16, 32, 0)

    def seqs(lens):
        return pack_sequences(p.table.data_ptr(), p.table.stride(0), lens.data_ptr(), starts.data_ptr(), 2, p.table.shape[1], 2)

    def rotate(device):
        d = pack_rotate(1, 2, 4, 32, 32, 0, 128, 32, 0, 128, 32, 0, 1, 64, 2, 0, 0, 0, device)
        return lib.bfft_rotate_positions(d, q.data_ptr(), held.data_ptr(), table.data_ptr(), out.data_ptr(), stream)

    def append(device):
        d = pack_append(x.data_ptr(), x.data_ptr(), 0, 0, 0, 0, 64, 32, 64, 32, 0, 0, 0, 0, 0, 0, 0, 2, 0, 0, device)
        return lib.bfft_cache_append(cache, seqs(held), d, stream)

    def read(device):
        return lib.bfft_cache_read(cache, seqs(held), 2, k.data_ptr(), v.data_ptr(), device, stream)

    def attend(device):
        d = pack_attention(q.data_ptr(), out.data_ptr(), 0, 128, 32, 128, 32, 4, 2, 1, 0, 0.2, 0, 0, device)
        return lib.bfft_cache_attention(cache, seqs(lens), d, stream)

    calls = (rotate, append, read, attend)
    for bad in calls:
        for good in calls:
            assert bad(99) == _lib.ERR_CUDA and "99" in _lib.last_error()
            assert good(0) == _lib.OK, (bad.__name__, good.__name__, _lib.last_error())
        assert bad(99) == _lib.ERR_CUDA
        y, _ = bfft.run_fft(torch.ones(64, dtype=torch.complex64, device="cuda"), "dit", profile_hash=None)
        assert abs(complex(y[0]) - 64) < 1e-3
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------- queries near the largest float

@pytest.mark.parametrize("new, tiles", [([1], False), ([40], False), ([300], True)])
def test_attention_of_queries_near_the_largest_float(new, tiles):
    """bfloat16 queries go through float16 by a power of two of their row, up to the type's last binade."""
    p = Pages(33, [4100], [0], code="int8", page=64, heads=2, dim=128)
    p.cache.k_scale.mul_(2.0 ** -120)
    q = normal(p.g, new[0], 8, 128).clamp(-3.9, 3.9)
    q[..., 5] = 3.9
    q = (q * 2.0 ** 126).to(BF16)                            # 3.9 * 2^126 lies in [2^127, 2^128)
    assert q.isfinite().all() and (q.abs().amax(-1) >= 2.0 ** 127).all()
    check_relative(p, q, [4100], new, tiles=tiles, scale=2.0 ** -8)

"""Limits of the position and cache calls that the host decides, without a GPU."""
import ctypes

import pytest

from bfft import _build, _lib
from test_cache_host import A, cache_desc, pack_attention, pack_sequences


@pytest.fixture(scope="module")
def lib():
    _build.build(verbose=False)
    return _lib.load()


def workspace(lib, *, seqs, tokens, heads, dim, width, page=64, kv_heads=8, window=0):
    """Bytes that an attention of `tokens` rows over a table of `width` tokens a sequence asks for."""
    n = ctypes.c_size_t()
    q = pack_attention(A, A, 0, heads * dim, dim, heads * dim, dim, heads, 2, 1, window, 1.0, 0, 0, 0)
    s = pack_sequences(A, width // page, A, A, seqs, width // page, tokens)
    assert lib.bfft_cache_attention_workspace(cache_desc(pages=100000, heads=kv_heads, page=page, dim=dim), s, q,
                                              ctypes.byref(n)) == _lib.OK
    return n.value


LIMIT = 256 << 20  # of the parts of a call, where one part of each row is less


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("seqs, each, heads, dim", [
    (512, 4, 64, 128), (256, 1, 32, 128), (64, 1, 128, 64), (2000, 1, 32, 96), (512, 2, 32, 256), (64, 40, 8, 128),
])
@pytest.mark.parametrize("width", [4096, 131072])
def test_workspace_is_bounded_whatever_the_tables_width(lib, page, seqs, each, heads, dim, width):
    got = workspace(lib, seqs=seqs, tokens=seqs * each, heads=heads, dim=dim, width=width, page=page)
    one_part = seqs * each * heads * (dim + 2) * 4
    assert got <= max(LIMIT, 2 * one_part)


def test_workspace_of_an_axis_of_two_million_tokens(lib):
    """A chunk's page entries are held in shared memory, so the axis is cut into that many at least."""
    one_part = 512 * 4 * 64 * 130 * 4
    got = workspace(lib, seqs=512, tokens=2048, heads=64, dim=128, width=1 << 21, page=16)
    assert got <= -(-(1 << 21) // 65536) * one_part


def test_workspace_of_few_rows_is_small(lib):
    assert workspace(lib, seqs=1, tokens=1, heads=32, dim=128, width=704) == 0
    assert workspace(lib, seqs=64, tokens=64, heads=32, dim=128, width=32768) <= 64 * 32 * 16 * 130 * 4

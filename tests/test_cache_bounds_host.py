"""Where a plan of the attention meets what a launch may ask for, without a GPU."""
import ctypes

import pytest

from bfft import _build, _lib
from test_cache_host import A, cache_desc, pack_attention, pack_sequences
from test_cache_spans_host import span_desc


@pytest.fixture(scope="module")
def lib():
    _build.build(verbose=False)
    return _lib.load()


MOST = 226 * 1024  # bytes of shared memory that a CTA of the kernel of few rows is given


def held(dim, rows, pages):
    """Bytes that the kernel of few rows needs for a chunk that touches `pages` pages: the warps' rings or, in their
    place, the rows' parts, and 20 bytes a page."""
    return 1024 + max(4 * 2 * 4 * 16 * dim, 5 * rows * (dim + 2) * 4) + 20 * pages + 64


@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("dim, seqs, each, q_heads, kv_heads, rows", [
    (256, 1, 4096, 32, 1, 8), (128, 4096, 2, 32, 8, 8), (128, 2731, 3, 32, 4, 16), (64, 8192, 2, 32, 8, 8),
    (160, 3500, 2, 32, 8, 8),
])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("sinks", [0, 4, 200])
def test_the_pages_of_the_longest_chunk_fit(lib, page, dim, seqs, each, q_heads, kv_heads, rows, causal, sinks):
    """Many rows over a wide axis: chunks grow as far as shared memory holds their pages.  A window and first tokens
    cut it at up to four places more than a page's ends: five entries beside the whole pages, without them two."""
    tokens = seqs * each
    part = tokens * q_heads * (dim + 2) * 4
    assert 128 << 20 < part <= 256 << 20                     # one chunk, where it can be
    spare = 5 if sinks else 2
    room = (MOST - held(dim, rows, 0)) // 20
    cache = cache_desc(pages=100000, heads=kv_heads, page=page, dim=dim)
    tile = max(1, rows // (q_heads // kv_heads))
    cut = set()
    for pages in range(room - 12, room + 9):                 # the axis, in pages: across the bound
        cover = min(pages * page, 1 << 20)
        # causal: the window, its rows and its ends in a page; else the table's width
        window = cover - (tile - 1) - 15 - (sinks + 15) // 16 * 16 if causal else 300
        width = pages + 999 if causal else pages
        q = pack_attention(A, A, 0, q_heads * dim, dim, q_heads * dim, dim, q_heads, 2, causal, window, 1.0, 0, 0, 0)
        s = pack_sequences(A, width, A, A, seqs, width, tokens)
        n = ctypes.c_size_t()
        assert lib.bfft_cache_attention_span_workspace(cache, s, q, span_desc(sinks=sinks, n=0), ctypes.byref(n)) == _lib.OK
        assert n.value % part == 0
        chunks = max(1, n.value // part)
        cut.add(chunks)
        assert held(dim, rows, -(-cover // chunks) // page + spare) <= MOST
    assert cut == ({1, 2} if (room + 8) * page <= 1 << 20 else {1})

"""Checks and workspaces of the attention with first tokens and shared prefixes, without a GPU."""
import ctypes
import struct

import pytest

from bfft import _build, _lib
from test_cache_host import A, attention_desc, cache_desc, pack_attention, pack_sequences, seq_desc


@pytest.fixture(scope="module")
def lib():
    _build.build(verbose=False)
    return _lib.load()


def span_desc(sinks=0, groups=A, shared=A, n=1):
    return struct.pack("q2Qq", sinks, groups, shared, n)


def test_descriptor_matches_the_header():
    text = open(_build.INCLUDE + "/bfft.h").read()
    body = text.split("typedef struct bfft_span_desc {")[1].split("} bfft_span_desc")[0]
    while "/*" in body:
        a, b = body.index("/*"), body.index("*/") + 2
        body = body[:a] + body[b:]
    assert 8 * sum(len(part.split(",")) for part in body.split(";") if part.strip()) == len(span_desc())


@pytest.mark.parametrize("span, status", [
    (span_desc(sinks=-1), _lib.ERR_VALUE), (span_desc(sinks=1 << 31), _lib.ERR_VALUE), (span_desc(n=-1), _lib.ERR_SHAPE),
    (span_desc(shared=0), _lib.ERR_VALUE), (span_desc(groups=0, n=2), _lib.ERR_VALUE),
    (span_desc(shared=A + 2), _lib.ERR_VALUE), (span_desc(groups=A + 1), _lib.ERR_VALUE), (None, _lib.ERR_VALUE),
])
def test_span_checks(lib, span, status):
    n = ctypes.c_size_t()
    assert lib.bfft_cache_attention_span(cache_desc(), seq_desc(), attention_desc(), span, None) == status
    assert lib.bfft_cache_attention_span_workspace(cache_desc(), seq_desc(), attention_desc(), span, ctypes.byref(n)) == status
    assert _lib.last_error()


def test_call_checks(lib):
    n = ctypes.c_size_t()
    for span in (span_desc(), span_desc(sinks=3, n=0)):
        assert lib.bfft_cache_attention_span(cache_desc(), seq_desc(), attention_desc(window=-1), span, None) == _lib.ERR_VALUE
        assert lib.bfft_cache_attention_span(cache_desc(), seq_desc(tokens=0), attention_desc(), span, None) == _lib.OK
        assert lib.bfft_cache_attention_span_workspace(cache_desc(), seq_desc(tokens=0), attention_desc(), span,
                                                       ctypes.byref(n)) == _lib.OK and n.value == 0
        wide = seq_desc(pages=1 << 28, seqs=3)
        assert lib.bfft_cache_attention_span_workspace(cache_desc(), wide, attention_desc(window=0 if span == span_desc() else 9),
                                                       span, ctypes.byref(n)) == _lib.ERR_SHAPE
    assert lib.bfft_cache_attention_span_workspace(cache_desc(), seq_desc(), attention_desc(), span_desc(), None) == _lib.ERR_VALUE


def workspace(lib, span, *, seqs, tokens, heads, dim, width, page=64, kv_heads=8, window=0):
    n = ctypes.c_size_t()
    q = pack_attention(A, A, 0, heads * dim, dim, heads * dim, dim, heads, 2, 1, window, 1.0, 0, 0, 0)
    s = pack_sequences(A, width // page, A, A, seqs, width // page, tokens)
    assert lib.bfft_cache_attention_span_workspace(cache_desc(pages=100000, heads=kv_heads, page=page, dim=dim), s, q, span,
                                                   ctypes.byref(n)) == _lib.OK
    return n.value


def test_workspaces(lib):
    """Without sharing as the windowed call's; with it, bounded by the rows and the GPU's size, not the table's width."""
    for window in (0, 512):
        plain = ctypes.c_size_t()
        q = pack_attention(A, A, 0, 4096, 128, 4096, 128, 32, 2, 1, window, 1.0, 0, 0, 0)
        s = pack_sequences(A, 64, A, A, 3, 64, 300)
        assert lib.bfft_cache_attention_workspace(cache_desc(pages=1000, heads=8, page=64, dim=128), s, q,
                                                  ctypes.byref(plain)) == _lib.OK
        same = span_desc(n=0) if window else span_desc(sinks=9, n=0)
        assert workspace(lib, same, seqs=3, tokens=300, heads=32, dim=128, width=4096, window=window) == plain.value
    narrow, wide = (workspace(lib, span_desc(), seqs=64, tokens=64, heads=32, dim=128, width=w) for w in (4096, 1 << 20))
    assert narrow == wide < 128 << 20


def test_workspace_with_groups_is_bounded(lib):
    """Where the parts would pass 512 MB the call is made, and its workspace counted, as without groups."""
    for seqs, each, heads in ((64, 1, 32), (4096, 1, 32), (4096, 1, 64), (4096, 31, 64), (20000, 7, 128), (512, 4, 64)):
        n, plain = ctypes.c_size_t(), ctypes.c_size_t()
        q = pack_attention(A, A, 0, heads * 128, 128, heads * 128, 128, heads, 2, 1, 0, 1.0, 0, 0, 0)
        s = pack_sequences(A, 512, A, A, seqs, 512, seqs * each)
        c = cache_desc(pages=100000, heads=8, page=64, dim=128)
        assert lib.bfft_cache_attention_span_workspace(c, s, q, span_desc(), ctypes.byref(n)) == _lib.OK
        assert lib.bfft_cache_attention_workspace(c, s, q, ctypes.byref(plain)) == _lib.OK
        assert n.value <= 512 << 20 or n.value == plain.value
        if seqs * each <= 4096:
            assert n.value <= 512 << 20

"""Rotation tables and the position and cache calls' checks, without a GPU."""
import ctypes
import math
import struct

import pytest
import torch

import bfft
from bfft import _build, _lib

# struct bfft_rotate_desc, bfft_cache_desc, ... of include/bfft.h: every field is 8 bytes wide
pack_rotate = struct.Struct("19q").pack
pack_cache = struct.Struct("4Q5q").pack
pack_sequences = struct.Struct("Qq2Q3q").pack
pack_append = struct.Struct("6Q15q").pack
pack_attention = struct.Struct("3Q8qdQ2q").pack


@pytest.fixture(scope="module")
def lib():
    _build.build(verbose=False)
    return _lib.load()


def angles(positions, rotated, base=10000.0):
    w = [base ** (-2 * j / rotated) for j in range(rotated // 2)]
    return [[p * x for x in w] for p in range(positions)], w


def test_rotary_table_is_float64_rounded_once():
    t = bfft.rotary_table(300, 10, base=500.0, amplitude=1.5, device="cpu")
    assert t.shape == (300, 5, 2) and t.dtype == torch.float32
    a, _ = angles(300, 10, 500.0)
    want = torch.tensor([[(1.5 * math.cos(x), 1.5 * math.sin(x)) for x in row] for row in a], dtype=torch.float64)
    # float64 angles of up to 300 are off by 300 * 2^-52; then one rounding
    assert ((t.double() - want).abs() <= 2.0 ** -24 * want.abs() + 1e-12).all()


def test_rotary_table_scalings():
    def frequencies(**kw):  # the angle of position 1
        t = bfft.rotary_table(2, 16, device="cpu", **kw)[1].double()
        return torch.atan2(t[:, 1], t[:, 0])

    plain = frequencies()
    assert torch.allclose(frequencies(scaling="linear", factor=4.0), plain / 4, rtol=1e-6)
    ntk = frequencies(scaling="ntk", factor=4.0)
    assert torch.allclose(ntk[0], plain[0], rtol=1e-6) and torch.allclose(ntk[-1], plain[-1] / 4, rtol=1e-5)
    banded = frequencies(scaling="banded", factor=4.0, original=1000, low_turns=1.0, high_turns=32.0)
    turns = 1000 * plain / (2 * math.pi)
    assert torch.allclose(banded[turns > 32], plain[turns > 32], rtol=1e-6)
    assert torch.allclose(banded[turns < 1], plain[turns < 1] / 4, rtol=1e-5)
    middle = (turns > 1) & (turns < 32)
    assert middle.any() and ((banded < plain) & (banded > plain / 4))[middle].all()


@pytest.mark.parametrize("args, kw", [
    ((0, 8), {}), ((4, 7), {}), ((4, 0), {}), ((4, 8), {"scaling": "cubic"}), ((4, 8), {"factor": 0.5}),
    ((4, 8), {"base": -1.0}), ((4, 8), {"scaling": "banded", "factor": 2.0}),
    ((4, 8), {"scaling": "banded", "original": 100, "low_turns": 5.0, "high_turns": 5.0}),
])
def test_rotary_table_refusals(args, kw):
    with pytest.raises(ValueError):
        bfft.rotary_table(*args, device="cpu", **kw)


@pytest.mark.parametrize("args, kw", [
    ((0, 1, 16, 16), {}), ((1, 0, 16, 16), {}), ((1, 1, 24, 16), {}), ((1, 1, 16, 24), {}), ((1, 1, 16, 272), {}),
    ((1, 1, 16, 16), {"code": "int4"}),
])
def test_paged_cache_refusals(args, kw):
    with pytest.raises(ValueError):
        bfft.paged_cache(*args, device="cpu", **kw)


def test_paged_cache_shapes():
    c = bfft.paged_cache(5, 3, 32, 48, code="e4m3", device="cpu")
    assert c.k.shape == c.v.shape == (5, 3, 32, 48) and c.k.dtype == torch.float8_e4m3fn
    assert c.k_scale.shape == c.v_scale.shape == (5, 3) and not c.k_scale.any()


def test_calls_refuse_host_tensors():
    c = bfft.paged_cache(2, 1, 16, 16, device="cpu")
    x, i = torch.zeros(1, 1, 16, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        bfft.rotate_positions(x, i[:1], bfft.rotary_table(4, 16, device="cpu"))
    with pytest.raises(ValueError, match="CUDA"):
        bfft.append_rotated(c, x, x, i[None], i[:1], i)
    with pytest.raises(ValueError, match="CUDA"):
        bfft.read_cache(c, i[None], i[:1], i, 1)
    with pytest.raises(ValueError, match="CUDA"):
        bfft.cache_attention(x, c, i[None], i[:1], i)


A = 1 << 20  # a 16-byte aligned address: nothing dereferences it before a launch


def cache_desc(k=A, v=A, ks=A, vs=A, pages=4, heads=2, page=16, dim=32, code=0):
    return pack_cache(k, v, ks, vs, pages, heads, page, dim, code)


def seq_desc(table=A, lens=A, starts=A, seqs=1, pages=4, tokens=3):
    return pack_sequences(table, pages, lens, starts, seqs, pages, tokens)


def attention_desc(q=A, out=A, heads=4, kind=2, window=0, scale=1.0, ws=0, size=0):
    return pack_attention(q, out, 0, 128, 32, 128, 32, heads, kind, 1, window, scale, ws, size, 0)


def append_desc(k=A, v=A, q=0, out=0, table=A, rotated=32, kind=2, layout=0, q_heads=0):
    return pack_append(k, v, q, out, 0, table, 64, 32, 64, 32, 0, 0, 0, 0, 100, rotated, q_heads, kind, layout, 0, 0)


def rotate_desc(tokens=3, dim=32, rotated=32, kind=2, layout=0, direction=0):
    return pack_rotate(1, tokens, 2, dim, rotated, 0, 64, 32, 0, 64, 32, 0, 1, 100, kind, layout, direction, 0, 0)


def test_descriptors_match_the_header():
    """Every field of the header's descriptors is 8 bytes wide, as the packed forms are."""
    text = open(_build.INCLUDE + "/bfft.h").read()
    for name, desc in (("rotate", rotate_desc()), ("cache", cache_desc()), ("sequence", seq_desc()),
                       ("append", append_desc()), ("attention", attention_desc())):
        body = text.split(f"typedef struct bfft_{name}_desc {{")[1].split("}")[0]
        body = "".join(line.split("/*")[0] for line in body.splitlines())
        fields = sum(len(part.split(",")) for part in body.split(";") if part.strip())
        assert len(desc) == 8 * fields, name
    assert struct.calcsize("Q") == ctypes.sizeof(ctypes.c_void_p)


@pytest.mark.parametrize("cache, seqs, status", [
    (cache_desc(k=0), seq_desc(), _lib.ERR_VALUE), (cache_desc(v=A + 8), seq_desc(), _lib.ERR_VALUE),
    (cache_desc(ks=A + 2), seq_desc(), _lib.ERR_VALUE), (cache_desc(code=2), seq_desc(), _lib.ERR_VALUE),
    (cache_desc(page=24), seq_desc(), _lib.ERR_SHAPE), (cache_desc(dim=24), seq_desc(), _lib.ERR_SHAPE),
    (cache_desc(dim=272), seq_desc(), _lib.ERR_SHAPE), (cache_desc(heads=0), seq_desc(), _lib.ERR_SHAPE),
    (cache_desc(pages=0), seq_desc(), _lib.ERR_SHAPE), (cache_desc(), seq_desc(table=0), _lib.ERR_VALUE),
    (cache_desc(), seq_desc(lens=A + 1), _lib.ERR_VALUE), (cache_desc(), seq_desc(seqs=0), _lib.ERR_SHAPE),
    (cache_desc(), seq_desc(tokens=-1), _lib.ERR_SHAPE), (cache_desc(), seq_desc(pages=0), _lib.ERR_SHAPE),
])
def test_cache_and_sequence_checks(lib, cache, seqs, status):
    n = ctypes.c_size_t()
    assert lib.bfft_cache_append(cache, seqs, append_desc(), None) == status
    assert lib.bfft_cache_read(cache, seqs, 2, A, A, 0, None) == status
    assert lib.bfft_cache_attention(cache, seqs, attention_desc(), None) == status
    assert lib.bfft_cache_attention_workspace(cache, seqs, attention_desc(), ctypes.byref(n)) == status
    assert _lib.last_error()


def test_call_checks(lib):
    c, s, n = cache_desc(), seq_desc(), ctypes.c_size_t()
    for desc, status in ((append_desc(k=0), _lib.ERR_VALUE), (append_desc(v=A + 1), _lib.ERR_VALUE),
                         (append_desc(kind=3), _lib.ERR_VALUE), (append_desc(layout=2), _lib.ERR_VALUE),
                         (append_desc(rotated=34), _lib.ERR_SHAPE), (append_desc(rotated=0), _lib.ERR_SHAPE),
                         (append_desc(q=A), _lib.ERR_VALUE), (append_desc(q=A, out=A), _lib.ERR_SHAPE)):
        assert lib.bfft_cache_append(c, s, desc, None) == status
    for desc, status in ((attention_desc(q=0), _lib.ERR_VALUE), (attention_desc(kind=0), _lib.ERR_UNSUPPORTED),
                         (attention_desc(heads=3), _lib.ERR_SHAPE), (attention_desc(window=-1), _lib.ERR_VALUE),
                         (attention_desc(scale=math.inf), _lib.ERR_VALUE), (attention_desc(out=A + 1), _lib.ERR_VALUE)):
        assert lib.bfft_cache_attention(c, s, desc, None) == status
        assert lib.bfft_cache_attention_workspace(c, s, desc, ctypes.byref(n)) == status
    assert lib.bfft_cache_attention_workspace(c, s, attention_desc(), None) == _lib.ERR_VALUE
    assert lib.bfft_cache_read(c, s, 3, A, A, 0, None) == _lib.ERR_VALUE
    assert lib.bfft_cache_read(c, s, 2, A + 8, A, 0, None) == _lib.ERR_VALUE
    for desc, status in ((rotate_desc(dim=31), _lib.ERR_SHAPE), (rotate_desc(rotated=34), _lib.ERR_SHAPE),
                         (rotate_desc(rotated=0), _lib.ERR_SHAPE), (rotate_desc(kind=5), _lib.ERR_VALUE),
                         (rotate_desc(layout=-1), _lib.ERR_VALUE), (rotate_desc(direction=2), _lib.ERR_VALUE),
                         (rotate_desc(tokens=-1), _lib.ERR_SHAPE), (rotate_desc(dim=514, rotated=4), _lib.ERR_SHAPE)):
        assert lib.bfft_rotate_positions(desc, A, A, A, A, None) == status
    assert lib.bfft_rotate_positions(rotate_desc(), A, A, A + 4, A, None) == _lib.ERR_VALUE
    assert lib.bfft_rotate_positions(rotate_desc(), None, A, A, A, None) == _lib.ERR_VALUE
    # nothing to do: no device is touched
    assert lib.bfft_rotate_positions(rotate_desc(tokens=0), A, A, A, A, None) == _lib.OK
    empty = seq_desc(tokens=0)
    assert lib.bfft_cache_append(c, empty, append_desc(), None) == _lib.OK
    assert lib.bfft_cache_read(c, empty, 2, A, A, 0, None) == _lib.OK
    assert lib.bfft_cache_attention(c, empty, attention_desc(), None) == _lib.OK

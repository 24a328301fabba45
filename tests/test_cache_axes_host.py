"""Positions of several axes without a GPU: the pairs' axes, tables, and the C entry points' checks."""
import ctypes
import struct

import pytest
import torch

import bfft
from bfft import _build, _lib, cache
from test_cache_host import A, append_desc, cache_desc, rotate_desc, seq_desc


@pytest.fixture(scope="module")
def lib():
    _build.build(verbose=False)
    return _lib.load()


def test_pairs_axes():
    assert cache._axes_map((2, 1, 3), "blocks") == (0, 0, 1, 2, 2, 2)
    assert cache._axes_map((2, 1, 3), "cyclic") == (0, 1, 2, 0, 2, 2)
    assert cache._axes_map((24, 20, 20), "cyclic") == (0, 1, 2) * 20 + (0,) * 4
    assert cache._axes_map([0, 2], "cyclic") == (1, 1)
    assert cache._axes_bytes((1, 2), "blocks") == bytes((2, 0, 1, 1))


@pytest.mark.parametrize("axes", [(), (1,) * 5, (0, 0), (-1, 2), (1.0, 1), (True, 1), (200, 57)])
def test_bad_axes(axes):
    with pytest.raises(ValueError, match="axes"):
        cache._axes_map(axes, "blocks")


def test_numbers_that_compare_equal_are_not_taken_for_each_other():
    assert cache._axes((1, 6), "blocks") == bytes((2, 0, 1, 1, 1, 1, 1, 1)) == cache._axes([1, 6], "blocks")
    for axes in ((True, 6), (1.0, 6)):
        with pytest.raises(ValueError, match="axes"):
            cache._axes(axes, "blocks")


def test_bad_orders_and_spectra():
    for kw in ({"axis_order": "rows", "axes": (4,)}, {"spectrum": "own", "axes": (4,)}, {"spectrum": "axial"},
               {"axes": (3,)}):
        with pytest.raises(ValueError):
            bfft.rotary_table(4, 8, device="cpu", **kw)


@pytest.mark.parametrize("order", ["blocks", "cyclic"])
def test_tables_of_several_axes(order):
    axes = (3, 5, 4)
    plain = bfft.rotary_table(9, 24, device="cpu")
    assert torch.equal(bfft.rotary_table(9, 24, axes=axes, axis_order=order, device="cpu"), plain)
    own = bfft.rotary_table(9, 24, axes=axes, axis_order=order, spectrum="axial", device="cpu")
    of = torch.tensor(cache._axes_map(axes, order))
    for a, n in enumerate(axes):
        assert torch.equal(own[:, of == a], bfft.rotary_table(9, 2 * n, device="cpu"))
    long = bfft.rotary_table(9, 24, axes=axes, axis_order=order, spectrum="axial", scaling="ntk", factor=4.0, device="cpu")
    for a, n in enumerate(axes):
        assert torch.equal(long[:, of == a], bfft.rotary_table(9, 2 * n, scaling="ntk", factor=4.0, device="cpu"))


def test_descriptor_matches_the_header():
    text = open(_build.INCLUDE + "/bfft.h").read()
    body = text.split("typedef struct bfft_axes_desc {")[1].split("}")[0]
    body = "".join(line.split("/*")[0] for line in body.splitlines())
    assert sum(len(part.split(",")) for part in body.split(";") if part.strip()) == 3


def test_call_checks(lib):
    pairs = (ctypes.c_uint8 * 16)(*[0, 1] * 8)

    def axes(of=ctypes.addressof(pairs), n=2, stride=3):
        return struct.pack("Qqq", of, n, stride)

    c, s = cache_desc(), seq_desc()
    given = bytearray(append_desc())
    given[32:40] = struct.pack("Q", A)                         # positions
    given = bytes(given)
    for desc, status in ((axes(of=0), _lib.ERR_VALUE), (axes(n=0), _lib.ERR_VALUE), (axes(n=5), _lib.ERR_VALUE),
                         (axes(n=1), _lib.ERR_VALUE), (None, _lib.ERR_VALUE)):
        assert lib.bfft_rotate_axes(rotate_desc(), desc, A, A, A, A, None) == status
        assert lib.bfft_cache_append_axes(c, s, given, desc, None) == status
        assert _lib.last_error()
    assert lib.bfft_cache_append_axes(c, s, append_desc(), axes(), None) == _lib.ERR_VALUE          # no positions
    assert lib.bfft_cache_append_axes(c, s, append_desc(table=0), axes(), None) == _lib.ERR_VALUE
    assert lib.bfft_rotate_axes(rotate_desc(dim=31), axes(), A, A, A, A, None) == _lib.ERR_SHAPE
    assert lib.bfft_rotate_axes(rotate_desc(tokens=0), axes(), A, A, A, A, None) == _lib.OK
    assert lib.bfft_cache_append_axes(c, seq_desc(tokens=0), given, axes(), None) == _lib.OK

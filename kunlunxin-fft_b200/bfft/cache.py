"""Rotation by position, and attention over a paged 8-bit cache.

No counterpart in the reference, and no transform is part of it; what it shares with
them is the product by unit roots from a table made in float64.  An attention layer's
queries and keys are rotated by unit roots of their positions, the keys and values of
past tokens are kept in 8 bits, and new tokens attend to them.

* ``rotary_table`` / ``rotate_positions``: the rotation, forward and inverse;
  differentiable (the gradient is rotated by the conjugate roots).  Positions of
  several axes (time, height, width) turn each pair by its axis's.
* ``paged_cache`` / ``append_rotated``: pages of 16..128 tokens hold int8 or e4m3
  codes with one scale per page and kv head; new tokens are rotated, quantised
  and written by one launch (two where few sequences append long runs).
* ``cache_attention``: causal, windowed or full attention of ragged rows (one
  token, a few drafted ones, or a prompt's chunk per sequence) over the cache;
  first tokens that a window does not hide, prefixes that sequences share.
* ``read_cache``: the values that the cache stands for.

Ragged rows: sequence ``s`` owns rows ``starts[s] .. starts[s + 1]`` of a call's
tensors and its token ``i`` lies in page ``block_table[s, i // page]``.  These
tables are int32 tensors on the device and are read there: no call waits for the
device, and ``starts[-1]`` has to be the number of rows.

Calls enqueue on the current stream of the tensors' device.  Bad arguments raise
before any launch: TypeError for a non-tensor or a wrong dtype, ValueError for
shapes, strides and devices.  Only ``x`` of ``rotate_positions`` has a gradient: where
gradients are enabled, the other calls and arguments refuse tensors that require one
(ValueError).  There is no forward-mode gradient.  An ``out`` may be the input itself,
but not overlap it otherwise.  The checks and the calls themselves are in
``csrc/bfft_torch.cpp``.
"""
from __future__ import annotations

import ctypes
import functools
import importlib.machinery
import importlib.util
import math
import os
import threading
from typing import NamedTuple

import torch

from . import _build, _lib

TYPE_IDS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
CODE_DTYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LAYOUT_IDS = {"half": 0, "interleaved": 1}
SCALINGS = ("none", "linear", "ntk", "banded")
AXIS_ORDERS = ("blocks", "cyclic")
SPECTRA = ("shared", "axial")
PAGE_SIZES = (16, 32, 64, 128)

_native = None
_native_lock = threading.Lock()


def _load():
    """The torch binding, bound to libbfft.so (raises RuntimeError when it has not been built)."""
    global _native
    with _native_lock:
        if _native is None:
            path = _build.TORCH_LIB_PATH
            if not os.path.exists(path):
                raise RuntimeError(f"bfft_torch.so not found at {path}; build it with bfft._build.build() "
                                   "-- there is no fallback")
            if not _build.torch_module_fits():
                raise RuntimeError(f"{path} was built for another torch or Python; build it again with bfft._build.build()")
            lib = _lib.load()
            loader = importlib.machinery.ExtensionFileLoader("bfft_torch", path)
            module = importlib.util.module_from_spec(importlib.util.spec_from_loader("bfft_torch", loader))
            loader.exec_module(module)
            module.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value
                          for name in ("bfft_rotate_positions", "bfft_cache_append", "bfft_cache_read",
                                       "bfft_cache_attention_workspace", "bfft_cache_attention", "bfft_last_error",
                                       "bfft_rotate_axes", "bfft_cache_append_axes", "bfft_cache_attention_span_workspace",
                                       "bfft_cache_attention_span")))
            _native = module
    return _native


class PagedCache(NamedTuple):
    """Codes (pages, kv_heads, page, dim) and scales (pages, kv_heads): a token's
    key is ``k[page, head, slot] * k_scale[page, head]``."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def paged_cache(pages: int, kv_heads: int, page: int, dim: int, *, code: str = "int8", device="cuda") -> PagedCache:
    """An empty cache of ``pages`` pages of ``page`` tokens."""
    if code not in CODE_DTYPES:
        raise ValueError(f"code must be one of {sorted(CODE_DTYPES)}, got {code!r}")
    if page not in PAGE_SIZES:
        raise ValueError(f"page must be one of {PAGE_SIZES}, got {page!r}")
    if pages < 1 or kv_heads < 1 or dim < 16 or dim > 256 or dim % 16:
        raise ValueError(f"bad cache shape: {pages} pages, {kv_heads} heads of {dim} (a multiple of 16 up to 256)")
    shape = (pages, kv_heads, page, dim)
    return PagedCache(*(torch.zeros(shape, dtype=torch.uint8, device=device).view(CODE_DTYPES[code]) for _ in "kv"),
                      *(torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in "kv"))


def _axes_map(axes, axis_order) -> tuple[int, ...]:
    """The axis of each pair."""
    axes = tuple(axes)
    if axis_order not in AXIS_ORDERS:
        raise ValueError(f"axis_order must be one of {AXIS_ORDERS}, got {axis_order!r}")
    if not 1 <= len(axes) <= 4 or any(type(n) is not int or n < 0 for n in axes) or not 1 <= sum(axes) <= 256:
        raise ValueError(f"axes must be the pairs of each of 1 to 4 axes, up to 256 together, got {axes}")
    if axis_order == "blocks":
        return tuple(a for a, n in enumerate(axes) for _ in range(n))
    return tuple(a for i in range(max(axes)) for a, n in enumerate(axes) if i < n)


@functools.lru_cache(maxsize=64)
def _axes_bytes(axes, axis_order) -> bytes:
    """The number of axes, then the axis of each pair (a function of the numbers alone: made once for a model)."""
    return bytes((len(axes), *_axes_map(axes, axis_order)))


def _axes(axes, axis_order):
    axes = axes if type(axes) is tuple else tuple(axes)
    for n in axes:  # (4.0, 6) and (True, 6) would be found as (4, 6) and (1, 6)
        if type(n) is not int:
            raise ValueError(f"axes must be integers, got {axes}")
    return _axes_bytes(axes, axis_order)


def _frequencies(rotated, base, scaling, factor, original, low_turns, high_turns, device):
    if scaling == "ntk" and rotated > 2:
        base = base * factor ** (rotated / (rotated - 2))
    w = base ** (-torch.arange(0, rotated, 2, dtype=torch.float64, device=device) / rotated)
    if scaling == "linear":
        w = w / factor
    elif scaling == "banded":
        keep = ((original * w / (2 * math.pi) - low_turns) / (high_turns - low_turns)).clamp(0.0, 1.0)
        w = w * keep + w / factor * (1.0 - keep)
    return w


def rotary_table(positions: int, rotated: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original: int | None = None, low_turns: float = 1.0, high_turns: float = 32.0,
                 amplitude: float = 1.0, axes=None, axis_order: str = "blocks", spectrum: str = "shared",
                 device="cuda") -> torch.Tensor:
    """(positions, rotated / 2, 2) float32: amplitude * (cos, sin) of p * w_j with
    w_j = base^(-2 j / rotated), made in float64 and rounded once.

    ``scaling`` stretches the frequencies for contexts ``factor`` times longer than
    those trained on: "linear" divides them all; "ntk" raises the base to
    base * factor^(rotated / (rotated - 2)), so that the slowest is divided by the
    factor and the fastest stays; "banded" divides those that make fewer than
    ``low_turns`` turns over the ``original`` context, keeps those that make more
    than ``high_turns`` and blends between them linearly in their turns (a blend that
    is linear in the index j, as some models are trained with, gives other
    frequencies: make that table yourself).

    A table for positions of several axes (``axes`` and ``axis_order`` as in
    ``rotate_positions``) has the same columns with ``spectrum`` "shared": the axes
    take the frequencies where their pairs lie.  "axial" gives each axis a spectrum of
    its own: pair i of an axis's n has base^(-i / n) (and the scaling of a rotated part
    of 2 n elements)."""
    if positions < 1 or rotated < 2 or rotated % 2:
        raise ValueError(f"need positions >= 1 and an even rotated part, got {positions} and {rotated}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not factor >= 1.0 or not base > 0.0:
        raise ValueError(f"need factor >= 1 and base > 0, got {factor} and {base}")
    if scaling == "banded" and (original is None or original < 1 or not high_turns > low_turns):
        raise ValueError("banded scaling needs the original context length and low_turns < high_turns")
    if spectrum not in SPECTRA:
        raise ValueError(f"spectrum must be one of {SPECTRA}, got {spectrum!r}")
    how = (base, scaling, factor, original, low_turns, high_turns, device)
    if axes is None:
        if spectrum != "shared":
            raise ValueError("an axial spectrum needs axes")
        w = _frequencies(rotated, *how)
    else:
        axis_of = _axes_map(axes, axis_order)
        if 2 * len(axis_of) != rotated:
            raise ValueError(f"axes have {len(axis_of)} pairs, a rotated part of {rotated} has {rotated // 2}")
        w = _frequencies(rotated, *how)
        if spectrum == "axial":
            of = torch.tensor(axis_of, device=device)
            for a in set(axis_of):
                w[of == a] = _frequencies(2 * axis_of.count(a), *how)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * w
    return (torch.stack((angle.cos(), angle.sin()), -1) * amplitude).float()


# ------------------------------------------------------------------------------- rotation

def _layout(layout: str) -> int:
    kind = LAYOUT_IDS.get(layout)
    if kind is None:
        raise ValueError(f"layout must be one of {sorted(LAYOUT_IDS)}, got {layout!r}")
    return kind


def rotate_positions(x, positions, table, *, layout: str = "half", transform_direction: str = "forward", axes=None,
                     axis_order: str = "blocks", out=None):
    """x with the first ``2 * table.shape[1]`` elements of each head rotated by its
    token's position; the other elements pass through.

    x: (tokens, heads, dim) or (batch, tokens, heads, dim), float32, float16 or
    bfloat16, any strides with adjacent elements (heads before tokens: pass the
    transposed view).  positions: int32 or int64, (tokens,) or (batch, tokens); one
    outside the table makes its token's rotated part NaN.  layout "half" pairs
    elements j and j + rotated / 2, "interleaved" 2 j and 2 j + 1.
    transform_direction "inverse" rotates back (conjugate roots; with an amplitude m
    in the table it is m^2 times the inverse, the adjoint).  ``out`` may be x.

    ``axes``: tokens have positions on up to four axes (time, height, width of a
    patch), and each pair belongs to one: ``axes=(16, 24, 24)`` gives the first 16
    pairs to axis 0, the next 24 to axis 1 and so on with axis_order "blocks", and
    deals them out in turn with "cyclic" (0, 1, 2, 0, 1, 2, ..., an axis that has its
    share drops out).  positions are then (axes, tokens) or (axes, batch, tokens), pair
    j's root is row ``positions[axis(j)]``, column j of the table, and a position
    outside the table makes the pairs of its axis NaN."""
    direction = _lib.TRANSFORM_DIRECTION_IDS.get(transform_direction)
    if direction is None:
        raise ValueError(f"transform_direction must be one of {sorted(_lib.TRANSFORM_DIRECTION_IDS)}, "
                         f"got {transform_direction!r}")
    return (_native or _load()).rotate(x, positions, table, _layout(layout), direction, out,
                                       None if axes is None else _axes(axes, axis_order))


# ------------------------------------------------------------------------------- cache

def append_rotated(cache, k, v, block_table, held, starts, table=None, *, layout: str = "half", positions=None, axes=None,
                   axis_order: str = "blocks", q=None):
    """Append each sequence's new rows behind the ``held[s]`` tokens it has.

    k, v: (tokens, kv_heads, dim), float32, float16 or bfloat16.  Keys are rotated
    by ``table`` (None: as they are) at their place in the sequence, or at
    ``positions`` ((tokens,) int32 or int64); codes and scales are written to
    ``cache``.  A block's scale is the largest magnitude it has held over 127
    (int8) or 448 (e4m3); where new rows make it grow, the block's earlier codes
    are rounded again.  A sequence's first token of a page starts its blocks anew.
    Two sequences must not append to one page.  Rows whose page is not in the table
    are dropped.

    ``axes`` and ``axis_order``: positions of several axes, as in ``rotate_positions``;
    the table and ``positions``, (axes, tokens), have to be given.

    q: (tokens, q_heads, dim) of k's type; its rotated rows are returned (else None).
    ``cache_attention`` takes them in float16 or bfloat16."""
    return (_native or _load()).append(cache, k, v, block_table, held, starts, table, _layout(layout), positions, q,
                                       None if axes is None else _axes(axes, axis_order))


def read_cache(cache, block_table, first, starts, tokens: int, *, dtype=torch.bfloat16):
    """(k, v), each (tokens, kv_heads, dim) of ``dtype``: row ``starts[s] + i`` is what
    the cache holds for token ``first[s] + i`` of sequence s (NaN where the table has
    no page for it)."""
    kind = TYPE_IDS.get(dtype)
    if kind is None:
        raise TypeError(f"dtype must be one of {[str(d) for d in TYPE_IDS]}, got {dtype}")
    return (_native or _load()).read(cache, block_table, first, starts, tokens, kind)


def cache_attention(q, cache, block_table, lens, starts, *, softmax_scale: float | None = None, causal: bool = True,
                    window: int = 0, sinks: int = 0, shared=None, groups=None, return_lse: bool = False, out=None):
    """softmax(softmax_scale q k^T) v of ragged query rows over the cache.

    q: (tokens, q_heads, dim), float16 or bfloat16, q_heads a multiple of the
    cache's kv heads (query head h reads kv head h // (q_heads / kv_heads)).
    lens[s]: tokens that sequence s has in the cache, those of its new rows among
    them.  Row i of a sequence's n rows is its token lens[s] - n + i; causal rows
    see the tokens up to their own, and with ``window`` > 0 only the last ``window``
    of those (rows that are not causal: from there to the sequence's end).  A row that
    sees no token gets zeros and a log-sum-exp of -inf.

    ``sinks``: the window does not hide the first ``sinks`` tokens of a sequence.

    ``shared``: sequences that begin with the same tokens and name the same pages for
    them.  Sequences ``groups[g] .. groups[g + 1]`` (int32, (groups + 1,), ascending; None:
    all are one group) share their first ``shared[g]`` tokens (int32, (groups,)): the whole
    pages among these are read once for the group, from the block table's row of its first
    sequence.  The results are those of a call without, but for roundings.  Sequences in
    no group share nothing.  The call goes without over 128 rows a kv head (query tokens
    times heads) of a sequence, where the prefixes would be under 24 MB to read again, were
    they as long as the table is wide, and where the workspace would pass 512 MB.  It knows
    the table's width only: where most tokens are the sequences' own, or with one or two kv
    heads and short prefixes, it can be slower than without (32 sequences over 2048 + 2000
    tokens 71 us for 60, 128 of one kv head over 1024 + 100 37 for 21): leave `shared` out there.

    With ``shared``, and with ``sinks`` beside a window, tables are up to 2^30 tokens wide.

    The weights, times their block's value scale, are rounded to float16 before they
    meet the codes, with a row's largest near float16's top: to 2^-11 down to 2^-24 of
    the largest (few rows: 2^-28), to nothing under 2^-34 (2^-38).

    Returns out (tokens, q_heads, dim), with ``return_lse`` also the rows' log-sum-exp
    (tokens, q_heads) float32."""
    return (_native or _load()).attention(q, cache, block_table, lens, starts, softmax_scale, causal, window, return_lse,
                                          out, sinks, shared, groups)

"""Rotation by position, and attention over a paged 8-bit cache.

No counterpart in the reference.  What an attention layer needs next to the
transforms: its queries and keys are rotated by unit roots of their positions
(the twiddle product, with a table made in float64), the keys and values of past
tokens are kept in 8 bits, and new tokens attend to them.

* ``rotary_table`` / ``rotate_positions``: the rotation, forward and inverse;
  differentiable (the gradient is rotated by the conjugate roots).
* ``paged_cache`` / ``append_rotated``: pages of 16..128 tokens hold int8 or e4m3
  codes with one scale per page and kv head; new tokens are rotated, quantised
  and written by one launch.
* ``cache_attention``: causal, windowed or full attention of ragged rows (one
  token, a few drafted ones, or a prompt's chunk per sequence) over the cache.
* ``read_cache``: the values that the cache stands for.

Ragged rows: sequence ``s`` owns rows ``starts[s] .. starts[s + 1]`` of a call's
tensors and its token ``i`` lies in page ``block_table[s, i // page]``.  These
tables are int32 tensors on the device and are read there: no call waits for the
device, and ``starts[-1]`` has to be the number of rows.

Calls enqueue on the current stream of the tensors' device.  Bad arguments raise
before any launch: TypeError for a non-tensor or a wrong dtype, ValueError for
shapes, strides and devices.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import NamedTuple

import torch

from . import _lib
from ._lib import TRANSFORM_DIRECTION_IDS

TYPE_IDS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
CODE_IDS = {torch.int8: 0, torch.float8_e4m3fn: 1}
CODE_DTYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LAYOUT_IDS = {"half": 0, "interleaved": 1}
SCALINGS = ("none", "linear", "ntk", "banded")
PAGE_SIZES = (16, 32, 64, 128)

# struct bfft_rotate_desc, bfft_cache_desc, ... of include/bfft.h: every field is 8 bytes wide
_ROTATE = struct.Struct("19q").pack
_CACHE = struct.Struct("4Q5q").pack
_SEQUENCES = struct.Struct("Qq2Q3q").pack
_APPEND = struct.Struct("6Q15q").pack
_ATTENTION = struct.Struct("3Q8qdQ2q").pack


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


def rotary_table(positions: int, rotated: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original: int | None = None, low_turns: float = 1.0, high_turns: float = 32.0,
                 amplitude: float = 1.0, device="cuda") -> torch.Tensor:
    """(positions, rotated / 2, 2) float32: amplitude * (cos, sin) of p * w_j with
    w_j = base^(-2 j / rotated), made in float64 and rounded once.

    ``scaling`` stretches the frequencies for contexts ``factor`` times longer than
    those trained on: "linear" divides them all; "ntk" raises the base to
    base * factor^(rotated / (rotated - 2)), so that the slowest is divided by the
    factor and the fastest stays; "banded" divides those that make fewer than
    ``low_turns`` turns over the ``original`` context, keeps those that make more
    than ``high_turns`` and blends between them by their turns."""
    if positions < 1 or rotated < 2 or rotated % 2:
        raise ValueError(f"need positions >= 1 and an even rotated part, got {positions} and {rotated}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not factor >= 1.0 or not base > 0.0:
        raise ValueError(f"need factor >= 1 and base > 0, got {factor} and {base}")
    if scaling == "ntk" and rotated > 2:
        base = base * factor ** (rotated / (rotated - 2))
    w = base ** (-torch.arange(0, rotated, 2, dtype=torch.float64, device=device) / rotated)
    if scaling == "linear":
        w = w / factor
    elif scaling == "banded":
        if original is None or original < 1 or not high_turns > low_turns:
            raise ValueError("banded scaling needs the original context length and low_turns < high_turns")
        keep = ((original * w / (2 * math.pi) - low_turns) / (high_turns - low_turns)).clamp(0.0, 1.0)
        w = w * keep + w / factor * (1.0 - keep)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * w
    return (torch.stack((angle.cos(), angle.sin()), -1) * amplitude).float()


# ------------------------------------------------------------------------------- checks

def _tensor(x, name: str, dtypes, device: int | None = None) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(x).__name__}")
    if x.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {[str(d) for d in dtypes]}, got {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device, got {x.device}")
    if device is not None and x.get_device() != device:
        raise ValueError(f"{name} is on {x.device}, not on device {device} with the other tensors")


def _rows(x, name: str, dtypes, tokens: int | None, dim: int | None, device: int | None) -> tuple:
    """Checks (tokens, heads, dim) rows with adjacent elements; their strides."""
    _tensor(x, name, dtypes, device)
    shape = x.shape
    if len(shape) != 3 or (tokens is not None and shape[0] != tokens) or (dim is not None and shape[2] != dim):
        raise ValueError(f"{name} must be ({tokens or 'tokens'}, heads, {dim or 'dim'}), got {tuple(shape)}")
    stride = x.stride()
    if stride[2] != 1 and shape[2] > 1:
        raise ValueError(f"{name} must have adjacent elements in its last dimension, got strides {stride}")
    return stride


def _table(table, rotated_most: int, device: int) -> int:
    _tensor(table, "table", (torch.float32,), device)
    if table.dim() != 3 or table.shape[2] != 2 or not table.is_contiguous():
        raise ValueError(f"table must be a contiguous (positions, rotated / 2, 2) tensor, got {tuple(table.shape)}")
    rotated = 2 * table.shape[1]
    if not 2 <= rotated <= rotated_most:
        raise ValueError(f"table rotates {rotated} elements of heads of {rotated_most}")
    return rotated


def _layout(layout: str) -> int:
    if layout not in LAYOUT_IDS:
        raise ValueError(f"layout must be one of {sorted(LAYOUT_IDS)}, got {layout!r}")
    return LAYOUT_IDS[layout]


_INTS = (torch.int32, torch.int64)
_INT32 = (torch.int32,)
_FLOAT = (torch.float32,)


def _cache_desc(cache, device: int | None):
    """Packed bfft_cache_desc, (kv_heads, page, dim), device."""
    if not isinstance(cache, (tuple, list)) or len(cache) != 4:
        raise TypeError("cache must be a PagedCache: (k, v, k_scale, v_scale)")
    k, v, ks, vs = cache
    _tensor(k, "cache k", CODE_IDS, device)
    device = k.get_device()
    _tensor(v, "cache v", (k.dtype,), device)
    _tensor(ks, "cache k_scale", _FLOAT, device)
    _tensor(vs, "cache v_scale", _FLOAT, device)
    shape = k.shape
    if len(shape) != 4 or v.shape != shape:
        raise ValueError(f"cache codes must both be (pages, kv_heads, page, dim), got {tuple(shape)} and {tuple(v.shape)}")
    if ks.shape != shape[:2] or vs.shape != shape[:2]:
        raise ValueError(f"cache scales must be {tuple(shape[:2])}, got {tuple(ks.shape)} and {tuple(vs.shape)}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("cache tensors must be contiguous")
    pages, heads, page, dim = shape
    return (_CACHE(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, heads, page, dim,
                   CODE_IDS[k.dtype]), heads, page, dim, device)


def _sequence_desc(block_table, lens, starts, tokens: int, device: int, lens_name: str) -> bytes:
    _tensor(block_table, "block_table", _INT32, device)
    _tensor(lens, lens_name, _INT32, device)
    _tensor(starts, "starts", _INT32, device)
    shape = block_table.shape
    if len(shape) != 2 or shape[0] < 1 or shape[1] < 1 or (block_table.stride(1) != 1 and shape[1] > 1):
        raise ValueError(f"block_table must be (sequences, pages) with adjacent pages, got {tuple(shape)}")
    if lens.shape != shape[:1] or not lens.is_contiguous():
        raise ValueError(f"{lens_name} must be contiguous ({shape[0]},), got {tuple(lens.shape)}")
    if starts.dim() != 1 or starts.shape[0] != shape[0] + 1 or not starts.is_contiguous():
        raise ValueError(f"starts must be contiguous ({shape[0] + 1},), got {tuple(starts.shape)}")
    return _SEQUENCES(block_table.data_ptr(), block_table.stride(0), lens.data_ptr(), starts.data_ptr(), shape[0],
                      shape[1], tokens)


def _stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# ------------------------------------------------------------------------------- rotation

def _rotate(x, positions, table, layout: int, direction: int, out):
    _tensor(x, "x", TYPE_IDS)
    device = x.get_device()
    shape = x.shape
    if len(shape) not in (3, 4):
        raise ValueError(f"x must be (tokens, heads, dim) or (batch, tokens, heads, dim), got {tuple(shape)}")
    dim, heads, tokens = shape[-1], shape[-2], shape[-3]
    batch = shape[0] if len(shape) == 4 else 1
    rotated = _table(table, dim, device)
    xs = x.stride()
    if xs[-1] != 1:
        raise ValueError(f"x must have adjacent elements in its last dimension, got strides {xs}")
    _tensor(positions, "positions", _INTS, device)
    pshape, ps = positions.shape, positions.stride()
    if pshape == (tokens,):
        pos = (0, ps[0])
    elif len(shape) == 4 and pshape == (batch, tokens):
        pos = ps
    else:
        raise ValueError(f"positions must be ({tokens},){f' or ({batch}, {tokens})' if len(shape) == 4 else ''}, "
                         f"got {tuple(pshape)}")
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
    else:
        _tensor(out, "out", (x.dtype,), device)
        if out.shape != shape or out.stride(-1) != 1:
            raise ValueError(f"out must be {tuple(shape)} with adjacent elements, got {tuple(out.shape)}")
    if not out.numel():
        return out
    ys = out.stride()
    if len(shape) == 3:
        xs, ys = (0, *xs), (0, *ys)
    desc = _ROTATE(batch, tokens, heads, dim, rotated, xs[0], xs[1], xs[2], ys[0], ys[1], ys[2], pos[0], pos[1],
                   table.shape[0], TYPE_IDS[x.dtype], layout, direction, positions.dtype is torch.int64, device)
    status = _lib.load().bfft_rotate_positions(desc, x.data_ptr(), positions.data_ptr(), table.data_ptr(),
                                               out.data_ptr(), _stream(device))
    if status:
        _lib.check(status, "rotate_positions")
    return out


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, table, layout, direction):
        ctx.save_for_backward(positions, table)
        ctx.knobs = layout, direction
        return _rotate(x, positions, table, layout, direction, None)

    @staticmethod
    def backward(ctx, dy):
        positions, table = ctx.saved_tensors
        layout, direction = ctx.knobs
        if dy.stride(-1) != 1:
            dy = dy.contiguous()
        return _Rotate.apply(dy, positions, table, layout, 1 - direction), None, None, None, None


def rotate_positions(x, positions, table, *, layout: str = "half", transform_direction: str = "forward", out=None):
    """x with the first ``2 * table.shape[1]`` elements of each head rotated by its
    token's position; the other elements pass through.

    x: (tokens, heads, dim) or (batch, tokens, heads, dim), float32, float16 or
    bfloat16, any strides with adjacent elements (heads before tokens: pass the
    transposed view).  positions: int32 or int64, (tokens,) or (batch, tokens); one
    outside the table makes its token's rotated part NaN.  layout "half" pairs
    elements j and j + rotated / 2, "interleaved" 2 j and 2 j + 1.
    transform_direction "inverse" rotates back (conjugate roots; with an amplitude m
    in the table it is m^2 times the inverse, the adjoint).  ``out`` may be x."""
    kind = _layout(layout)
    if transform_direction not in TRANSFORM_DIRECTION_IDS:
        raise ValueError(f"transform_direction must be one of {sorted(TRANSFORM_DIRECTION_IDS)}, "
                         f"got {transform_direction!r}")
    direction = TRANSFORM_DIRECTION_IDS[transform_direction]
    if isinstance(x, torch.Tensor) and x.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("out cannot be given where x requires a gradient")
        return _Rotate.apply(x, positions, table, kind, direction)
    return _rotate(x, positions, table, kind, direction, out)


# ------------------------------------------------------------------------------- cache

def append_rotated(cache, k, v, block_table, held, starts, table=None, *, layout: str = "half", positions=None, q=None):
    """Append each sequence's new rows behind the ``held[s]`` tokens it has.

    k, v: (tokens, kv_heads, dim), float32, float16 or bfloat16.  Keys are rotated
    by ``table`` (None: as they are) at their place in the sequence, or at
    ``positions`` ((tokens,) int32 or int64); codes and scales are written to
    ``cache``.  A block's scale is the largest magnitude it has held over 127
    (int8) or 448 (e4m3); where new rows make it grow, the block's earlier codes
    are rounded again.  A sequence's first token of a page starts its blocks anew.
    Two sequences must not append to one page.  Rows whose page is not in the table
    are dropped.

    q: (tokens, q_heads, dim) of k's type; its rotated rows are returned (else None)."""
    desc, heads, _, dim, device = _cache_desc(cache, None)
    kt, kh, _ = _rows(k, "k", TYPE_IDS, None, dim, device)
    kind, tokens = k.dtype, k.shape[0]
    vt, vh, _ = _rows(v, "v", (kind,), tokens, dim, device)
    if k.shape[1] != heads or v.shape[1] != heads:
        raise ValueError(f"k and v must have the cache's {heads} heads, got {k.shape[1]} and {v.shape[1]}")
    seqs = _sequence_desc(block_table, held, starts, tokens, device, "held")
    rotated = _table(table, dim, device) if table is not None else 0
    pos64 = 0
    if positions is not None:
        _tensor(positions, "positions", _INTS, device)
        if positions.shape != (tokens,) or not positions.is_contiguous():
            raise ValueError(f"positions must be contiguous ({tokens},), got {tuple(positions.shape)}")
        pos64 = int(positions.dtype is torch.int64)
    out, qt, qh, ot, oh, q_heads = None, 0, 0, 0, 0, 0
    if q is not None:
        qt, qh, _ = _rows(q, "q", (kind,), tokens, dim, device)
        q_heads = q.shape[1]
        out = torch.empty(q.shape, dtype=kind, device=q.device)
        ot, oh, _ = out.stride()
    if tokens == 0:
        return out
    work = _APPEND(k.data_ptr(), v.data_ptr(), q.data_ptr() if q is not None else 0,
                   out.data_ptr() if out is not None else 0, positions.data_ptr() if positions is not None else 0,
                   table.data_ptr() if table is not None else 0, kt, kh, vt, vh, qt, qh, ot, oh,
                   table.shape[0] if table is not None else 0, rotated, q_heads, TYPE_IDS[kind], _layout(layout), pos64,
                   device)
    status = _lib.load().bfft_cache_append(desc, seqs, work, _stream(device))
    if status:
        _lib.check(status, "append_rotated")
    return out


def read_cache(cache, block_table, first, starts, tokens: int, *, dtype=torch.bfloat16):
    """(k, v), each (tokens, kv_heads, dim) of ``dtype``: row ``starts[s] + i`` is what
    the cache holds for token ``first[s] + i`` of sequence s (NaN where the table has
    no page for it)."""
    desc, heads, _, dim, device = _cache_desc(cache, None)
    if dtype not in TYPE_IDS:
        raise TypeError(f"dtype must be one of {[str(d) for d in TYPE_IDS]}, got {dtype}")
    if not isinstance(tokens, int) or tokens < 0:
        raise ValueError(f"tokens must be a row count, got {tokens!r}")
    seqs = _sequence_desc(block_table, first, starts, tokens, device, "first")
    k, v = torch.empty((2, tokens, heads, dim), dtype=dtype, device=cache[0].device)
    status = _lib.load().bfft_cache_read(desc, seqs, TYPE_IDS[dtype], k.data_ptr(), v.data_ptr(), device,
                                         _stream(device))
    if status:
        _lib.check(status, "read_cache")
    return k, v


_HALF = (torch.bfloat16, torch.float16)
_WORKSPACE: dict = {}  # bytes of workspace by the call's sizes


def cache_attention(q, cache, block_table, lens, starts, *, softmax_scale: float | None = None, causal: bool = True,
                    window: int = 0, return_lse: bool = False, out=None):
    """softmax(softmax_scale q k^T) v of ragged query rows over the cache.

    q: (tokens, q_heads, dim), float16 or bfloat16, q_heads a multiple of the
    cache's kv heads (query head h reads kv head h // (q_heads / kv_heads)).
    lens[s]: tokens that sequence s has in the cache, those of its new rows among
    them.  Row i of a sequence's n rows is its token lens[s] - n + i; causal rows
    see the tokens up to their own, and with ``window`` > 0 only the last ``window``
    of those.  A row that sees no token gets zeros and a log-sum-exp of -inf.

    Returns out (tokens, q_heads, dim), with ``return_lse`` also the rows' log-sum-exp
    (tokens, q_heads) float32."""
    desc, heads, page, dim, device = _cache_desc(cache, None)
    qt, qh, _ = _rows(q, "q", _HALF, None, dim, device)
    tokens, q_heads = q.shape[0], q.shape[1]
    if q_heads < 1 or q_heads % heads:
        raise ValueError(f"{q_heads} query heads are no multiple of the cache's {heads}")
    if not isinstance(window, int) or window < 0:
        raise ValueError(f"window must be a token count, got {window!r}")
    seqs = _sequence_desc(block_table, lens, starts, tokens, device, "lens")
    scale = dim ** -0.5 if softmax_scale is None else float(softmax_scale)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ot, oh, _ = _rows(out, "out", (q.dtype,), tokens, dim, device)
    if out.shape != q.shape:
        raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    lse = torch.empty((tokens, q_heads), dtype=torch.float32, device=q.device) if return_lse else None
    if tokens:
        lib = _lib.load()

        def work(ptr, size):
            return _ATTENTION(q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, qt, qh, ot, oh, q_heads,
                              TYPE_IDS[q.dtype], bool(causal), window, scale, ptr, size, device)

        key = (device, tokens, q_heads, heads, page, dim, block_table.shape, bool(causal), window)
        size = _WORKSPACE.get(key)
        if size is None:
            n = ctypes.c_size_t()
            _lib.check(lib.bfft_cache_attention_workspace(desc, seqs, work(0, 0), ctypes.byref(n)), "cache_attention")
            if len(_WORKSPACE) > 4096:
                _WORKSPACE.clear()
            size = _WORKSPACE[key] = int(n.value)
        scratch = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        status = lib.bfft_cache_attention(desc, seqs, work(scratch.data_ptr() if size else 0, size), _stream(device))
        if status:
            _lib.check(status, "cache_attention")
    return (out, lse) if return_lse else out

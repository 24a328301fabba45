"""Limits of the position and cache calls that the host decides, without a GPU."""
import ctypes
import os
import subprocess

import pytest

from bfft import _build, _lib, cache
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


# ------------------------------------------------------------------------------- the two libraries' builds

class Compilers:
    """Stands in for the compilers: nvcc writes its output, g++ does or fails."""

    def __init__(self, monkeypatch, tmp_path, host_compiler=True):
        self.host_compiler, self.ran = host_compiler, []
        for name in ("LIB_PATH", "META_PATH", "TORCH_LIB_PATH", "TORCH_META_PATH"):
            monkeypatch.setattr(_build, name, str(tmp_path / os.path.basename(getattr(_build, name))))
        monkeypatch.setattr(_build, "LIB_DIR", str(tmp_path))
        monkeypatch.setattr(_build.subprocess, "run", self.run)

    def run(self, cmd, check=False, **kw):
        if "--version" in cmd:
            return subprocess.CompletedProcess(cmd, 0, stdout="release 1.0, V1.0.1", stderr="")
        kind = "binding" if _build.TORCH_SRC in cmd else "library"
        self.ran.append(kind)
        if kind == "binding" and not self.host_compiler:
            raise subprocess.CalledProcessError(1, cmd)
        with open(cmd[cmd.index("-o") + 1], "wb"):
            return subprocess.CompletedProcess(cmd, 0)


def test_library_is_complete_where_the_binding_cannot_be_built(monkeypatch, tmp_path):
    c = Compilers(monkeypatch, tmp_path, host_compiler=False)
    with pytest.warns(UserWarning, match="bfft_torch"):
        assert _build.build(verbose=False) == _build.LIB_PATH
    assert c.ran == ["library", "binding"] and _build.up_to_date()
    assert _build.build_meta()["source_hash"] == _build.source_hash()
    assert not os.path.exists(_build.TORCH_LIB_PATH) and not _build.torch_module_up_to_date()
    with pytest.raises(subprocess.CalledProcessError):
        _build.build_torch_module(verbose=False)
    monkeypatch.setattr(cache, "_native", None)
    with pytest.raises(RuntimeError, match="not found"):
        cache._load()
    c.host_compiler, c.ran = True, []
    _build.build(verbose=False)                               # only what is missing
    assert c.ran == ["binding"] and _build.torch_module_up_to_date()
    _build.build(verbose=False)
    assert c.ran == ["binding"]


def test_binding_of_another_torch_is_built_again(monkeypatch, tmp_path):
    c = Compilers(monkeypatch, tmp_path)
    _build.build(verbose=False)
    assert c.ran == ["library", "binding"]
    now = _build.torch_target()
    monkeypatch.setattr(_build, "torch_target", lambda: {**now, "torch": "9.9.9"})
    assert _build.up_to_date() and not _build.torch_module_up_to_date()
    monkeypatch.setattr(cache, "_native", None)
    with pytest.raises(RuntimeError, match="another torch"):
        cache._load()
    _build.build(verbose=False)
    assert c.ran == ["library", "binding", "binding"] and _build.torch_module_up_to_date()


def test_binding_of_other_sources_does_not_stay(monkeypatch, tmp_path):
    """Its descriptors may not be the library's: where it cannot be built again, it is gone."""
    c = Compilers(monkeypatch, tmp_path)
    _build.build(verbose=False)
    other = tmp_path / "bfft_torch.cpp"
    other.write_text("// changed")
    monkeypatch.setattr(_build, "TORCH_SRC", str(other))
    assert _build.up_to_date() and not _build.torch_module_up_to_date()
    c.host_compiler = False
    with pytest.warns(UserWarning, match="bfft_torch"):
        _build.build(verbose=False)
    assert not os.path.exists(_build.TORCH_LIB_PATH)

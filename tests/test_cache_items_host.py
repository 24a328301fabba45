"""How the axis of a call with groups is cut into items, by the kernels' own functions compiled for the host."""
import os
import subprocess

import pytest

from bfft import _build

PROGRAM = r"""
#include <cstdio>

#include "bfft_attention.cuh"

// Reads target, unit, least, count and the units' row tiles and lengths; prints the tokens of an item and the items.
int main() {
    int target, unit, least, count;
    while (std::scanf("%d %d %d %d", &target, &unit, &least, &count) == 4) {
        bfft::ItemArgs x{};
        x.target = target;
        x.unit = unit;
        x.least = least;
        bfft::Unit* units = new bfft::Unit[count]();
        float total = 0.f;
        for (int i = 0; i < count; ++i) {
            if (std::scanf("%d %d", &units[i].tiles, &units[i].length) != 2) return 1;
            total += (float)units[i].tiles * (float)units[i].length;
        }
        const unsigned chunk = bfft::item_tokens(x, total);
        long long items = 0;
        for (int i = 0; i < count; ++i) items += (long long)units[i].tiles * bfft::pieces_of(units[i], chunk);
        std::printf("%u %lld\n", chunk, items);
        delete[] units;
    }
}
"""


@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    where = tmp_path_factory.mktemp("items")
    source, program = where / "items.cu", where / "items"
    source.write_text(PROGRAM)
    subprocess.run([_build.nvcc_path(), *_build.ARCH_FLAGS, "-std=c++17", "-I", _build.CSRC, "-o", str(program), str(source)],
                   check=True)

    def run(target, unit, least, units):
        text = f"{target} {unit} {least} {len(units)}\n" + "\n".join(f"{t} {n}" for t, n in units)
        out = subprocess.run([str(program)], input=text, capture_output=True, text=True, check=True).stdout.split()
        return int(out[0]), int(out[1])

    return run


WIDEST = (1 << 30) - 128  # tokens of the widest table


@pytest.mark.parametrize("target, unit, least", [(888, 32, 256), (148, 128, 512), (1, 32, 256), (18, 128, 512)])
@pytest.mark.parametrize("units", [
    [(1, 1)], [(1, 0)] * 50, [(1, WIDEST)], [(1, WIDEST)] * 1000, [(40, WIDEST), (1, 7)] * 300, [(3, 1_000_000_100)] * 700,
    [(1, 999_999_000)] * 700, [(2, 100 + i) for i in range(2000)], [(1 + i % 5, 1 << (i % 30)) for i in range(900)],
    [(1000, 131072 + i % 77) for i in range(300)], [(1, 300)] * 100000,
], ids=lambda u: f"{len(u)}x{u[0][1]}")
def test_every_item_has_a_block(cut, target, unit, least, units):
    """A launch has target + 2 + row tiles blocks a kv head: the items may not be more, whatever the lengths."""
    chunk, items = cut(target, unit, least, units)
    assert chunk % unit == 0 and chunk >= least
    assert sum(t for t, _ in units) <= items <= target + 2 + sum(t for t, _ in units)

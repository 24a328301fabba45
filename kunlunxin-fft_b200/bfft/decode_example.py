"""An attention layer that reads a prompt and then decodes token by token.

Shows the position and cache calls as they are used together: one rotation table,
one paged 8-bit cache, and per step

    q = append_rotated(cache, k, v, pages, held, starts, table, q=q)
    y = cache_attention(q, cache, pages, lens, starts)

for two sequences of different lengths, first with their whole prompts as rows,
then with one row each.  ``window`` and ``sinks`` make it a stream that sees its last
tokens and its first ones; with ``common`` tokens the prompts begin alike, and the
second user's block table names the first one's pages for them.  The result is compared
with float64 attention over the unquantised rows; the gradient of the rotation is
compared with its adjoint.

Run: ``python -m bfft.decode_example [--prompt N] [--steps N] [--code int8|e4m3]
[--window N] [--sinks N] [--common N]`` with the package directory on PYTHONPATH; prints
one JSON object.
"""
from __future__ import annotations

import argparse
import json

import torch

from .cache import append_rotated, cache_attention, paged_cache, read_cache, rotary_table, rotate_positions


def _exact(q, k, v, table, group: int, window: int, sinks: int):
    """Causal attention of one sequence's rows in float64: rows (tokens, heads, dim)."""
    where = torch.arange(q.shape[0], device=q.device)
    c, s = table[where].double().unsqueeze(1).unbind(-1)

    def turn(x):
        a, b = x.double().chunk(2, -1)
        return torch.cat((a * c - b * s, a * s + b * c), -1)

    z = torch.einsum("qhd,khd->hqk", turn(q), turn(k).repeat_interleave(group, 1)) * q.shape[-1] ** -0.5
    hidden = where > where[:, None]
    if window:
        hidden |= (where <= where[:, None] - window) & (where >= sinks)
    z = z.masked_fill(hidden, float("-inf"))
    return torch.einsum("hqk,khd->qhd", torch.softmax(z, -1), v.double().repeat_interleave(group, 1))


def run(prompt: int = 300, steps: int = 20, code: str = "int8", q_heads: int = 16, kv_heads: int = 4, dim: int = 128,
        page: int = 32, seed: int = 0, device="cuda", window: int = 0, sinks: int = 0, common: int = 0) -> dict:
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    prompts = [prompt, max(1, prompt // 3)]  # two users
    common = common // page * page  # whole pages are shared
    if not 0 <= common < min(prompts):
        raise ValueError(f"the common tokens must be fewer than the shorter prompt's {min(prompts)}, got {common}")
    total = [n + steps for n in prompts]
    table = rotary_table(max(total), dim, device=device)
    per = -(-max(total) // page)
    cache = paged_cache(2 * per, kv_heads, page, dim, code=code, device=device)
    pages = torch.randperm(2 * per, device=device, generator=g).to(torch.int32).view(2, per)
    rows = [[torch.randn(n, h, dim, device=device, generator=g).bfloat16() for h in (q_heads, kv_heads, kv_heads)]
            for n in total]
    for i in (0, 1, 2):
        rows[1][i][:common] = rows[0][i][:common]
    pages[1, :common // page] = pages[0, :common // page]

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=device)

    def step(held, new):
        """The rows [held, held + new) of both sequences through the layer."""
        q, k, v = (torch.cat([rows[s][i][held[s]:held[s] + new[s]] for s in (0, 1)]) for i in (0, 1, 2))
        starts = ints([0, new[0], new[0] + new[1]])
        q = append_rotated(cache, k, v, pages, ints(held), starts, table, q=q)
        y = cache_attention(q, cache, pages, ints([held[s] + new[s] for s in (0, 1)]), starts, window=window, sinks=sinks,
                            shared=ints([common]) if common else None)
        return y.split(new)

    first = [0, common]  # what the second user finds in the cache
    out = [[y] for y in step(first, [n - f for n, f in zip(prompts, first)])]
    held = list(prompts)
    for _ in range(steps):
        for s, y in enumerate(step(held, [1, 1])):
            out[s].append(y)
        held = [h + 1 for h in held]
    error = 0.0
    for s in (0, 1):
        want = _exact(*rows[s], table, q_heads // kv_heads, window, sinks)[first[s]:]
        error = max(error, float((torch.cat(out[s]).double() - want).norm() / want.norm()))

    # what the cache stands for, and the rotation's gradient
    _, values = read_cache(cache, pages[:1], ints([0]), ints([0, total[0]]), total[0])
    stored = float((values.double() - rows[0][2].double()).norm() / rows[0][2].double().norm())
    x = rows[0][0].float().requires_grad_(True)
    w = torch.randn(x.shape, device=device, generator=g)
    where = torch.arange(total[0], device=device)
    dx, = torch.autograd.grad(rotate_positions(x, where, table), x, w)
    back = rotate_positions(w, where, table, transform_direction="inverse")
    return {"code": code, "prompts": prompts, "steps": steps, "attention_rel_error": error, "value_rel_error": stored,
            "gradient_is_adjoint": bool(torch.equal(dx, back))}


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--prompt", type=int, default=300)
    p.add_argument("--steps", type=int, default=20)
    p.add_argument("--code", choices=("int8", "e4m3"), default="int8")
    for name in ("window", "sinks", "common"):
        p.add_argument(f"--{name}", type=int, default=0)
    a = p.parse_args()
    print(json.dumps(run(a.prompt, a.steps, a.code, window=a.window, sinks=a.sinks, common=a.common)))


if __name__ == "__main__":
    main()

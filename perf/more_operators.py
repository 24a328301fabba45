"""Cases of the position and cache operators' wider forms: rotation by positions of several axes
(time, height, width), appending with it, and attention over the paged 8-bit cache with first
tokens that stay visible beside a window and with prefixes that a group of sequences shares.

Each case is one pass through one of them, in its plain form (elementary torch operations in
32 bits) or through the library's entry points (``own``):

* ``turn``: ``bfft.rotate_positions`` with ``axes``, and its gradient where the case trains;
* ``write``: ``bfft.append_rotated`` with ``axes`` (rotate queries and keys, quantise keys and
  values into their pages) and ``bfft.read_cache`` (the values that the touched pages stand for);
* ``attend``: ``bfft.cache_attention`` with ``sinks`` or with ``shared`` and ``groups``, and the
  log-sum-exp of each row.

Head counts, page sizes and lengths are generic; the power-of-two lengths and batches are the
ones that the library's transforms are measured at.
"""
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_POSITIONS = 1 << 15  # rows of the rotation table


def _library():
    if "bfft" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "kunlunxin-fft_b200"))
    import bfft

    return bfft


# ------------------------------------------------------------------------------- cases

def listed():
    turn = {"op": "turn", "batch": 1, "dim": 128, "rotated": 128, "axes": "16,24,24", "order": "blocks",
            "spectrum": "shared", "layout": "half", "type": "bf16", "train": False, "high": 24, "wide": 32}
    write = {"op": "write", "q_heads": 32, "kv_heads": 8, "dim": 128, "rotated": 128, "axes": "16,24,24",
             "order": "blocks", "spectrum": "shared", "layout": "half", "type": "bf16", "code": "int8", "page": 64,
             "high": 24, "wide": 32}
    attend = {"op": "attend", "q_heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "code": "int8", "page": 64,
              "window": 0, "sinks": 0, "groups": 0, "prefix_lo": 0, "prefix_hi": 0, "empty": 0}
    return [
        # the queries of one new text token behind images: the smallest call, all latency
        {**turn, "name": "axes one token", "tokens": 1, "heads": 32, "high": 0},
        # a training step on video frames, forward and backward, axes dealt in turn over the pairs
        {**turn, "name": "axes video training", "batch": 2, "tokens": 8192, "heads": 32, "axes": "24,20,20",
         "order": "cyclic", "train": True},
        # an image encoder's odd patch count in full precision: two axes with a spectrum each, part of the head
        {**turn, "name": "axes image odd f32", "tokens": 4999, "heads": 12, "dim": 96, "rotated": 80, "axes": "20,20",
         "spectrum": "axial", "layout": "interleaved", "type": "f32", "train": True, "high": 70, "wide": 72},
        # a few users' next text tokens behind images
        {**write, "name": "write 8 tokens", "seqs": 8, "new_lo": 1, "new_hi": 1, "held_lo": 100, "held_hi": 4000,
         "high": 0, "mix": 1},
        # prompts with images, some continuing a cached prefix
        {**write, "name": "write image prompts", "seqs": 16, "new_lo": 65, "new_hi": 2048, "held_lo": 0,
         "held_hi": 1000, "mix": 2},
        # odd head count and width, part of the head, axes in turn, interleaved pairs
        {**write, "name": "write odd f16", "seqs": 7, "new_lo": 1, "new_hi": 333, "held_lo": 0, "held_hi": 77,
         "q_heads": 9, "kv_heads": 3, "dim": 96, "rotated": 48, "axes": "10,7,7", "order": "cyclic",
         "layout": "interleaved", "type": "f16", "code": "e4m3", "page": 32, "high": 9, "wide": 13, "mix": 3},
        # one user's next token of an endless stream: four first tokens and a window of a long cache
        {**attend, "name": "sinks decode one", "seqs": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 131001, "kv_hi": 131001,
         "window": 4096, "sinks": 4, "mix": 4},
        # a decoding batch of streams of ragged lengths, some shorter than the window
        {**attend, "name": "sinks decode 64", "seqs": 64, "q_lo": 1, "q_hi": 1, "kv_lo": 1024, "kv_hi": 32768,
         "window": 8192, "sinks": 16, "code": "e4m3", "mix": 5},
        # chunks of long prompts with a window: matrix products
        {**attend, "name": "sinks prompt chunks", "seqs": 2, "q_lo": 2048, "q_hi": 2048, "kv_lo": 8192,
         "kv_hi": 16384, "window": 4096, "sinks": 4, "mix": 6},
        # a few drafted tokens of five users behind one instruction text: small heads and pages, a user without tokens
        {**attend, "name": "shared small f16", "seqs": 5, "q_lo": 1, "q_hi": 4, "kv_lo": 5, "kv_hi": 333,
         "q_heads": 12, "kv_heads": 4, "dim": 64, "type": "f16", "code": "e4m3", "page": 16, "groups": 1,
         "prefix_lo": 2001, "prefix_hi": 2001, "empty": 1, "mix": 7},
        # a decoding batch that shares one long document
        {**attend, "name": "shared decode 64", "seqs": 64, "q_lo": 1, "q_hi": 1, "kv_lo": 16, "kv_hi": 1024,
         "groups": 1, "prefix_lo": 16384, "prefix_hi": 16384, "mix": 8},
        # several documents, answers sampled and drafted from each
        {**attend, "name": "shared groups 200", "seqs": 200, "q_lo": 1, "q_hi": 4, "kv_lo": 16, "kv_hi": 2048,
         "q_heads": 64, "code": "e4m3", "groups": 7, "prefix_lo": 1024, "prefix_hi": 32768, "mix": 9},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _parts(rng, total, n):
    """n numbers from 1 on that add up to total."""
    cuts = sorted(rng.sample(range(1, total), n - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    op = rng.choice(["turn", "write", "attend", "attend"])
    kind = rng.choice(["bf16", "bf16", "f16"])
    dim = rng.choice([64, 80, 128, 128])
    group = rng.choice([1, 4, 5, 8])
    kv_heads = rng.choice([1, 2, 5, 8])
    rotated = rng.choice([dim, dim, dim // 2])
    turns = {"rotated": rotated, "order": rng.choice(["blocks", "cyclic"]),
             "axes": ",".join(str(n) for n in _parts(rng, rotated // 2, rng.choice([2, 3, 3, 4]))),
             "spectrum": rng.choice(["shared", "axial"]), "layout": rng.choice(["half", "interleaved"]),
             "high": rng.choice([0, 1, 7, 24, 33]), "wide": rng.choice([1, 13, 32, 41])}
    if op == "turn":
        heads = rng.choice([1, 7, 16, 32, 40])
        return {"op": op, "batch": rng.choice([1, 2]), "tokens": _spread(rng, 1, 131072 // heads), "heads": heads,
                "dim": dim, "type": rng.choice(["bf16", "f16", "f32"]), "train": rng.random() < 0.5, **turns}
    share = max(1, kv_heads * group // 32)  # more query heads: fewer tokens
    both = {"op": op, "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "type": kind,
            "code": rng.choice(["int8", "e4m3"]), "page": rng.choice([16, 32, 64, 128]), "mix": rng.randrange(10**6)}
    if op == "write":
        seqs = _spread(rng, 1, 128)
        top = _spread(rng, 1, 16384 // share // seqs)
        return {**both, **turns, "seqs": seqs, "new_lo": max(1, top // 16), "new_hi": top, "held_lo": 0,
                "held_hi": _spread(rng, 1, 2000)}
    both |= {"empty": rng.choice([0, 0, 1]), "window": 0, "sinks": 0, "groups": 0, "prefix_lo": 0, "prefix_hi": 0}
    shares = rng.random() < 0.5
    if shares:
        both["groups"] = rng.choice([1, 1, 2, 5])
        both["prefix_hi"] = _spread(rng, 16, 32768 // both["groups"])
        both["prefix_lo"] = both["prefix_hi"] // 3
    if not shares or rng.random() < 0.3:
        both |= {"window": _spread(rng, 16, 8192), "sinks": _spread(rng, 1, 200)}
    if rng.random() < 0.7:  # decoding, single or a few drafted tokens
        seqs = max(both["groups"], _spread(rng, 1, 100))
        top = _spread(rng, 16, min(2000 if shares else 65536, 262144 // seqs))
        few = rng.choice([1, 1, 1, 4])
        return {**both, "seqs": seqs, "q_lo": 1, "q_hi": few, "kv_lo": max(few, top // 16), "kv_hi": max(few, top)}
    seqs = max(both["groups"], _spread(rng, 1, 8))  # prompts
    top = _spread(rng, 16, 2048 // share // seqs)
    return {**both, "seqs": seqs, "q_lo": max(1, top // 8), "q_hi": top, "kv_lo": top,
            "kv_hi": top + _spread(rng, 16, 8000)}


def _axis_of(case):
    """The axis of each pair: a run of pairs for each axis, or one pair to each axis in turn while it has some left."""
    left = [int(n) for n in case["axes"].split(",")]
    if case["order"] == "blocks":
        return [a for a, n in enumerate(left) for _ in range(n)]
    out = []
    while any(left):
        for a, n in enumerate(left):
            if n:
                out.append(a)
                left[a] -= 1
    return out


def _ragged(case):
    """Per sequence, tokens before the call behind the shared prefix (of the cache, where none is) and new tokens;
    the sequences' groups as (first, end, shared tokens), where the case has some."""
    r = random.Random(case["mix"])
    n = case["seqs"]
    if case["op"] == "write":
        new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(n)]
        return [r.randint(case["held_lo"], case["held_hi"]) for _ in range(n)], new, []
    new = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(n)]
    held = [max(q, r.randint(case["kv_lo"], case["kv_hi"])) - q for q in new]
    cuts = [0] + sorted(r.sample(range(1, n), case["groups"] - 1)) + [n] if case["groups"] else []
    groups = [(a, b, r.randint(case["prefix_lo"], case["prefix_hi"])) for a, b in zip(cuts, cuts[1:])]
    return held, new, groups


def _layout(case):
    """Per sequence: all its tokens before the call, new ones, and whole-page tokens that it shares."""
    held, new, groups = _ragged(case)
    share = [0] * len(new)
    for a, b, tokens in groups:
        for s in range(a, b):
            share[s] = tokens // case["page"] * case["page"]
            held[s] += tokens
    for s in range(min(case["empty"], len(new) - 1)):
        held[-1 - s] = -new[-1 - s]  # no tokens at all: every row of this sequence is empty
    return held, new, share, groups


def _seen(case):
    """(query, key) pairs of one head that the masks leave, and keys that some query sees, shared ones once a group."""
    held, new, share, groups = _layout(case)
    w, k = case["window"], case["sinks"]
    pairs = keys = 0

    def union(spans, first, last):  # keys of [first, last) in the rows' spans [lo, hi) or among their sinks
        spans = [(lo, hi) for lo, hi in spans if hi > 0]
        if not spans:
            return 0
        lo = max(first, min(lo for lo, _ in spans))
        hi = min(last, max(hi for _, hi in spans))
        return max(0, hi - lo) + max(0, min(k, lo, last) - first)

    rows = []
    for h, n in zip(held, new):
        mine = [(max(0, p + 1 - w) if w else 0, max(0, p + 1)) for p in range(h, h + n)]
        pairs += sum(hi - lo + min(k, lo) for lo, hi in mine)
        rows.append(mine)
    for a, b, _ in groups:
        keys += union([x for s in range(a, b) for x in rows[s]], 0, share[a])
    keys += sum(union(rows[s], share[s], held[s] + new[s]) for s in range(len(new)))
    return pairs, keys


def work(case):
    e = _BYTES[case["type"]]
    axes = len(case["axes"].split(",")) if "axes" in case else 0
    if case["op"] == "turn":
        values = case["batch"] * case["tokens"] * case["heads"] * case["dim"]
        passes = 2 if case["train"] else 1
        table = case["batch"] * case["tokens"] * (4 * axes + case["rotated"] * 4)
        return {"bytes": passes * (2 * values * e + table), "flops": passes * 3 * values}
    wide, page = case["kv_heads"] * case["dim"], case["page"]
    if case["op"] == "write":
        held, new, _ = _ragged(case)
        tokens = sum(new)
        back = sum(h % page + n for h, n in zip(held, new))  # rows of the touched pages, read back
        old = sum(h % page for h in held)                    # rows whose scale may grow
        moved = tokens * case["dim"] * e * 2 * (case["q_heads"] + case["kv_heads"])  # q in, out; k and v in
        moved += 2 * wide * (tokens + 2 * old) + 2 * wide * back * (1 + e) + tokens * (case["rotated"] * 4 + 4 * axes)
        return {"bytes": moved, "flops": 12 * wide * tokens + 3 * tokens * case["q_heads"] * case["dim"]}
    pairs, keys = _seen(case)
    rows = sum(_layout(case)[1]) * case["q_heads"]
    return {"bytes": 2 * keys * wide + 8 * -(-keys // page) * case["kv_heads"] + rows * (2 * case["dim"] * e + 4),
            "flops": 4 * pairs * case["q_heads"] * case["dim"]}


# ------------------------------------------------------------------------------- inputs

def _table(case):
    """(positions, rotated / 2, 2): cos and sin of position times frequency, made in 64 bits.  Spectrum "shared": pair
    j of the head has base^(-2 j / rotated), whatever its axis; "axial": pair i of an axis's n has base^(-i / n)."""
    axis, pairs = _axis_of(case), case["rotated"] // 2
    counts = [axis.count(a) for a in range(max(axis) + 1)]
    at = [j / pairs if case["spectrum"] == "shared" else axis[:j].count(axis[j]) / counts[axis[j]] for j in range(pairs)]
    freq = 10000.0 ** -torch.tensor(at, dtype=torch.float64, device="cuda")
    angle = torch.arange(_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), -1).float()


def _grid(case, tokens, first, device="cpu"):
    """(axes, tokens) positions: frames of high x wide patches (the first axes stay at 0 where there are more than
    three), each axis from `first` on; text (high 0) has the same position on every axis."""
    i = torch.arange(tokens, device=device)
    axes = len(case["axes"].split(","))
    if not case["high"]:
        return (first + i).repeat(axes, 1)
    patch = case["high"] * case["wide"]
    t, h, w = i // patch, i // case["wide"] % case["high"], i % case["wide"]
    return first + torch.stack(([torch.zeros_like(i)] * (axes - 3) + [t, h, w])[-axes:])


def _codes(shape, code, g):
    dtype, most = _CODES[code]
    x = torch.randn(shape, dtype=torch.float16, device="cuda", generator=g).mul_(most / 3.5)
    return (x.round_() if code == "int8" else x).clamp_(-most, most).to(dtype)


def _cache(case, total, groups, g):
    """Scattered pages that hold tokens (their free slots: what earlier users left there), and the page table: the
    sequences of a group have their shared whole pages in common."""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    need = [max(1, -(-n // page)) for n in total]
    shared = [0] * len(need)
    for a, b, tokens in groups:
        need[a] = max(need[a], tokens // page)
        for s in range(a, b):
            need[s] = max(need[s], tokens // page)
            shared[s] = tokens // page if s > a else 0
    pages = sum(need) - sum(shared) + 3
    ids = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, shared[s]:n] = ids[at:at + n - shared[s]]
        at += n - shared[s]
    for a, b, tokens in groups:
        table[a:b, :tokens // page] = table[a, :tokens // page].clone()
    most = _CODES[case["code"]][1]
    scales = [(2.0 + 2.0 * torch.rand(pages, heads, device="cuda", generator=g)) / most for _ in range(2)]
    return (_codes((pages, heads, page, dim), case["code"], g), _codes((pages, heads, page, dim), case["code"], g),
            scales[0], scales[1]), table


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sums(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    kind = _TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, dtype=torch.float32, device="cuda", generator=g).to(kind)

    r = random.Random(int(seed))
    if case["op"] == "turn":
        shape = (case["batch"], case["tokens"], case["heads"], case["dim"])
        top = max(1, _POSITIONS - (case["tokens"] if not case["high"] else
                                   case["tokens"] // (case["high"] * case["wide"]) + case["high"] + case["wide"]))
        grids = [_grid(case, case["tokens"], r.randrange(min(top, 4096))) % _POSITIONS for _ in range(case["batch"])]
        state = {"case": case, "x": normal(*shape), "table": _table(case),
                 "positions": torch.stack(grids, 1).to(torch.int32).cuda()}
        if case["train"]:
            state["x"].requires_grad_(True)
            state["dy"] = normal(*shape)
        return state
    if case["op"] == "write":
        held, new, groups = _ragged(case)
        share = [0] * len(new)
    else:
        held, new, share, groups = _layout(case)
    total = [h + n for h, n in zip(held, new)]
    cache, pages = _cache(case, total, groups, g)
    tokens = sum(new)
    state = {"case": case, "cache": cache, "pages": pages, "starts": _int(_sums(new)),
             "q": normal(tokens, case["q_heads"], case["dim"])}
    if case["op"] == "write":
        low = [h - h % case["page"] for h in held]
        back = _sums([h + n - f for h, n, f in zip(held, new, low)])
        # images compress positions: a sequence's new tokens start at a place of their own
        where = torch.cat([_grid(case, n, r.randint(h // 2, h)) for h, n in zip(held, new)], 1)
        state |= {"k": normal(tokens, case["kv_heads"], case["dim"]),
                  "v": normal(tokens, case["kv_heads"], case["dim"]), "held": _int(held),
                  "positions": where.to(torch.int32).cuda(), "table": _table(case), "back_first": _int(low),
                  "back_starts": _int(back), "back": back[-1]}
    else:
        state["lens"] = _int(total)
        state["q"] *= 1.5
        if groups:
            state["groups"] = _int([a for a, _, _ in groups] + [len(new)])
            state["shared"] = _int([tokens for _, _, tokens in groups])
    return state


# ------------------------------------------------------------------------------- plain forms

def _roots(table, positions, axis):
    """cos and sin (..., pairs) of positions (axes, ...): pair j's from row positions[axis[j]]."""
    axis = torch.tensor(axis, device=table.device)
    rows = positions.long()[axis].movedim(0, -1)
    return table[rows, torch.arange(len(axis), device=table.device)].unbind(-1)


def _turn(x, cos, sin, layout, rotated):
    """Rotated pairs of x (..., heads, dim) in 32 bits; cos, sin: (..., rotated / 2)."""
    x = x.float()
    c, s = cos.unsqueeze(-2), sin.unsqueeze(-2)
    part = x[..., :rotated]
    if layout == "half":
        a, b = part[..., :rotated // 2], part[..., rotated // 2:]
        y = torch.cat((a * c - b * s, a * s + b * c), -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    return torch.cat((y, x[..., rotated:]), -1)


def _owner(starts, tokens):
    """The sequence of each of the `tokens` ragged rows, and its place in it."""
    row = torch.arange(tokens, dtype=torch.int32, device=starts.device)
    seq = torch.searchsorted(starts, row, right=True) - 1
    return seq, (row - starts[seq]).long()


def _to_code(x, code):
    dtype, most = _CODES[code]
    x = x.round() if code == "int8" else x
    return x.clamp(-most, most).to(dtype)


def _plain_write(st):
    case = st["case"]
    page, rotated, layout = case["page"], case["rotated"], case["layout"]
    most = _CODES[case["code"]][1]
    tokens, held, pages = st["q"].shape[0], st["held"].long(), st["pages"].long()
    seq, place = _owner(st["starts"], tokens)
    at = held[seq] + place
    cos, sin = _roots(st["table"], st["positions"], _axis_of(case))
    q = _turn(st["q"], cos, sin, layout, rotated).to(st["q"].dtype)
    to, slot = pages[seq, at // page], at % page
    old = held % page  # rows that a sequence's last page held before
    last = pages.gather(1, (held // page).clamp(max=pages.shape[1] - 1)[:, None])[:, 0]
    for_k, for_v = _turn(st["k"], cos, sin, layout, rotated), st["v"].float()
    for x, codes, scale in ((for_k, st["cache"][0], st["cache"][2]), (for_v, st["cache"][1], st["cache"][3])):
        before = torch.where((old > 0)[:, None], scale[last], 0.0)
        grown = torch.zeros_like(scale).index_reduce_(0, to, x.abs().amax(-1), "amax") / most
        grown[last] = torch.maximum(grown[last], before)
        inverse = torch.where(grown > 0, 1.0 / grown, 0.0)
        kept = _to_code(codes[last].float() * (before * inverse[last])[..., None, None], case["code"])
        stays = (torch.arange(page, device=old.device) < old[:, None])[:, None, :, None]
        mine = torch.where(stays, kept.float(), codes[last].float()).to(codes.dtype)
        codes.view(torch.uint8)[last] = mine.view(torch.uint8)
        codes.view(torch.uint8)[to, :, slot] = _to_code(x * inverse[to][..., None], case["code"]).view(torch.uint8)
        scale[to] = grown[to]
    seq, place = _owner(st["back_starts"], st["back"])
    at = st["back_first"].long()[seq] + place
    to, slot = pages[seq, at // page], at % page
    back = [(c.view(torch.uint8)[to, :, slot].view(c.dtype).float() * s[to][..., None]).to(q.dtype)
            for c, s in (st["cache"][0::2], st["cache"][1::2])]
    return {"q": q, "k": back[0], "v": back[1], "k_scale": st["cache"][2], "v_scale": st["cache"][3]}


def _plain_attend(st):
    """A group at a time (one of all sequences, where none shares): scores of its rows against the shared tokens, once
    for the group, and against each sequence's own, and one softmax over both."""
    case = st["case"]
    page, kv, dim, group = case["page"], case["kv_heads"], case["dim"], case["q_heads"] // case["kv_heads"]
    held, new, share, groups = _layout(case)
    pages, q = st["pages"].long(), st["q"].float()
    first, out, lse = _sums(new), [], []

    def dense(ids, codes, scale):  # (..., pages) -> (..., kv heads, tokens, dim)
        x = codes.view(torch.uint8)[ids].view(codes.dtype).float() * scale[ids][..., None, None]
        return x.movedim(-4, -3).flatten(-3, -2)

    def scores(rows, keys, where, at):  # masked, of rows at `where` (..., rows) and keys at `at` (..., tokens)
        z = torch.matmul(rows, keys.transpose(-1, -2)) * dim ** -0.5
        key, pos = at[..., None, None, :], where[..., None, :, None]
        hidden = key > pos
        if case["window"]:
            hidden = hidden | ((key <= pos - case["window"]) & (key >= case["sinks"]))
        return z.masked_fill_(hidden, -math.inf)

    for a, b in [(x, y) for x, y, _ in groups] or [(0, len(new))]:
        n, most, common = b - a, max(new[a:b]), share[a]
        ends = torch.tensor([held[s] + new[s] for s in range(a, b)], device="cuda")
        counts = torch.tensor(new[a:b], device="cuda")
        rows = torch.zeros(n, most, kv, group, dim, device="cuda")
        seq = torch.repeat_interleave(torch.arange(n, device="cuda"), counts)
        place = torch.arange(first[b] - first[a], device="cuda") - torch.tensor(first[a:b], device="cuda")[seq] + first[a]
        rows[seq, place] = q[first[a]:first[b]].view(-1, kv, group, dim)
        rows = rows.permute(0, 2, 1, 3, 4).reshape(n, kv, most * group, dim)
        where = (ends - counts)[:, None] + torch.arange(most * group, device="cuda") // group
        longest = max(max(held[s] + new[s] for s in range(a, b)), common + 1)
        mine = pages[a:b, common // page:-(-longest // page)]
        k, v = (dense(mine, c, s) for c, s in (st["cache"][0::2], st["cache"][1::2]))
        at = common + torch.arange(k.shape[-2], device="cuda")
        z = scores(rows, k, where, at)
        parts, values = [z], [v]
        if common:
            ids = pages[a, :common // page]
            k, v = (dense(ids, c, s) for c, s in (st["cache"][0::2], st["cache"][1::2]))
            flat = rows.transpose(0, 1).reshape(kv, n * most * group, dim)
            z = scores(flat, k, where.reshape(-1), torch.arange(common, device="cuda"))
            parts.append(z.view(kv, n, most * group, common).transpose(0, 1))
            values.append(v)
        peak = torch.stack([z.amax(-1) for z in parts]).amax(0)[..., None].clamp(min=-1e30)
        total = torch.zeros_like(peak)
        y = torch.zeros_like(rows)
        for z, v in zip(parts, values):
            p = torch.exp(z - peak)
            total += p.sum(-1, keepdim=True)
            if v.dim() == 4:
                y += torch.matmul(p, v)
            else:
                p = p.transpose(0, 1).reshape(kv, n * most * group, -1)
                y += torch.matmul(p, v).view(kv, n, most * group, dim).transpose(0, 1)
        y = y / torch.where(total > 0, total, 1.0)
        l = (torch.log(total) + peak)[..., 0].masked_fill(total[..., 0] == 0, -math.inf)
        y = y.reshape(n, kv, most, group, dim).transpose(1, 2).reshape(n, most, kv * group, dim)
        l = l.reshape(n, kv, most, group).transpose(1, 2).reshape(n, most, kv * group)
        out.append(y[seq, place])
        lse.append(l[seq, place])
    return {"out": torch.cat(out).to(st["q"].dtype), "lse": torch.cat(lse)}


def run(st):
    case = st["case"]
    if case["op"] == "attend":
        if not own:
            return _plain_attend(st)
        out, lse = _library().cache_attention(st["q"], st["cache"], st["pages"], st["lens"], st["starts"],
                                              window=case["window"], sinks=case["sinks"], shared=st.get("shared"),
                                              groups=st.get("groups"), return_lse=True)
        return {"out": out, "lse": lse}
    if own:
        axes = tuple(int(n) for n in case["axes"].split(","))
    if case["op"] == "write":
        if not own:
            return _plain_write(st)
        bfft = _library()
        q = bfft.append_rotated(st["cache"], st["k"], st["v"], st["pages"], st["held"], st["starts"], st["table"],
                                layout=case["layout"], positions=st["positions"], axes=axes,
                                axis_order=case["order"], q=st["q"])
        k, v = bfft.read_cache(st["cache"], st["pages"], st["back_first"], st["back_starts"], st["back"],
                               dtype=st["q"].dtype)
        return {"q": q, "k": k, "v": v, "k_scale": st["cache"][2], "v_scale": st["cache"][3]}
    x = st["x"]
    if own:
        bfft = _library()
        y = bfft.rotate_positions(x, st["positions"], st["table"], layout=case["layout"], axes=axes,
                                  axis_order=case["order"])
        if not case["train"]:
            return {"y": y}
        dx, = torch.autograd.grad(y, x, st["dy"])
        return {"y": y.detach(), "dx": dx}
    cos, sin = _roots(st["table"], st["positions"], _axis_of(case))
    with torch.no_grad():
        got = {"y": _turn(x, cos, sin, case["layout"], case["rotated"]).to(x.dtype)}
        if case["train"]:
            got["dx"] = _turn(st["dy"], cos, -sin, case["layout"], case["rotated"]).to(x.dtype)
    return got


# ------------------------------------------------------------------------------- 64 bits

def _units(case, table, positions):
    """Unit roots (..., pairs) as complex numbers, a pair at a time from its axis's positions."""
    out = []
    for j, a in enumerate(_axis_of(case)):
        t = table[:, j].double()[positions[a].long()]
        out.append(torch.complex(t[..., 0], t[..., 1]))
    return torch.stack(out, -1)


def _rotate64(case, x, unit):
    """One pair at a time as complex numbers: (a + ib)(c + is)."""
    x, rotated = x.detach().double(), case["rotated"]
    if case["layout"] == "half":
        z = torch.complex(x[..., :rotated // 2], x[..., rotated // 2:rotated]) * unit[..., None, :]
        y = torch.cat((z.real, z.imag), -1)
    else:
        z = torch.view_as_complex(x[..., :rotated].reshape(*x.shape[:-1], rotated // 2, 2)) * unit[..., None, :]
        y = torch.view_as_real(z).reshape(*x.shape[:-1], rotated)
    return torch.cat((y, x[..., rotated:]), -1)


def _exact_write(case, st):
    held, new, _ = _ragged(case)
    page, most = case["page"], _CODES[case["code"]][1]
    table = st["pages"].tolist()
    unit = _units(case, st["table"], st["positions"])
    fresh = [_rotate64(case, st["k"], unit), st["v"].double()]

    def code(x):  # the nearest value that 8 bits hold
        if case["code"] == "int8":
            return x.round().clamp(-most, most)
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
        return ((x / step).round() * step).clamp(-most, most)

    back, scales = [], []
    for x, codes, scale in zip(fresh, st["cache"][:2], st["cache"][2:]):
        scale, rows, first = scale.double(), [], 0
        for s, (h, n) in enumerate(zip(held, new)):
            for p in range(h // page, (h + n - 1) // page + 1):
                a, b = max(h, p * page), min(h + n, (p + 1) * page)
                mine = x[first + a - h:first + b - h].transpose(0, 1)
                g = table[s][p]
                keep = codes[g].double()[:, :a - p * page] * scale[g][:, None, None]
                big = mine.abs().amax((1, 2)) / most
                if a > p * page:
                    big = torch.maximum(big, scale[g])
                scale[g] = big
                big = big[:, None, None]
                rows.append((torch.cat((code(keep / big), code(mine / big)), 1) * big).transpose(0, 1))
            first += n
        back.append(torch.cat(rows))
        scales.append(scale)
    return {"q": _rotate64(case, st["q"], unit), "k": back[0], "v": back[1], "k_scale": scales[0], "v_scale": scales[1]}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "turn":
        unit = _units(case, st["table"], st["positions"])
        got = {"y": _rotate64(case, st["x"], unit)}
        if case["train"]:
            got["dx"] = _rotate64(case, st["dy"], unit.conj())
        return got
    if case["op"] == "write":
        return _exact_write(case, st)
    # every sequence by itself, over the tokens that its own page table names
    held, new, _, _ = _layout(case)
    page, group, dim = case["page"], case["q_heads"] // case["kv_heads"], case["dim"]
    out = torch.zeros(sum(new), case["q_heads"], dim, dtype=torch.float64, device="cuda")
    lse = torch.full((sum(new), case["q_heads"]), -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for s, (h, n) in enumerate(zip(held, new)):
        last = h + n
        if last > 0:
            low = max(0, h + 1 - case["window"]) if case["window"] else 0
            key = torch.cat((torch.arange(min(case["sinks"], low)), torch.arange(low, last))).cuda()
            ids, slot = st["pages"][s].long()[key // page], key % page
            gap = torch.arange(h, last, device="cuda")[:, None] - key
            hidden = gap < 0
            if case["window"]:
                hidden |= (gap >= case["window"]) & (key >= case["sinks"])
            for j in range(case["kv_heads"]):
                k, v = (c.view(torch.uint8)[ids, j, slot].view(c.dtype).double() * x[ids, j].double()[:, None]
                        for c, x in zip(st["cache"][:2], st["cache"][2:]))
                mine = slice(j * group, (j + 1) * group)
                z = torch.matmul(st["q"][first:first + n, mine].double(), k.T) / math.sqrt(dim)
                z = z.masked_fill(hidden[:, None, :], -math.inf)
                lse[first:first + n, mine] = torch.logsumexp(z, -1)
                out[first:first + n, mine] = torch.matmul(torch.softmax(z, -1), v)
        first += n
    return {"out": out, "lse": lse}

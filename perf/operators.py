"""Cases of the position and cache operators: rotation by position, appending to the paged
8-bit cache, reading it back, and attention over it.

Each case is one pass through one of them, in its plain form (elementary torch operations in
32 bits) or through the library's entry points (``own``):

* ``rotate``: ``bfft.rotate_positions``, and its gradient where the case trains;
* ``append``: ``bfft.append_rotated`` (rotate queries and keys, quantise keys and values into
  their pages) and ``bfft.read_cache`` (the values that the touched pages now stand for);
* ``attend``: ``bfft.cache_attention`` over such a cache, with the log-sum-exp of each row.

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
_POSITIONS = 1 << 17  # rows of the rotation table: the longest context of the cases


def _library():
    if "bfft" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "kunlunxin-fft_b200"))
    import bfft

    return bfft


# ------------------------------------------------------------------------------- cases

def listed():
    rotate = {"op": "rotate", "batch": 1, "dim": 128, "rotated": 128, "layout": "half", "type": "bf16", "train": False}
    append = {"op": "append", "q_heads": 32, "kv_heads": 8, "dim": 128, "rotated": 128, "layout": "half",
              "type": "bf16", "code": "int8", "page": 64}
    attend = {"op": "attend", "q_heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "code": "int8", "page": 64,
              "window": 0, "empty": 0}
    return [
        # the queries of one new token: the smallest call, all latency
        {**rotate, "name": "rotate one token", "tokens": 1, "heads": 32},
        # a training step's queries, forward and backward
        {**rotate, "name": "rotate training batch", "batch": 4, "tokens": 4096, "heads": 32, "train": True},
        # a small model's odd length, in full precision, part of the head, interleaved pairs
        {**rotate, "name": "rotate odd f32 part", "tokens": 4999, "heads": 12, "dim": 96, "rotated": 64,
         "layout": "interleaved", "type": "f32", "train": True},
        # a few users, one new token each, in pages that already hold some
        {**append, "name": "append 8 tokens", "seqs": 8, "new_lo": 1, "new_hi": 1, "held_lo": 100, "held_hi": 4000,
         "mix": 1},
        # a large decoding batch with small pages
        {**append, "name": "append 256 tokens e4m3", "seqs": 256, "new_lo": 1, "new_hi": 1, "held_lo": 0,
         "held_hi": 2000, "page": 16, "code": "e4m3", "mix": 2},
        # ragged prompts, some continuing a cached prefix
        {**append, "name": "append prompts", "seqs": 16, "new_lo": 65, "new_hi": 2048, "held_lo": 0, "held_hi": 1000,
         "mix": 3},
        # odd head count and width, part of the head, interleaved
        {**append, "name": "append odd f16", "seqs": 7, "new_lo": 1, "new_hi": 333, "held_lo": 0, "held_hi": 77,
         "q_heads": 9, "kv_heads": 3, "dim": 96, "rotated": 48, "layout": "interleaved", "type": "f16",
         "code": "e4m3", "page": 32, "mix": 4},
        # one user's next token over a short context: latency
        {**attend, "name": "decode one short", "seqs": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 700, "kv_hi": 700, "mix": 5},
        # a decoding batch of ragged long contexts: bandwidth
        {**attend, "name": "decode 64 ragged", "seqs": 64, "q_lo": 1, "q_hi": 1, "kv_lo": 1024, "kv_hi": 32768,
         "mix": 6},
        # one user's next token over the longest context, few rows over a long axis
        {**attend, "name": "decode one long e4m3", "seqs": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 131001, "kv_hi": 131001,
         "q_heads": 64, "code": "e4m3", "mix": 7},
        # chunks of long prompts over what is cached of them: matrix products
        {**attend, "name": "prompt chunks", "seqs": 2, "q_lo": 2048, "q_hi": 2048, "kv_lo": 8192, "kv_hi": 16384,
         "mix": 8},
        # prompts, drafted and single tokens together, sliding window, small heads and pages, a user with an empty cache
        {**attend, "name": "mixed window f16", "seqs": 23, "q_lo": 1, "q_hi": 300, "kv_lo": 300, "kv_hi": 5000,
         "q_heads": 12, "kv_heads": 4, "dim": 64, "type": "f16", "code": "e4m3", "page": 16, "window": 1000,
         "empty": 1, "mix": 9},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotate", "append", "attend", "attend"])
    kind = rng.choice(["bf16", "bf16", "f16"])
    dim = rng.choice([64, 80, 128, 128])
    group = rng.choice([1, 4, 5, 8])
    kv_heads = rng.choice([1, 2, 5, 8])
    if op == "rotate":
        train = rng.random() < 0.5
        heads = rng.choice([1, 7, 16, 32, 40])
        tokens = _spread(rng, 1, 131072 // heads)
        return {"op": op, "batch": rng.choice([1, 2]), "tokens": tokens, "heads": heads, "dim": dim,
                "rotated": rng.choice([dim, dim, dim // 2]), "layout": rng.choice(["half", "interleaved"]),
                "type": rng.choice(["bf16", "f16", "f32"]), "train": train}
    share = max(1, kv_heads * group // 32)  # more query heads: fewer tokens
    both = {"op": op, "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "type": kind,
            "code": rng.choice(["int8", "e4m3"]), "page": rng.choice([16, 32, 64, 128]), "mix": rng.randrange(10**6)}
    if op == "append":
        seqs = _spread(rng, 1, 128)
        top = _spread(rng, 1, 16384 // share // seqs)
        return {**both, "rotated": rng.choice([dim, dim // 2]), "layout": rng.choice(["half", "interleaved"]),
                "seqs": seqs, "new_lo": max(1, top // 16), "new_hi": top, "held_lo": 0,
                "held_hi": _spread(rng, 1, 2000)}
    both |= {"window": rng.choice([0, 0, _spread(rng, 16, 4000)]), "empty": rng.choice([0, 0, 1])}
    if rng.random() < 0.6:  # decoding, single or a few drafted tokens
        seqs = _spread(rng, 1, 64)
        top = _spread(rng, 16, min(131072, 524288 // seqs))
        few = rng.choice([1, 1, 1, 4])
        return {**both, "seqs": seqs, "q_lo": 1, "q_hi": few, "kv_lo": max(few, top // 16), "kv_hi": top}
    seqs = _spread(rng, 1, 8)
    top = _spread(rng, 16, 4096 // share // seqs)
    return {**both, "seqs": seqs, "q_lo": max(1, top // 8), "q_hi": top, "kv_lo": top,
            "kv_hi": top + _spread(rng, 16, 8000)}


def _ragged(case):
    """Per sequence: tokens in the cache before the call, new tokens (the queries)."""
    r = random.Random(case["mix"])
    n = case["seqs"]
    if case["op"] == "append":
        new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(n)]
        return [r.randint(case["held_lo"], case["held_hi"]) for _ in range(n)], new
    new = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(n)]
    total = [max(q, r.randint(case["kv_lo"], case["kv_hi"])) for q in new]
    held = [t - q for t, q in zip(total, new)]
    for s in range(min(case["empty"], n - 1)):
        held[s] = -new[s]  # nothing cached at all: every row of this sequence is empty
    return held, new


def _visible(case):
    """(query, key) pairs that the causal mask and the window leave, of one head, and keys that some query sees."""
    pairs = keys = 0
    w = case["window"]
    for held, new in zip(*_ragged(case)):
        last = held + new
        if last <= 0:
            continue
        if w <= 0:
            pairs += new * held + new * (new + 1) // 2
            keys += last
        else:
            grow = max(0, min(new, w - held))  # queries whose window reaches the first key
            pairs += grow * held + grow * (grow + 1) // 2 + (new - grow) * w
            keys += last - max(0, held + 1 - w)
    return pairs, keys


def work(case):
    e = _BYTES[case["type"]]
    if case["op"] == "rotate":
        values = case["batch"] * case["tokens"] * case["heads"] * case["dim"]
        passes = 2 if case["train"] else 1
        table = case["batch"] * case["tokens"] * (4 + case["rotated"] * 4)
        return {"bytes": passes * (2 * values * e + table), "flops": passes * 3 * values}
    held, new = _ragged(case)
    tokens, wide, page = sum(new), case["kv_heads"] * case["dim"], case["page"]
    if case["op"] == "append":
        back = sum(h % page + n for h, n in zip(held, new))  # rows of the touched pages, read back
        old = sum(h % page for h in held)                    # rows whose scale may grow
        moved = tokens * case["dim"] * e * 2 * (case["q_heads"] + case["kv_heads"])  # q in, out; k and v in
        moved += 2 * wide * (tokens + 2 * old) + 2 * wide * back * (1 + e) + tokens * case["rotated"] * 4
        return {"bytes": moved, "flops": 12 * wide * tokens + 3 * tokens * case["q_heads"] * case["dim"]}
    pairs, keys = _visible(case)
    rows = tokens * case["q_heads"]
    pages = sum(-(-(h + n) // page) for h, n in zip(held, new) if h + n > 0)
    return {"bytes": 2 * keys * wide + 8 * pages * case["kv_heads"] + rows * (2 * case["dim"] * e + 4),
            "flops": 4 * pairs * case["q_heads"] * case["dim"]}


# ------------------------------------------------------------------------------- inputs

def _table(rotated, device):
    """(positions, rotated / 2, 2): cos and sin of position times frequency, made in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, rotated, 2, dtype=torch.float64, device=device) / rotated)
    angle = torch.arange(_POSITIONS, dtype=torch.float64, device=device)[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), -1).float()


def _codes(shape, code, g):
    dtype, most = _CODES[code]
    x = torch.randn(shape, dtype=torch.float16, device="cuda", generator=g).mul_(most / 3.5)
    return (x.round_() if code == "int8" else x).clamp_(-most, most).to(dtype)


def _cache(case, held, new, g):
    """Scattered pages that hold tokens (their free slots: what earlier users left there), and the page table."""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    need = [max(1, -(-(h + n) // page)) for h, n in zip(held, new)]
    pages = sum(need) + 3
    ids = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
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

    if case["op"] == "rotate":
        shape = (case["batch"], case["tokens"], case["heads"], case["dim"])
        positions = torch.arange(case["tokens"], dtype=torch.int32, device="cuda").repeat(case["batch"], 1)
        positions += torch.randint(0, _POSITIONS - case["tokens"], (case["batch"], 1), dtype=torch.int32, device="cuda",
                                   generator=g)
        state = {"case": case, "x": normal(*shape), "positions": positions, "table": _table(case["rotated"], "cuda")}
        if case["train"]:
            state["x"].requires_grad_(True)
            state["dy"] = normal(*shape)
        return state
    held, new = _ragged(case)
    cache, pages = _cache(case, held, new, g)
    tokens = sum(new)
    state = {"case": case, "cache": cache, "pages": pages, "starts": _int(_sums(new)),
             "q": normal(tokens, case["q_heads"], case["dim"])}
    if case["op"] == "append":
        low = [h - h % case["page"] for h in held]
        back = _sums([h + n - f for h, n, f in zip(held, new, low)])
        state |= {"k": normal(tokens, case["kv_heads"], case["dim"]),
                  "v": normal(tokens, case["kv_heads"], case["dim"]), "held": _int(held),
                  "table": _table(case["rotated"], "cuda"), "back_first": _int(low), "back_starts": _int(back),
                  "back": back[-1]}
    else:
        state["lens"] = _int([h + n for h, n in zip(held, new)])
        state["longest"], state["most_new"] = max(max(h + n, 1) for h, n in zip(held, new)), max(new)
        state["q"] *= 1.5
    return state


# ------------------------------------------------------------------------------- plain forms

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


def _plain_append(st):
    case = st["case"]
    page, rotated, layout = case["page"], case["rotated"], case["layout"]
    most = _CODES[case["code"]][1]
    tokens, held, pages = st["q"].shape[0], st["held"].long(), st["pages"].long()
    seq, place = _owner(st["starts"], tokens)
    at = held[seq] + place
    cos, sin = st["table"][at].unbind(-1)
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
    case = st["case"]
    page, kv, dim, group = case["page"], case["kv_heads"], case["dim"], case["q_heads"] // case["kv_heads"]
    pages, lens, starts = st["pages"].long(), st["lens"].long(), st["starts"]
    seqs, top, most = pages.shape[0], st["longest"], st["most_new"]

    def dense(codes, scale):  # (seqs, kv heads, longest, dim)
        x = codes.view(torch.uint8)[pages].view(codes.dtype).float() * scale[pages][..., None, None]
        return x.transpose(1, 2).reshape(seqs, kv, -1, dim)[:, :, :top]

    seq, place = _owner(starts, st["q"].shape[0])
    q = torch.zeros(seqs, most, kv, group, dim, device="cuda")
    q[seq, place] = st["q"].float().reshape(-1, kv, group, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(seqs, kv, most * group, dim)
    score = torch.matmul(q, dense(st["cache"][0], st["cache"][2]).transpose(-1, -2)) * dim ** -0.5
    new = (starts[1:] - starts[:-1]).long()
    where = (lens - new)[:, None] + torch.arange(most, device="cuda")
    key = torch.arange(top, device="cuda")
    seen = (key <= where[..., None]) & (key < lens[:, None, None])
    if case["window"] > 0:
        seen &= key > where[..., None] - case["window"]
    seen = seen.repeat_interleave(group, 1)[:, None]
    score = score.masked_fill(~seen, -math.inf)
    peak = score.amax(-1, keepdim=True).clamp(min=-1e30)
    score = torch.exp(score - peak)
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score, dense(st["cache"][1], st["cache"][3])) / torch.where(total > 0, total, 1.0)
    lse = (torch.log(total) + peak)[..., 0].masked_fill(total[..., 0] == 0, -math.inf)
    out = out.reshape(seqs, kv, most, group, dim).transpose(1, 2).reshape(seqs, most, kv * group, dim)
    lse = lse.reshape(seqs, kv, most, group).transpose(1, 2).reshape(seqs, most, kv * group)
    return {"out": out[seq, place].to(st["q"].dtype), "lse": lse[seq, place]}


def run(st):
    case = st["case"]
    if case["op"] == "rotate":
        x = st["x"]
        if own:
            bfft = _library()
            y = bfft.rotate_positions(x, st["positions"], st["table"], layout=case["layout"])
            if not case["train"]:
                return {"y": y}
            dx, = torch.autograd.grad(y, x, st["dy"])
            return {"y": y.detach(), "dx": dx}
        cos, sin = st["table"][st["positions"].long()].unbind(-1)
        with torch.no_grad():
            got = {"y": _turn(x, cos, sin, case["layout"], case["rotated"]).to(x.dtype)}
            if case["train"]:
                got["dx"] = _turn(st["dy"], cos, -sin, case["layout"], case["rotated"]).to(x.dtype)
        return got
    if case["op"] == "append":
        if not own:
            return _plain_append(st)
        bfft = _library()
        q = bfft.append_rotated(st["cache"], st["k"], st["v"], st["pages"], st["held"], st["starts"], st["table"],
                                layout=case["layout"], q=st["q"])
        k, v = bfft.read_cache(st["cache"], st["pages"], st["back_first"], st["back_starts"], st["back"],
                               dtype=st["q"].dtype)
        return {"q": q, "k": k, "v": v, "k_scale": st["cache"][2], "v_scale": st["cache"][3]}
    if not own:
        return _plain_attend(st)
    out, lse = _library().cache_attention(st["q"], st["cache"], st["pages"], st["lens"], st["starts"],
                                          window=case["window"], return_lse=True)
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------------------- 64 bits

def _rotate64(x, angle_cos, angle_sin, layout, rotated, sign):
    """One pair at a time as complex numbers: (a + ib)(c + is)."""
    x = x.detach().double()
    unit = torch.complex(angle_cos.double(), sign * angle_sin.double())
    if layout == "half":
        z = torch.complex(x[..., :rotated // 2], x[..., rotated // 2:rotated]) * unit[..., None, :]
        y = torch.cat((z.real, z.imag), -1)
    else:
        z = torch.view_as_complex(x[..., :rotated].reshape(*x.shape[:-1], rotated // 2, 2)) * unit[..., None, :]
        y = torch.view_as_real(z).reshape(*x.shape[:-1], rotated)
    return torch.cat((y, x[..., rotated:]), -1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotate":
        t = st["table"][st["positions"].long()]
        got = {"y": _rotate64(st["x"], t[..., 0], t[..., 1], case["layout"], case["rotated"], 1.0)}
        if case["train"]:
            got["dx"] = _rotate64(st["dy"], t[..., 0], t[..., 1], case["layout"], case["rotated"], -1.0)
        return got
    held, new = _ragged(case)
    page = case["page"]
    table = st["pages"].tolist()
    if case["op"] == "append":
        most = _CODES[case["code"]][1]
        where = torch.cat([torch.arange(h, h + n) for h, n in zip(held, new)]).cuda()
        t = st["table"][where]
        fresh = [_rotate64(st["k"], t[..., 0], t[..., 1], case["layout"], case["rotated"], 1.0), st["v"].double()]
        q = _rotate64(st["q"], t[..., 0], t[..., 1], case["layout"], case["rotated"], 1.0)

        def code(x):  # the nearest value that 8 bits hold
            if case["code"] == "int8":
                return x.round().clamp(-most, most)
            unit = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
            return ((x / unit).round() * unit).clamp(-most, most)

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
        return {"q": q, "k": back[0], "v": back[1], "k_scale": scales[0], "v_scale": scales[1]}
    group, dim = case["q_heads"] // case["kv_heads"], case["dim"]
    out = torch.zeros(sum(new), case["q_heads"], dim, dtype=torch.float64, device="cuda")
    lse = torch.full((sum(new), case["q_heads"]), -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for s, (h, n) in enumerate(zip(held, new)):
        last = h + n
        low = max(0, h + 1 - case["window"]) if case["window"] > 0 else 0
        if last > 0:
            ids = torch.tensor(table[s][low // page:-(-last // page)], device="cuda")
            cut = slice(low - low // page * page, last - low // page * page)
            gap = torch.arange(h, last, device="cuda")[:, None] - torch.arange(low, last, device="cuda")
            hidden = (gap < 0) | ((gap >= case["window"]) if case["window"] > 0 else gap < 0)
            for j in range(case["kv_heads"]):
                k, v = ((c.view(torch.uint8)[ids, j].view(c.dtype).double() * x[ids, j].double()[:, None, None])
                        .reshape(-1, dim)[cut] for c, x in zip(st["cache"][:2], st["cache"][2:]))
                for i in range(j * group, (j + 1) * group):
                    z = (st["q"][first:first + n, i].double() @ k.T) / math.sqrt(dim)
                    z = z.masked_fill(hidden, -math.inf)
                    lse[first:first + n, i] = torch.logsumexp(z, -1)
                    out[first:first + n, i] = torch.softmax(z, -1) @ v
        first += n
    return {"out": out, "lse": lse}

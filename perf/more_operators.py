"""The operators of a server's step around the paged 8-bit KV cache that this library is measured on
beside those of ``operators.py``: the maps of a step's packed rows from its requests' lengths and the
pages that groups of sequences share, rotary positions with several axes (alone, and fused with the
heads' norms and the paged cache's writer), and attention of new rows, one or many for each
sequence, over the paged cache, with a prefix that a group shares computed once for all of it.

``run`` computes each in plain torch where ``own`` is false and calls ``brasa_amd`` where it is true. Head
counts are those of the benchmark and the tests (32 query heads over 8 KV heads of 128, and other
GQA groups); keys are per-head RMS-normed, values N(0, 1). The cache's layout and scale are the
paged cache's: pages of 64 positions of every KV head, e4m3 codes and one power of two 2^(x - 127)
for each (page, head), the smallest with which the block's largest magnitude fits 448.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DIM = 128
PAGE = 64
TOP = 448.0  # the largest e4m3 value
EPS = 1e-6


# ---- cases -------------------------------------------------------------------------------------
def listed():
    return [
        # the maps of a decode step: one token for each of 64 sequences behind two system prompts
        {"name": "rows_step", "op": "rows", "n": 64, "new_min": 1, "new_max": 1, "old_min": 100,
         "old_max": 8000, "groups": 2, "prefix": 64, "behind": 0, "lens": 1},
        # the maps of a full turn: a thousand requests, prompts of any length beside single tokens
        {"name": "rows_turn", "op": "rows", "n": 1000, "new_min": 1, "new_max": 400, "old_min": 0,
         "old_max": 4000, "groups": 40, "prefix": 512, "behind": 1000, "lens": 2},
        # an image's patches in a vision encoder: rows and columns, heads of 72
        {"name": "rope_patches", "op": "rope", "tokens": 1027, "heads": 16, "dim": 72, "axes": 2,
         "interleaved": False, "behind": 0},
        # a video's and its text's queries of a long prompt: time, height and width
        {"name": "rope_video", "op": "rope", "tokens": 16000, "heads": 32, "dim": 128, "axes": 3,
         "interleaved": True, "behind": 384},
        # one layer's cache write of a decode step: a token for each of 64 sequences
        {"name": "store_step", "op": "store", "hq": 32, "hkv": 8, "n": 64, "new_min": 1,
         "new_max": 1, "old_min": 100, "old_max": 8000, "axes": 1, "interleaved": False, "lens": 3},
        # the cache write behind packed prompts with images, some of them after a cached prefix
        {"name": "store_prompts", "op": "store", "hq": 32, "hkv": 8, "n": 12, "new_min": 40,
         "new_max": 2500, "old_min": 0, "old_max": 700, "axes": 3, "interleaved": True, "lens": 4},
        # the first reply token of one short chat: bound by launch and latency
        {"name": "attend_short", "op": "attend", "hq": 32, "hkv": 8, "out": "f32", "n": 1,
         "groups": 0, "prefix": 0, "new_min": 1, "new_max": 1, "old_min": 256, "old_max": 256,
         "layers": 1, "lens": 5},
        # four beams of one answer to a long document, every layer of a model
        {"name": "attend_beams", "op": "attend", "hq": 32, "hkv": 8, "out": "f32", "n": 4,
         "groups": 1, "prefix": 15936, "new_min": 1, "new_max": 1, "old_min": 40, "old_max": 300,
         "layers": 36, "lens": 6},
        # a serving batch behind one system prompt: a token for each of 64 sequences
        {"name": "attend_batch", "op": "attend", "hq": 32, "hkv": 8, "out": "f16", "n": 64,
         "groups": 1, "prefix": 8192, "new_min": 1, "new_max": 1, "old_min": 100, "old_max": 1200,
         "layers": 4, "lens": 7},
        # drafted tokens under verification: a few rows for each sequence, behind three prompts
        {"name": "attend_drafts", "op": "attend", "hq": 32, "hkv": 8, "out": "f32", "n": 24,
         "groups": 3, "prefix": 2048, "new_min": 2, "new_max": 7, "old_min": 30, "old_max": 3000,
         "layers": 1, "lens": 8},
        # a dozen chat prompts behind one system prompt
        {"name": "attend_prompts", "op": "attend", "hq": 32, "hkv": 8, "out": "f16", "n": 12,
         "groups": 1, "prefix": 4096, "new_min": 5, "new_max": 600, "old_min": 0, "old_max": 0,
         "layers": 1, "lens": 9},
        # chunks of long documents after what is cached of them: the largest pass
        {"name": "attend_chunks", "op": "attend", "hq": 32, "hkv": 8, "out": "f16", "n": 3,
         "groups": 0, "prefix": 0, "new_min": 1000, "new_max": 4096, "old_min": 500,
         "old_max": 9000, "layers": 1, "lens": 10},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rows", "rope", "store", "attend", "attend", "attend"])
    hq, hkv = rng.choice([(32, 8), (32, 8), (16, 8), (32, 4), (32, 32), (8, 8)])
    seed = rng.randrange(1 << 20)
    if op == "rows":
        n = _log(rng, 1, 1500)
        return {"op": op, "n": n, "new_min": rng.choice([0, 1]),
                "new_max": rng.choice([1, _log(rng, 1, max(2, 40000 // n))]), "old_min": 0,
                "old_max": _log(rng, 2, min(16000, 8000000 // n)), "groups": rng.randint(0, min(n, 50)),
                "prefix": PAGE * rng.randint(0, 20), "behind": rng.choice([0, _log(rng, 1, 1000)]),
                "lens": seed}
    if op == "rope":
        dim, axes = 2 * rng.randint(8, 128), rng.randint(1, 4)
        heads = rng.choice([1, 3, 16, 32, 40])
        return {"op": op, "tokens": _log(rng, 1, min(30000, 60000000 // (heads * dim))),
                "heads": heads, "dim": dim, "axes": axes, "interleaved": rng.random() < 0.5,
                "behind": rng.choice([0, _log(rng, 1, 300)])}
    if op == "store":
        n = _log(rng, 1, 128)
        step = rng.random() < 0.4
        return {"op": op, "hq": hq, "hkv": hkv, "n": n, "new_min": 1,
                "new_max": rng.choice([1, 1, 4]) if step else _log(rng, 2, max(3, 12000 // n)),
                "old_min": 0, "old_max": _log(rng, 1, 100000 // n), "axes": rng.randint(1, 4),
                "interleaved": rng.random() < 0.5, "lens": seed}
    kind = rng.choice(["decode", "decode", "drafts", "prompts"])
    n = _log(rng, 1, 150 if kind == "decode" else 24)
    groups = rng.choice([0, 1, 1, min(n, 3), max(1, n // 4)])
    new = {"decode": 1, "drafts": 8, "prompts": _log(rng, 10, max(12, 6000 // n))}[kind]
    prefix = PAGE * _log(rng, 1, 200) if groups else 0
    prefix = min(prefix, 600000 // (n * hkv) * PAGE if kind != "decode" else prefix)
    return {"op": op, "hq": hq, "hkv": hkv, "out": rng.choice(["f32", "f16"]), "n": n,
            "groups": groups, "prefix": prefix, "new_min": rng.choice([0, 1]) if n > 2 else 1,
            "new_max": new, "old_min": 0, "old_max": _log(rng, 2, max(3, min(8000, 800000 // (n * hkv)))),
            "layers": rng.choice([1, 1, 2, 8]) if n < 12 and kind == "decode" else 1, "lens": seed}


# ---- inputs ------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _lens(case, lo, hi, salt=0):
    """n lengths of [lo, hi], spread over their logarithm; the case's own, whatever the seed."""
    r = random.Random(case["lens"] * 7 + salt)
    if case[hi] <= case[lo]:
        return [case[lo]] * case["n"]
    return [_log(r, max(case[lo], 1), case[hi]) if case[lo] or r.random() < 0.95 else 0
            for _ in range(case["n"])]


def _new(case):
    """New rows of each sequence; one at least in all."""
    new = _lens(case, "new_min", "new_max", 1)
    return new if sum(new) else [1] * len(new)


def _groups(case):
    """First sequence of each group, and the end of the last: equal runs of the sequences."""
    g = case["groups"]
    return [case["n"] * i // g for i in range(g + 1)] if g else []


def _held(case):
    """Positions each sequence holds before the step, a group's prefix included."""
    return [x + (case["prefix"] if case["groups"] else 0) for x in _lens(case, "old_min", "old_max")]


def _starts(lens):
    out = [0]
    for x in lens:
        out.append(out[-1] + x)
    return out


def _blocks(lens):
    return [-(-n // PAGE) for n in lens]


def _normed(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _tables(g, case, lens, spare):
    """Page tables of sequences of `lens` positions: ids from all over the pool, -1 where a row has
    none, a group's first pages alike in all of its rows. Returns the table and the pool's pages."""
    counts = _blocks(lens)
    groups = _groups(case) if "groups" in case else []
    shared = case["prefix"] // PAGE if groups else 0
    group = [0] * len(lens)
    for j, (a, b) in enumerate(zip(groups, groups[1:])):
        group[a:b] = [j] * (b - a)
    pages = sum(counts) - shared * (len(lens) - max(len(groups) - 1, 0)) + spare
    ids = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    table = torch.full((len(lens), max(max(counts), 1)), -1, dtype=torch.int32, device="cuda")
    at = shared * max(len(groups) - 1, 0)
    for i, c in enumerate(counts):
        table[i, :shared] = ids[group[i] * shared:(group[i] + 1) * shared]
        table[i, shared:c] = ids[at:at + c - shared]
        at += c - shared
    return table, pages


def _pool(g, layers, pages, hkv, kind):
    """Codes and scales of a pool: quantised keys (normed) or values of every position."""
    codes = torch.empty(layers, pages, hkv, PAGE, DIM, dtype=torch.uint8, device="cuda")
    exps = torch.empty(layers, pages, hkv, dtype=torch.uint8, device="cuda")
    gain = 2.0 ** torch.randint(-2, 3, (hkv, 1, 1), generator=g, device="cuda")
    for i in range(layers):
        for a in range(0, pages, 2048):
            x = torch.randn(min(2048, pages - a), hkv, PAGE, DIM, generator=g, device="cuda")
            x = (_normed(x) if kind == "k" else x) * gain
            e = _exponent(x.abs().amax((-1, -2)))
            codes[i, a:a + 2048], exps[i, a:a + 2048] = _codes(x, e[..., None, None]), e.to(torch.uint8)
    return codes, exps


def _sections(half, axes):
    """Pairs of each axis: nearly equal shares, the first axis the largest."""
    each = half // axes
    return [half - each * (axes - 1)] + [each] * (axes - 1)


def _axis_of(half, axes, interleaved):
    """Axis of each pair: one run for each axis, or the axes in turn while each has pairs left."""
    left = _sections(half, axes)
    if not interleaved:
        return [a for a in range(axes) for _ in range(left[a])]
    out = []
    while len(out) < half:
        for a in range(axes):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


def _grid(pos, axes):
    """Positions of each axis [axes, rows] of rows at `pos`: a hundred text rows, alike in every axis,
    then an image of 16 x 16 patches or a few of its frames, and so on."""
    at = pos % 868
    text = at < 100
    base, i = pos - at + 100, (at - 100).clamp(min=0)
    ways = [base + i // 256, base + i % 256 // 16, base + i % 16, base + i % 7]
    return torch.stack([torch.where(text, pos, ways[a]) for a in range(axes)]).to(torch.int32)


def _angles(max_pos, dim):
    """cos and sin of p * 1e6^(-2 i / dim), in 64 bits, as a program's tables hold them."""
    i = torch.arange(dim // 2, dtype=torch.float64, device="cuda")
    a = torch.arange(max_pos, dtype=torch.float64, device="cuda")[:, None] * 1e6 ** (-2 * i / dim)
    return torch.cos(a).float(), torch.sin(a).float()


def _inputs(case, seed):
    """What the case reads, from the seed alone."""
    g, op = _gen(seed), case["op"]
    if op == "rope":
        tokens, heads, dim = case["tokens"], case["heads"], case["dim"]
        start = int(torch.randint(0, 1000, (1,), generator=g, device="cuda"))
        pos = _grid(torch.arange(start, start + tokens, device="cuda"), case["axes"])
        rows = tokens + case["behind"]
        full = torch.full((case["axes"], rows), -1, dtype=torch.int32, device="cuda")
        full[:, :tokens] = pos
        cos, sin = _angles(32768, dim)
        return {"x": torch.randn(rows, heads, dim, generator=g, device="cuda"), "rope_pos": full,
                "cos": cos, "sin": sin, "rows": rows}
    n, new, old = case["n"], _new(case), _held(case) if "groups" in case else _lens(case, "old_min", "old_max")
    rows, starts = sum(new), _starts(new)
    lens = [a + b for a, b in zip(new, old)]
    if op == "rows":
        table, pages = _tables(g, case, lens, 16)
        return {"add": _ints(new), "len": _ints(old), "table": table, "pages": pages,
                "group": _ints(_groups(case) or [0]), "rows": rows + case["behind"]}
    s = {"cu": _ints(starts), "pos": _ints(old), "rows": rows}
    s["table"], s["pages"] = _tables(g, case, lens, 16)
    if op == "store":
        hkv = case["hkv"]
        s["k"], s["k_exp"] = _pool(g, 1, s["pages"], hkv, "k")
        s["v"], s["v_exp"] = _pool(g, 1, s["pages"], hkv, "v")
        s["q_new"], s["k_new"], s["v_new"] = (
            torch.randn(rows, h, DIM, generator=g, device="cuda") for h in (case["hq"], hkv, hkv))
        # a projection's rows are of any size before their norm
        s["q_new"] *= 3 * torch.rand(rows, 1, 1, generator=g, device="cuda") + 0.1
        s["q_norm"] = torch.rand(DIM, generator=g, device="cuda") + 0.5
        s["k_norm"] = torch.rand(DIM, generator=g, device="cuda") + 0.5
        row = torch.arange(rows, device="cuda", dtype=torch.int32)
        seq = torch.searchsorted(s["cu"], row, right=True) - 1
        s["rope_pos"] = _grid(s["pos"][seq] + row - s["cu"][seq], case["axes"])
        s["cos"], s["sin"] = _angles(32768, DIM)
        return s
    s["k"], s["k_exp"] = _pool(g, case["layers"], s["pages"], case["hkv"], "k")
    s["v"], s["v_exp"] = _pool(g, case["layers"], s["pages"], case["hkv"], "v")
    s["q"] = _normed(torch.randn(case["layers"], rows, case["hq"], DIM, generator=g, device="cuda"))
    s["group"] = _ints(_groups(case) or [0])
    s["prefix"] = _ints([case["prefix"]] * max(case["groups"], 1))
    return s


def prepare(case, seed):
    s = dict(case, **_inputs(case, seed))
    op = s["op"]
    if op == "rows":
        rows = s["rows"]
        s["cu"], s["lk"] = _ints([0] * (s["n"] + 1)), torch.empty_like(s["len"])
        s["seq"], s["pos"], s["slot"] = (torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(3))
        s["prefix_out"] = torch.zeros(max(s["groups"], 1), dtype=torch.int32, device="cuda")
    elif op in ("rope", "store"):
        dim = s.get("dim", DIM)
        s["axis_of"] = _axis_of(dim // 2, s["axes"], s["interleaved"])
    elif op == "attend":
        s["new"], s["held"], s["first"] = _new(case), _held(case), _groups(case)
        s["o"] = torch.zeros(s["layers"], s["rows"], s["hq"], DIM, device="cuda",
                             dtype=torch.float32 if s["out"] == "f32" else torch.float16)
        if own:  # the step's scratch, as large as the library says
            from brasa_amd import attention_paged_workspace_len
            need = attention_paged_workspace_len(s["n"], s["groups"], s["rows"], s["hq"], s["hkv"])
            s["work"] = torch.zeros(max(need, 256), dtype=torch.uint8, device="cuda")
    return s


# ---- the plain forms ---------------------------------------------------------------------------
def _exponent(amax):
    """The scale byte of blocks by their largest magnitude: the least x >= 0 with
    amax <= 448 * 2^(x - 127). Whole numbers of the magnitude's bits, so no rounding is near."""
    bits = amax.view(torch.int32)
    # a mantissa over 1.75 (448 = 1.75 * 2^8) takes the next power of two
    return ((bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000).int()).clamp_(min=0)


def _codes(x, exps):
    """x / 2^(exps - 127) rounded to e4m3 (exact up to that rounding), as bytes."""
    # in two steps, as 2^(127 - exps) itself may leave the range
    half = (127 - exps.int()) // 2
    y = torch.ldexp(torch.ldexp(x, half), 127 - exps.int() - half)
    return y.to(torch.float8_e4m3fn).view(torch.uint8)


def _values(codes, exps):
    one = torch.ones((), device="cuda")
    return codes.view(torch.float8_e4m3fn).float() * torch.ldexp(one, exps.int() - 127)[..., None, None]


def _rows_plain(s):
    n, rows, width = s["n"], s["rows"], s["table"].shape[1]
    cu = torch.cat([s["add"].new_zeros(1), torch.cumsum(s["add"], 0).int()])
    row = torch.arange(rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(cu, row, right=True).int() - 1
    there = seq < n
    at = seq.clamp(max=n - 1).long()
    pos = s["len"][at] + row - cu[at]
    page = s["table"][at, (pos // PAGE).clamp(max=width - 1).long()]
    slot = torch.where(page >= 0, page * PAGE + pos % PAGE, -1)
    got = {"cu": cu, "lk": s["len"] + s["add"]}
    for name, x in (("seq", seq), ("pos", pos), ("slot", slot)):
        got[name] = torch.where(there, x, -1)
    # leading full pages that every row of a group with positions names alike
    if not s["groups"]:
        return dict(got, prefix=s["prefix_out"])
    full = s["len"] // PAGE
    live = s["len"] > 0
    group = torch.searchsorted(s["group"], torch.arange(n, device="cuda", dtype=torch.int32), right=True) - 1
    none = torch.full((s["groups"],), n, dtype=torch.long, device="cuda")
    index = torch.arange(n, device="cuda")
    first = none.scatter_reduce(0, group, torch.where(live, index, n), "amin")
    lead = s["table"][first.clamp(max=n - 1)][group]
    col = torch.arange(width, device="cuda")[None]
    alike = (s["table"] == lead) & (lead >= 0) & (col < full[:, None])
    run = torch.cumprod(alike.int(), 1).sum(1)
    run = torch.where(live, run, width)
    least = torch.full_like(none, width).scatter_reduce(0, group, run, "amin")
    count = torch.zeros_like(none).scatter_add(0, group, live.long())
    return dict(got, prefix=torch.where(count > 1, least * PAGE, 0).int())


def _rotated(x, s, bits):
    """x [rows, heads, dim] rotated at the rows' positions; rows at -1 as they are."""
    half = x.shape[-1] // 2
    pos = s["rope_pos"][torch.tensor(s["axis_of"], device="cuda")].t()  # [rows, half]
    pair = torch.arange(half, device="cuda")[None]
    at = pos.clamp(min=0).long()
    c, n = s["cos"][at, pair].to(bits)[:, None], s["sin"][at, pair].to(bits)[:, None]
    a, b = x[..., :half].to(bits), x[..., half:].to(bits)
    y = torch.cat([a * c - b * n, b * c + a * n], -1)
    return torch.where((s["rope_pos"] >= 0).all(0)[:, None, None], y, x.to(bits))


def _norm_rotated(x, w, s):
    """In 64 bits: what it gives is rounded to codes, and a value may lie next to a border."""
    y = x.double()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.double()
    return _rotated(y, s, torch.float64).float()


def _store_plain(s, new, codes, exps):
    """One of K and V: `new` [rows, hkv, 128] into the pages, in place."""
    rows, hkv, width = s["rows"], s["hkv"], s["table"].shape[1]
    row = torch.arange(rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["cu"], row, right=True) - 1
    pos = s["pos"][seq] + row - s["cu"][seq]
    page = s["table"][seq, pos // PAGE].long()
    most = torch.zeros(s["pages"], hkv, device="cuda")
    most.scatter_reduce_(0, page[:, None].expand(-1, hkv), new.abs().amax(-1), "amax")
    # a block whose first rows were there before keeps their scale as a lower bound
    held = s["pos"] % PAGE
    grows = (held > 0) & (s["cu"][1:] > s["cu"][:-1])
    first = s["table"].gather(1, (s["pos"] // PAGE).clamp(max=width - 1).long()[:, None])[:, 0].long()
    fresh = torch.ones(s["pages"] + 1, dtype=torch.bool, device="cuda")
    fresh[torch.where(grows, first, s["pages"])] = False
    touched = torch.zeros(s["pages"], dtype=torch.bool, device="cuda")
    touched[page] = True
    e = _exponent(most)
    e = torch.where(fresh[:-1, None], e, torch.maximum(e, exps.int()))
    e = torch.where(touched[:, None], e, exps.int())
    # the earlier rows of those blocks, to the new scale
    at = first.clamp(min=0)
    old = codes[at]
    again = _codes(old.view(torch.float8_e4m3fn).float(), (127 + e[at] - exps[at].int())[..., None, None])
    slot = torch.arange(PAGE, device="cuda")[None, None, :, None]
    again = torch.where(slot < held[:, None, None, None], again, old)
    codes[at[grows]] = again[grows]
    exps.copy_(e)
    codes[page, :, pos % PAGE] = _codes(new, e[page][..., None])


def _attend_plain(s, layer):
    hq, hkv, at = s["hq"], s["hkv"], 0
    for i, (new, held) in enumerate(zip(s["new"], s["held"])):
        if not new:
            continue
        ids = s["table"][i, :-(-(new + held) // PAGE)].long()
        k, v = (_values(s[c][layer, ids], s[c + "_exp"][layer, ids]).transpose(0, 1)
                .reshape(hkv, -1, DIM)[:, :new + held].contiguous() for c in ("k", "v"))
        q = s["q"][layer, at:at + new].reshape(new, hkv, hq // hkv, DIM).transpose(0, 1) / math.sqrt(DIM)
        p = q.reshape(hkv, -1, DIM) @ k.transpose(1, 2)
        p = p.view(hkv, new, hq // hkv, new + held)
        hidden = torch.arange(new + held, device="cuda")[None] > torch.arange(held, held + new, device="cuda")[:, None]
        p.masked_fill_(hidden[None, :, None], -math.inf)
        p.sub_(p.amax(-1, keepdim=True)).exp_()
        o = p.view(hkv, -1, new + held) @ v / p.sum(-1).view(hkv, -1, 1)
        s["o"][layer, at:at + new] = o.view(hkv, new, -1, DIM).transpose(0, 1).reshape(new, hq, DIM)
        at += new


# ---- one pass ----------------------------------------------------------------------------------
_kernels = None


def _calls(s):
    """The library's object and the state's addresses, kept as a program keeps them."""
    global _kernels
    if _kernels is None:
        from brasa_amd import Kernels
        _kernels = Kernels()
    if "at" not in s:
        s["at"] = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
        a = s["at"]
        if s["op"] in ("rope", "store"):
            from brasa_amd import RopeAxes, RopeTable
            s["axes_of"] = RopeAxes.of_pairs(s["axis_of"])
            s["angles"] = RopeTable.view(a["cos"], a["sin"], s.get("dim", DIM), s["cos"].shape[0])
        if s["op"] in ("store", "attend"):
            from brasa_amd import KvPool, OutDType
            s["pool"] = KvPool.view(a["k"], a["v"], a["k_exp"], a["v_exp"], s.get("layers", 1), s["pages"],
                                    s["hkv"])
        if s["op"] == "attend":
            s["kind"] = OutDType.F32 if s["out"] == "f32" else OutDType.F16
            s["q_at"] = [x.data_ptr() for x in s["q"]]
            s["o_at"] = [x.data_ptr() for x in s["o"]]
    return _kernels, s["at"], torch.cuda.current_stream().cuda_stream


def run(s):
    op = s["op"]
    if op == "rows":
        if not own:
            return _rows_plain(s)
        lib, a, stream = _calls(s)
        n, width = s["n"], s["table"].shape[1]
        lib.kv_rows(a["add"], a["len"], a["table"], n, width, s["pages"], s["rows"], a["cu"], a["lk"],
                    a["seq"], a["pos"], a["slot"], stream)
        if s["groups"]:
            lib.kv_pages_shared(a["table"], a["len"], a["group"], s["groups"], n, width, s["pages"],
                                a["prefix_out"], stream)
        return {"cu": s["cu"], "lk": s["lk"], "seq": s["seq"], "pos": s["pos"], "slot": s["slot"],
                "prefix": s["prefix_out"]}
    if op == "rope":
        if own:
            lib, a, stream = _calls(s)
            lib.rope_axes(a["x"], s["angles"], s["axes_of"], a["rope_pos"], s["rows"], s["heads"], s["dim"], stream)
        else:
            s["x"].copy_(_rotated(s["x"], s, torch.float32))
        return s["x"]
    if op == "store":
        if own:
            lib, a, stream = _calls(s)
            lib.qk_norm_rope_store_paged(s["pool"], 0, (a["q_new"], a["k_new"], a["v_new"]),
                                         (a["q_norm"], a["k_norm"]), EPS, s["angles"], s["axes_of"], a["rope_pos"],
                                         a["cu"], a["pos"], a["table"], s["n"], s["table"].shape[1], s["rows"],
                                         s["hq"], stream)
        else:
            s["q_new"].copy_(_norm_rotated(s["q_new"], s["q_norm"], s))
            s["k_new"].copy_(_norm_rotated(s["k_new"], s["k_norm"], s))
            _store_plain(s, s["k_new"], s["k"][0], s["k_exp"][0])
            _store_plain(s, s["v_new"], s["v"][0], s["v_exp"][0])
        return {"q": s["q_new"], "k_new": s["k_new"], "k": s["k"].view(torch.float8_e4m3fn),
                "v": s["v"].view(torch.float8_e4m3fn), "k_exp": s["k_exp"], "v_exp": s["v_exp"]}
    if own:
        lib, a, stream = _calls(s)
        n, width, rows, hq = s["n"], s["table"].shape[1], s["rows"], s["hq"]
        size = s["work"].numel()
        lib.attention_paged_plan(a["cu"], a["pos"], a["group"], a["prefix"], s["groups"], n, width, rows, hq,
                                 s["hkv"], a["work"], size, stream)
        for layer in range(s["layers"]):
            lib.attention_paged(s["q_at"][layer], s["pool"], layer, a["table"], n, width, rows, a["work"], size,
                                s["o_at"][layer], hq, s["kind"], stream)
    else:
        for layer in range(s["layers"]):
            _attend_plain(s, layer)
    return s["o"]


# ---- what a pass cannot do without -------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "rope":
        values = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 8 * values + case["tokens"] * 4 * (case["dim"] + case["axes"]), "flops": 3 * values}
    n, new = case["n"], _new(case)
    if op == "rows":
        old = _held(case)
        # lengths in, table entries of the new rows' pages, maps out; the shared pages' entries
        # of every row of a group
        named = sum((a + b - 1) // PAGE - a // PAGE + 1 for a, b in zip(old, new) if b)
        entries = n * (case["prefix"] // PAGE + 1) if case["groups"] else 0
        return {"bytes": 4 * (4 * n + named + 3 * (sum(new) + case["behind"]) + entries), "flops": 0}
    hq, hkv, rows = case["hq"], case["hkv"], sum(new)
    if op == "store":
        # q and k in and out, v in, codes out, angles and positions in
        values = rows * DIM * (8 * hq + 8 * hkv + 4 * hkv + 2 * hkv)
        return {"bytes": values + rows * 4 * (DIM + case["axes"]) + 8 * n,
                "flops": rows * DIM * (8 * (hq + hkv) + 4 * hkv)}
    old, first = _held(case), _groups(case)
    row = 2 * hkv * DIM  # bytes of one position's K and V codes
    # each position's codes once: a group's prefix for all of its sequences together
    own_rows = sum(a + b - (case["prefix"] if first else 0) for a, b in zip(old, new) if b)
    once = sum(case["prefix"] for a, b in zip(first, first[1:]) if any(new[a:b]))
    out = 4 if case["out"] == "f32" else 2
    pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(old, new))
    return {"bytes": case["layers"] * ((own_rows + once) * row + rows * hq * DIM * (4 + out)),
            "flops": case["layers"] * 4 * hq * DIM * pairs}


# ---- the same in 64 bits -----------------------------------------------------------------------
def _e4m3(codes):
    """The values of e4m3 codes by their bits: sign, four exponent bits (bias 7), three of mantissa."""
    c = codes.int()
    exp, man = (c >> 3) & 15, (c & 7).double()
    x = torch.where(exp > 0, (1 + man / 8) * torch.exp2(exp.double() - 7), man / 8 * 2.0 ** -6)
    return torch.where(c >= 128, -x, x)


def _nearest(y):
    """The e4m3 value nearest to y (|y| <= 448), ties to the even mantissa, in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _turn64(x, rope_pos, axis_of, cos, sin):
    """Each pair (i, i + half) turned by the angle of its axis' position, one pair at a time."""
    half = x.shape[-1] // 2
    out = x.double().clone()
    live = (rope_pos >= 0).all(0)
    for i in range(half):
        at = rope_pos[axis_of[i]][live].long()
        c, s = cos[at, i].double()[:, None], sin[at, i].double()[:, None]
        a, b = x[live, :, i].double(), x[live, :, i + half].double()
        out[live, :, i], out[live, :, i + half] = a * c - b * s, a * s + b * c
    return out


def _store64(x, new, codes, exps):
    """new [rows, hkv, 128] in 64 bits, page by page."""
    cu, pos, table = x["cu"].tolist(), x["pos"].tolist(), x["table"].tolist()
    val, exps = _e4m3(codes), exps.clone()
    for i in range(len(pos)):
        p, end, src = pos[i], pos[i] + cu[i + 1] - cu[i], cu[i]
        while p < end:
            page, slot = table[i][p // PAGE], p % PAGE
            take = min(PAGE - slot, end - p)
            rows = new[src:src + take].double().transpose(0, 1)  # [hkv, take, 128]
            e = (torch.ceil(torch.log2(rows.abs().amax((1, 2)) / TOP)) + 127).clamp(min=0)
            if slot:
                was = exps[page].double()
                e = torch.maximum(e, was)
                val[page, :, :slot] = _nearest(val[page, :, :slot] * torch.exp2(was - e)[:, None, None])
            val[page, :, slot:slot + take] = _nearest(rows * torch.exp2(127 - e)[:, None, None])
            exps[page] = e.to(torch.uint8)
            p, src = p + take, src + take
    return val, exps


def exact(case, seed):
    op = case["op"]
    if op == "rows":
        return None  # whole numbers
    x = _inputs(case, seed)
    if op == "rope":
        axis_of = _axis_of(case["dim"] // 2, case["axes"], case["interleaved"])
        return _turn64(x["x"], x["rope_pos"], axis_of, x["cos"], x["sin"])
    if op == "store":
        axis_of = _axis_of(DIM // 2, case["axes"], case["interleaved"])
        got = {}
        for name, to in (("q", "q"), ("k", "k_new")):
            y = x[name + "_new"].double()
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / DIM + EPS) * x[name + "_norm"].double()
            got[to] = _turn64(y, x["rope_pos"], axis_of, x["cos"], x["sin"])
        for name, rows in (("k", got["k_new"]), ("v", x["v_new"])):
            val, e = _store64(x, rows, x[name][0], x[name + "_exp"][0])
            got[name], got[name + "_exp"] = val[None], e[None]
        return got
    hq, hkv = case["hq"], case["hkv"]
    out = torch.empty(case["layers"], x["rows"], hq, DIM, dtype=torch.float64, device="cuda")
    table, cu, old = x["table"].long(), x["cu"].tolist(), x["pos"].tolist()
    for layer in range(case["layers"]):
        for i, held in enumerate(old):
            a, b = cu[i], cu[i + 1]
            if a == b:
                continue
            keys = held + b - a
            ids = table[i, :-(-keys // PAGE)]
            k, v = ((_e4m3(x[c][layer, ids]) * torch.exp2(x[c + "_exp"][layer, ids].double() - 127)[..., None, None])
                    .transpose(0, 1).reshape(hkv, -1, DIM)[:, :keys] for c in ("k", "v"))
            later = torch.arange(keys, device="cuda")[None] - torch.arange(held, keys, device="cuda")[:, None] > 0
            for h in range(hq):
                score = x["q"][layer, a:b, h].double() @ k[h // (hq // hkv)].t() * DIM ** -0.5
                w = torch.softmax(score.masked_fill(later, -math.inf), -1)
                out[layer, a:b, h] = w @ v[h // (hq // hkv)]
    return out

"""The serving operators this library is measured on: causal attention over packed prompts, the
8-bit paged KV cache (its writer and the decode attention that reads it) and the pages' forking,
reserving and compaction.

``run`` computes each in plain torch where ``own`` is false and calls ``brasa_amd`` where it is
true. Head counts are the ones the benchmark and the tests use (32 query heads over 8 KV heads,
head_dim 128, and the other GQA groups the kernels are compiled for); keys are per-head
RMS-normed as behind QK-norm, values N(0, 1).

The paged cache: a page holds 64 positions of every KV head of one layer, K and V each as
[hkv, 64, 128] e4m3 codes with one power-of-two scale 2^(x - 127) per (page, head), x a byte. The
scale is the smallest with which the block's largest finite magnitude fits e4m3's 448; a block that
grows past it has its earlier codes rounded to the new scale.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DIM = 128
PAGE = 64
TOP = 448.0  # the largest e4m3 value


# ---- cases -------------------------------------------------------------------------------------
def listed():
    return [
        # a server's turn: a dozen chat prompts that arrived together, packed without padding
        {"name": "packed_chats", "op": "packed", "kv": "f16", "precision": "f16", "hq": 32,
         "hkv": 8, "lens": "311,45,128,64,97,501,23,1,260,77,333,190", "behind": 0},
        # long documents beside short prompts, one of them empty: the largest prompt pass
        {"name": "packed_documents", "op": "packed", "kv": "f16", "precision": "f16", "hq": 32,
         "hkv": 8, "lens": "8192,4100,0,2047,1025,511,1", "behind": 0},
        # the exact variant on exact rows, a few odd prompts in a buffer that is not full
        {"name": "packed_exact", "op": "packed", "kv": "f32", "precision": "f32", "hq": 16,
         "hkv": 8, "lens": "130,257,1,600", "behind": 29},
        # one layer's cache write of a decode step: a token for each of 64 sequences
        {"name": "store_step", "op": "store", "hkv": 8, "n": 64, "new_min": 1, "new_max": 1,
         "old_min": 100, "old_max": 8000, "lens": 1},
        # the cache write behind packed prompts, some of them after a cached prefix
        {"name": "store_prompts", "op": "store", "hkv": 8, "n": 12, "new_min": 40,
         "new_max": 2500, "old_min": 0, "old_max": 700, "lens": 2},
        # the first reply token of one short chat: bound by launch and latency
        {"name": "decode_short", "op": "decode", "hq": 32, "hkv": 8, "out": "f32", "n": 1,
         "lk_min": 257, "lk_max": 257, "layers": 1, "lens": 3},
        # one conversation at 16K positions, every layer of a model
        {"name": "decode_16k", "op": "decode", "hq": 32, "hkv": 8, "out": "f32", "n": 1,
         "lk_min": 16384, "lk_max": 16384, "layers": 36, "lens": 4},
        # a serving batch of ragged lengths: the largest decode pass of one layer
        {"name": "decode_batch", "op": "decode", "hq": 32, "hkv": 8, "out": "f16", "n": 64,
         "lk_min": 300, "lk_max": 16000, "layers": 1, "lens": 5},
        # four beams of one answer choose their parents, then make room for the next token
        {"name": "fork_beams", "op": "fork", "hkv": 8, "layers": 36, "n": 4, "len_min": 200,
         "len_max": 900, "keep": 25, "add": 1, "lens": 6},
        # a busy server's turn: some sequences end, others fork, and all reserve a few tokens
        {"name": "fork_batch", "op": "fork", "hkv": 8, "layers": 4, "n": 128, "len_min": 100,
         "len_max": 4000, "keep": 70, "add": 8, "lens": 7},
        # a small pool after a few sequences have ended
        {"name": "compact_small", "op": "compact", "hkv": 8, "layers": 4, "n": 8, "pages": 160,
         "len_min": 100, "len_max": 1500, "lens": 8},
        # a large pool, half of its pages free, before it is shrunk
        {"name": "compact_pool", "op": "compact", "hkv": 8, "layers": 12, "n": 48, "pages": 1000,
         "len_min": 100, "len_max": 2500, "lens": 9},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["packed", "packed", "store", "decode", "decode", "fork", "compact"])
    hq, hkv = rng.choice([(32, 8), (32, 8), (16, 8), (32, 4), (32, 32), (8, 8)])
    seed = rng.randrange(1 << 20)
    if op == "packed":
        kv, precision = rng.choice([("f16", "f16"), ("f16", "f16"), ("f16", "f16"),
                                    ("f16", "f16_pf32"), ("f16", "f32"), ("f32", "f32")])
        exact = precision == "f32"
        n, hi = _log(rng, 1, 24), _log(rng, 4, 1000 if exact else 6000)
        lens, left = [], 3000 if exact else 12000
        for _ in range(n):
            lens.append(min(left, _log(rng, 1, hi) if rng.random() < 0.95 else 0))
            left -= lens[-1]
        if not sum(lens):
            lens[0] = hi
        return {"op": op, "kv": kv, "precision": precision, "hq": hq, "hkv": hkv,
                "lens": ",".join(map(str, lens)), "behind": rng.choice([0, 0, _log(rng, 1, 100)])}
    if op == "store":
        n = _log(rng, 1, 128)
        step = rng.random() < 0.4
        return {"op": op, "hkv": hkv, "n": n, "new_min": 1,
                "new_max": rng.choice([1, 1, 4]) if step else _log(rng, 2, max(3, 12000 // n)),
                "old_min": 0, "old_max": _log(rng, 1, 200000 // n), "lens": seed}
    if op == "decode":
        n = _log(rng, 1, 200)
        layers = rng.choice([1, 1, 2, 12]) if n < 8 else 1
        hi = _log(rng, 2, max(3, min(32768, 2000000 // (n * layers * hkv))))
        return {"op": op, "hq": hq, "hkv": hkv, "out": rng.choice(["f32", "f16"]), "n": n,
                "lk_min": rng.choice([0, max(1, hi // 4), hi]), "lk_max": hi, "layers": layers,
                "lens": seed}
    if op == "fork":
        n = _log(rng, 2, 200)
        hi = _log(rng, 2, min(8000, 400000 // n))
        most = max(1, 100000 // (hkv * n * (hi // PAGE + 2)))
        return {"op": op, "hkv": hkv, "layers": min(most, rng.choice([1, 4, 12, 36])), "n": n,
                "len_min": 1, "len_max": hi, "keep": rng.randint(0, 100), "add": rng.choice([1, 1, 8, 100]),
                "lens": seed}
    n = _log(rng, 1, 64)
    hi = _log(rng, 2, min(4000, 100000 // n))
    return {"op": op, "hkv": hkv, "layers": rng.choice([1, 4, 12]), "n": n,
            "pages": n * (hi // PAGE + 1) + _log(rng, 8, 400), "len_min": 1, "len_max": hi,
            "lens": seed}


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


def _parents(case):
    """Which row each row of the next step continues; -1: its sequence has ended."""
    r, n = random.Random(case["lens"] * 7 + 2), case["n"]
    return [i if 100 * r.random() < case["keep"] else r.randrange(-1, n) for i in range(n)]


def _normed(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


def _blocks(lens):
    return [-(-n // PAGE) for n in lens]


def _scatter_pages(g, counts, pages, width):
    """A table [n, width] whose rows take their pages from all over the pool; -1 where none."""
    ids = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = ids[at:at + c]
        at += c
    return table


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
            c = _codes(x, e[..., None, None])
            codes[i, a:a + 2048], exps[i, a:a + 2048] = c, e.to(torch.uint8)
    return codes, exps


def _raw_pool(g, layers, pages, hkv):
    """Bytes of a pool whose values do not matter."""
    shape = layers, pages, hkv
    return [torch.randint(0, 120, (*shape, PAGE, DIM), generator=g, device="cuda", dtype=torch.uint8),
            torch.randint(100, 140, shape, generator=g, device="cuda", dtype=torch.uint8)]


def _ref(table, pages):
    used = table[table >= 0].long()
    return torch.bincount(used, minlength=pages).to(torch.int32)


def _inputs(case, seed):
    """What the case reads, from the seed alone."""
    g, op = _gen(seed), case["op"]
    if op == "packed":
        lens = [int(x) for x in case["lens"].split(",")]
        hq, hkv, rows = case["hq"], case["hkv"], sum(lens) + case["behind"]
        starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
        kind = torch.float16 if case["kv"] == "f16" else torch.float32
        return {"q": _normed(torch.randn(rows, hq, DIM, generator=g, device="cuda")),
                "k": _normed(torch.randn(rows, hkv, DIM, generator=g, device="cuda")).to(kind),
                "v": torch.randn(rows, hkv, DIM, generator=g, device="cuda").to(kind),
                "cu": _ints(starts), "n": len(lens), "rows": rows}
    n, hkv = case["n"], case["hkv"]
    if op == "store":
        new, old = _lens(case, "new_min", "new_max"), _lens(case, "old_min", "old_max", 1)
        rows = sum(new)
        counts = _blocks([a + b for a, b in zip(new, old)])
        pages = sum(counts) + 16
        width = max(counts)
        k, ke = _pool(g, 1, pages, hkv, "k")
        v, ve = _pool(g, 1, pages, hkv, "v")
        # a new token's head may be larger than all before it
        up = 2.0 ** torch.randint(-1, 3, (rows, hkv, 1), generator=g, device="cuda")
        return {"k_new": _normed(torch.randn(rows, hkv, DIM, generator=g, device="cuda")) * up,
                "v_new": torch.randn(rows, hkv, DIM, generator=g, device="cuda") * up,
                "cu": _ints([sum(new[:i]) for i in range(n + 1)]), "pos": _ints(old),
                "table": _scatter_pages(g, counts, pages, width), "pages": pages, "width": width,
                "rows": rows, "k": k, "v": v, "k_exp": ke, "v_exp": ve, "layers": 1}
    if op == "decode":
        lens = _lens(case, "lk_min", "lk_max")
        counts = _blocks(lens)
        pages, width = sum(counts) + 4, max(max(counts), 1)
        k, ke = _pool(g, case["layers"], pages, hkv, "k")
        v, ve = _pool(g, case["layers"], pages, hkv, "v")
        q = torch.randn(case["layers"], n, case["hq"], DIM, generator=g, device="cuda")
        return {"q": _normed(q), "lk": _ints(lens), "table": _scatter_pages(g, counts, pages, width),
                "pages": pages, "width": width, "k": k, "v": v, "k_exp": ke, "v_exp": ve}
    lens = _lens(case, "len_min", "len_max")
    if op == "fork":
        width = max(_blocks([x + case["add"] for x in lens]))
        # room for every sequence's own pages, and for as many again
        pages = 2 * sum(_blocks(lens)) + n * (case["add"] // PAGE + 2)
        x = {"parent": _ints(_parents(case)),
             "add": torch.full((n,), case["add"], dtype=torch.int32, device="cuda")}
    else:
        width, pages, x = max(_blocks(lens)), case["pages"], {}
    table = _scatter_pages(g, _blocks(lens), pages, width)
    (k, ke), (v, ve) = _raw_pool(g, case["layers"], pages, hkv), _raw_pool(g, case["layers"], pages, hkv)
    x.update({"len": _ints(lens), "table": table, "ref": _ref(table, pages), "pages": pages,
              "width": width, "k": k, "v": v, "k_exp": ke, "v_exp": ve})
    return x


def prepare(case, seed):
    s = dict(case, **_inputs(case, seed))
    op, n = s["op"], s["n"]
    if op == "packed":
        s["o"] = torch.zeros(s["rows"], s["hq"], DIM, device="cuda",
                             dtype=torch.float32 if s["precision"] == "f32" else torch.float16)
    elif op == "decode":
        s["o"] = torch.zeros(s["layers"], n, s["hq"], DIM, device="cuda",
                             dtype=torch.float32 if s["out"] == "f32" else torch.float16)
        # the split's scratch, cleared once: 64 MB hold that of the largest batch here
        s["work"] = torch.zeros(1 << 26, dtype=torch.uint8, device="cuda")
    elif op != "store":
        s["table_out"], s["ref_out"] = torch.empty_like(s["table"]), torch.empty_like(s["ref"])
        s["work"] = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
        s["status"] = torch.zeros(2, dtype=torch.int32, device="cuda")
        if op == "fork":
            s["table_mid"], s["ref_mid"] = torch.empty_like(s["table"]), torch.empty_like(s["ref"])
            s["len_out"] = torch.empty_like(s["len"])
    return s


# ---- the plain forms ---------------------------------------------------------------------------
def _exponent(amax):
    """The scale byte of blocks by their largest finite magnitude: the least x >= 0 with
    amax <= 448 * 2^(x - 127). Whole numbers of the magnitude's bits, so no rounding is near."""
    bits = amax.view(torch.int32)
    # a mantissa over 1.75 (448 = 1.75 * 2^8) takes the next power of two
    return ((bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000).int()).clamp_(min=0)


def _pow2(exps):
    """2^(x - 127) of scale bytes, exact."""
    return torch.ldexp(torch.ones((), device="cuda"), exps.int() - 127)


def _codes(x, exps):
    """x / 2^(exps - 127) rounded to e4m3 (exact up to that rounding), as bytes."""
    # in two steps, as 2^(127 - exps) itself may leave the range
    half = (127 - exps.int()) // 2
    y = torch.ldexp(torch.ldexp(x, half), 127 - exps.int() - half)
    return y.to(torch.float8_e4m3fn).view(torch.uint8)


def _values(codes, exps):
    return codes.view(torch.float8_e4m3fn).float() * _pow2(exps)[..., None, None]


def _packed_plain(s):
    rows, hq, hkv = s["rows"], s["hq"], s["hkv"]
    group = hq // hkv
    row = torch.arange(rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["cu"], row, right=True)  # n + 1 behind the last sequence
    hidden = (seq[:, None] != seq[None]) | (row[None] > row[:, None])
    inside = (row < s["cu"][-1])[:, None, None]
    out = torch.empty(rows, hq, DIM, device="cuda")
    for h in range(hkv):  # one KV head's scores at a time
        q = s["q"][:, h * group:(h + 1) * group].transpose(0, 1)
        p = (q / math.sqrt(DIM)) @ s["k"][:, h].float().t()
        p.masked_fill_(hidden, -math.inf)
        p.sub_(p.amax(-1, keepdim=True)).exp_()
        o = (p @ s["v"][:, h].float()) / p.sum(-1, keepdim=True)
        out[:, h * group:(h + 1) * group] = o.transpose(0, 1)
    return torch.where(inside, out.to(s["o"].dtype), s["o"])


def _store_plain(s, new, codes, exps):
    """One of K and V: `new` [rows, hkv, 128] into the pages, in place."""
    rows, n, hkv = s["rows"], s["n"], s["hkv"]
    row = torch.arange(rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["cu"], row, right=True) - 1
    pos = s["pos"][seq] + row - s["cu"][seq]
    page = s["table"][seq, pos // PAGE].long()
    # the largest magnitude of each block's new rows
    most = torch.zeros(s["pages"], hkv, device="cuda")
    most.scatter_reduce_(0, page[:, None].expand(-1, hkv), new.abs().amax(-1), "amax")
    # a block whose first rows were there before keeps their scale as a lower bound
    fresh = torch.ones(s["pages"] + 1, dtype=torch.bool, device="cuda")
    held = s["pos"] % PAGE
    grows = (held > 0) & (s["cu"][1:] > s["cu"][:-1])
    first = s["table"].gather(1, (s["pos"] // PAGE).clamp(max=s["width"] - 1).long()[:, None])[:, 0].long()
    first = torch.where(grows, first, s["pages"])
    fresh[first] = False
    touched = torch.zeros(s["pages"], dtype=torch.bool, device="cuda")
    touched[page] = True
    e = _exponent(most)
    e = torch.where(fresh[:-1, None], e, torch.maximum(e, exps.int()))
    e = torch.where(touched[:, None], e, exps.int())
    # the earlier rows of those blocks, to the new scale
    at = first.clamp(max=s["pages"] - 1)
    old = codes[at]
    again = _codes(old.view(torch.float8_e4m3fn).float(), (127 + e[at] - exps[at].int())[..., None, None])
    slot = torch.arange(PAGE, device="cuda")[None, None, :, None]
    again = torch.where(slot < held[:, None, None, None], again, old)
    codes[at[grows]] = again[grows]
    exps.copy_(e)
    codes[page, :, pos % PAGE] = _codes(new, e[page][..., None])


def _decode_plain(s, layer):
    n, hq, hkv, width = s["n"], s["hq"], s["hkv"], s["width"]
    at = s["table"].clamp(min=0).long()

    def rows(codes, exps):
        x = _values(codes[layer][at], exps[layer][at])  # [n, blocks, hkv, 64, 128]
        return x.permute(0, 2, 1, 3, 4).reshape(n, hkv, width * PAGE, DIM)

    live = torch.arange(width * PAGE, device="cuda")[None] < s["lk"][:, None]
    q = s["q"][layer].reshape(n, hkv, hq // hkv, DIM) / math.sqrt(DIM)
    p = q @ rows(s["k"], s["k_exp"]).transpose(-1, -2)
    p.masked_fill_(~live[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    o = (p @ rows(s["v"], s["v_exp"])) / p.sum(-1, keepdim=True)
    o = torch.where((s["lk"] > 0)[:, None, None, None], o, 0.0)  # no keys: zeros
    s["o"][layer] = o.reshape(n, hq, DIM)


def _fork_plain(s):
    """Row i takes the pages of row parent[i] (none: -1); pages count their rows."""
    pages, none = s["pages"], s["parent"] < 0
    at = s["parent"].clamp(min=0).long()
    table = torch.where(none[:, None], -1, s["table"][at])
    length = torch.where(none, 0, s["len"][at])
    ref = torch.cat([s["ref"], s["ref"].new_zeros(1)])
    one = torch.ones((), dtype=torch.int32, device="cuda").expand(table.numel())
    ref.scatter_add_(0, torch.where(table < 0, pages, table).reshape(-1).long(), one)
    ref.scatter_add_(0, torch.where(s["table"] < 0, pages, s["table"]).reshape(-1).long(), -one)
    return table, length, ref[:-1]


def _reserve_plain(s, table, length, ref):
    """Positions [len, len + add) of every row get pages of their own: new ones, the lowest free
    ids in order, where there is none or it is shared; the rows a shared page held are copied. When
    every owner of a page wants it, the first keeps it."""
    n, width, pages = s["n"], s["width"], s["pages"]
    col = torch.arange(width, device="cuda", dtype=torch.int32)[None]
    first = length // PAGE
    wants = (col >= first[:, None]) & (col * PAGE < (length + s["add"])[:, None])
    flat = torch.where(wants & (table >= 0), table, pages).reshape(-1).long()
    one = torch.ones((), dtype=torch.int32, device="cuda").expand(flat.numel())
    count = ref.new_zeros(pages + 1).scatter_add_(0, flat, one)
    order = torch.arange(flat.numel(), device="cuda", dtype=torch.int32)
    lowest = torch.full_like(count, flat.numel()).scatter_reduce_(0, flat, order, "amin")
    kept = (torch.cat([ref, ref.new_zeros(1)])[flat] <= count[flat]) & (lowest[flat] == order) & (flat < pages)
    takes = wants.reshape(-1) & ~kept
    rank = torch.cumsum(takes, 0) - 1
    free = torch.argsort((ref > 0).to(torch.uint8), stable=True)
    fits = takes.sum() <= (ref == 0).sum()
    got = free[rank.clamp(min=0, max=pages - 1)].int()
    takes = takes & fits
    out = torch.where(takes, got, table.reshape(-1)).reshape(n, width)
    after = torch.cat([ref, ref.new_zeros(1)])
    after.scatter_add_(0, torch.where(takes, flat, pages), -one)
    after.scatter_add_(0, torch.where(takes, got, pages).long(), one)
    # the rows of a partly filled page that moved
    col = first.clamp(max=width - 1).long()[:, None]
    src, dst = table.gather(1, col)[:, 0], out.gather(1, col)[:, 0]
    moved = (src >= 0) & (src != dst) & (length % PAGE > 0)
    src, dst, held = src[moved].long(), dst[moved].long(), (length % PAGE)[moved]
    live = (torch.arange(PAGE, device="cuda")[None] < held[:, None])[None, :, None, :, None]
    for name in ("k", "v"):
        s[name][:, dst] = torch.where(live, s[name][:, src], s[name][:, dst])
        s[name + "_exp"][:, dst] = s[name + "_exp"][:, src]
    taken = rank[-1:].int() + 1
    free_pages = (ref == 0).sum().int()
    status = torch.cat([torch.where(fits, taken, 0), (taken - free_pages).clamp(min=0)])
    return out, after[:-1], status


def _compact_plain(s):
    """The pages in use, moved so that they are the first ones: the k-th page in use at or past
    their number moves to the k-th free one below it."""
    pages, ref = s["pages"], s["ref"]
    ids = torch.arange(pages, device="cuda", dtype=torch.int32)
    live = ref > 0
    count = live.sum()
    src, dst = ids[live & (ids >= count)].long(), ids[~live & (ids < count)].long()
    to = ids.clone()
    to[src] = dst.int()
    table = torch.where(s["table"] < 0, s["table"], to[s["table"].clamp(min=0).long()])
    after = ref.clone()
    after[dst], after[src] = ref[src], 0
    for name in ("k", "v", "k_exp", "v_exp"):
        s[name][:, dst] = s[name][:, src]
    return table, after, count.int()[None]


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
        if s["op"] == "packed":
            from brasa_amd import AttnShape, KvType, PrefillPrecision
            kv = KvType.F16 if s["kv"] == "f16" else KvType.F32
            s["shape"] = AttnShape(s["rows"], s["hq"], s["hkv"], DIM, 0, kv)
            s["prec"] = {"f16": PrefillPrecision.F16, "f16_pf32": PrefillPrecision.F16_PF32,
                         "f32": PrefillPrecision.F32}[s["precision"]]
        else:
            from brasa_amd import KvPool, OutDType
            a = s["at"]
            s["pool"] = KvPool.view(a["k"], a["v"], a["k_exp"], a["v_exp"], s["layers"], s["pages"],
                                    s["hkv"])
            if s["op"] == "decode":
                s["kind"] = OutDType.F32 if s["out"] == "f32" else OutDType.F16
                s["q_at"] = [x.data_ptr() for x in s["q"]]
                s["o_at"] = [x.data_ptr() for x in s["o"]]
    return _kernels, s["at"], torch.cuda.current_stream().cuda_stream


def run(s):
    op, n = s["op"], s["n"]
    if op == "packed":
        if own:
            lib, a, stream = _calls(s)
            lib.flash_attention_packed(a["q"], a["k"], a["v"], a["o"], a["cu"], n, s["shape"],
                                       s["prec"], stream)
            return s["o"]
        return _packed_plain(s)
    if op == "store":
        if own:
            lib, a, stream = _calls(s)
            lib.store_kv_paged(s["pool"], 0, a["k_new"], a["v_new"], a["cu"], a["pos"], a["table"],
                               n, s["width"], s["rows"], stream)
        else:
            _store_plain(s, s["k_new"], s["k"][0], s["k_exp"][0])
            _store_plain(s, s["v_new"], s["v"][0], s["v_exp"][0])
        return {"k": s["k"].view(torch.float8_e4m3fn), "v": s["v"].view(torch.float8_e4m3fn),
                "k_exp": s["k_exp"], "v_exp": s["v_exp"]}
    if op == "decode":
        if own:
            lib, a, stream = _calls(s)
            for layer in range(s["layers"]):
                lib.decode_attention_paged(s["q_at"][layer], s["pool"], layer, a["table"], a["lk"], n,
                                           s["width"], a["work"], s["work"].numel(), s["o_at"][layer],
                                           s["hq"], s["kind"], stream)
        else:
            for layer in range(s["layers"]):
                _decode_plain(s, layer)
        return s["o"]
    pool = {"k": s["k"], "v": s["v"], "k_exp": s["k_exp"], "v_exp": s["v_exp"]}
    if op == "fork":
        if own:
            lib, a, stream = _calls(s)
            lib.kv_pages_fork(a["parent"], a["table"], a["len"], a["ref"], a["table_mid"],
                              a["len_out"], a["ref_mid"], n, s["width"], s["pages"], stream)
            lib.kv_pages_reserve(s["pool"], a["add"], a["table_mid"], a["len_out"], a["ref_mid"],
                                 a["table_out"], a["ref_out"], a["status"], n, s["width"],
                                 a["work"], s["work"].numel(), stream)
            return dict(pool, table=s["table_out"], len=s["len_out"], ref=s["ref_out"],
                        status=s["status"])
        table, length, ref = _fork_plain(s)
        table, ref, status = _reserve_plain(s, table, length, ref)
        return dict(pool, table=table, len=length, ref=ref, status=status)
    if own:
        lib, a, stream = _calls(s)
        lib.kv_pages_compact(s["pool"], a["table"], a["ref"], a["table_out"], a["ref_out"],
                             a["status"], n, s["width"], a["work"], s["work"].numel(), stream)
        return dict(pool, table=s["table_out"], ref=s["ref_out"], live=s["status"][:1])
    table, ref, live = _compact_plain(s)
    return dict(pool, table=table, ref=ref, live=live)


# ---- what a pass cannot do without -------------------------------------------------------------
def work(case):
    op, hkv = case["op"], case["hkv"]
    row = 2 * hkv * DIM  # bytes of one position's K and V codes
    if op == "packed":
        lens, hq = [int(x) for x in case["lens"].split(",")], case["hq"]
        out = 4 if case["precision"] == "f32" else 2
        rows = sum(lens) * DIM
        return {"bytes": rows * (hq * (4 + out) + 2 * hkv * (2 if case["kv"] == "f16" else 4)),
                "flops": sum(4 * hq * DIM * x * (x + 1) / 2 for x in lens)}
    if op == "store":
        new = _lens(case, "new_min", "new_max")
        return {"bytes": sum(new) * row * 5 + case["n"] * 8 * hkv, "flops": 4 * sum(new) * row}
    if op == "decode":
        lens = _lens(case, "lk_min", "lk_max")
        out = 4 if case["out"] == "f32" else 2
        one = sum(lens) * row + sum(_blocks(lens)) * (2 * hkv + 4) + case["n"] * case["hq"] * DIM * (4 + out)
        return {"bytes": case["layers"] * one,
                "flops": case["layers"] * 4 * case["hq"] * DIM * sum(lens)}
    lens = _lens(case, "len_min", "len_max")
    if op == "fork":
        # tables and counts once in and out for each of the two calls; the rows of the partly
        # filled pages that are copied, in and out (a row that keeps its own needs none)
        pages = 2 * sum(_blocks(lens)) + case["n"] * (case["add"] // PAGE + 2)
        width = max(_blocks([x + case["add"] for x in lens]))
        parents = _parents(case)
        moved = sum(x % PAGE * max(0, parents.count(i) - 1) for i, x in enumerate(lens))
        return {"bytes": 4 * 4 * (case["n"] * width + pages) + 2 * moved * row * case["layers"],
                "flops": 0}
    used = sum(_blocks(lens))
    # of the pages in use, the share past their number moves
    moved = used * (case["pages"] - used) // case["pages"]
    return {"bytes": 2 * moved * PAGE * row * case["layers"] + 8 * case["pages"]
            + 8 * case["n"] * max(_blocks(lens)), "flops": 0}


# ---- the same in 64 bits -----------------------------------------------------------------------
def _attend64(q, k, v, causal):
    """q [t, g, 128] over k, v [t or lk, 128] of its KV head, in 64 bits."""
    s = torch.einsum("tgd,kd->gtk", q.double(), k.double()) * DIM ** -0.5
    if causal:
        s = s + torch.triu(torch.full(s.shape[1:], -math.inf, dtype=s.dtype, device="cuda"), 1)
    return torch.einsum("gtk,kd->tgd", torch.softmax(s, -1), v.double())


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


def _store64(x, new, codes, exps):
    cu, pos, table = x["cu"].tolist(), x["pos"].tolist(), x["table"].tolist()
    val, exps = _e4m3(codes), exps.clone()
    for i in range(len(pos)):
        p, end, src = pos[i], pos[i] + cu[i + 1] - cu[i], cu[i]
        while p < end:
            page, slot = table[i][p // PAGE], p % PAGE
            take = min(PAGE - slot, end - p)
            rows = new[src:src + take].double().transpose(0, 1)  # [hkv, take, 128]
            top = rows.abs().amax((1, 2))
            e = torch.ceil(torch.log2(top / TOP)) + 127
            e = e.clamp(min=0)
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
    if op in ("fork", "compact"):
        return None  # whole numbers and bytes that are moved
    x = _inputs(case, seed)
    hkv = case["hkv"]
    if op == "packed":
        group = case["hq"] // hkv
        out = torch.zeros(x["rows"], case["hq"], DIM, dtype=torch.float64, device="cuda")
        cu = x["cu"].tolist()
        for a, b in zip(cu, cu[1:]):
            for h in range(hkv):
                for j in range(h * group, (h + 1) * group):
                    out[a:b, j:j + 1] = _attend64(x["q"][a:b, j:j + 1], x["k"][a:b, h], x["v"][a:b, h], True)
        return out
    if op == "store":
        got = {}
        for name in ("k", "v"):
            val, e = _store64(x, x[name + "_new"], x[name][0], x[name + "_exp"][0])
            got[name], got[name + "_exp"] = val[None], e[None]
        return got
    group = case["hq"] // hkv
    out = torch.empty(case["layers"], case["n"], case["hq"], DIM, dtype=torch.float64, device="cuda")
    lens, table = x["lk"].tolist(), x["table"].long()
    for layer in range(case["layers"]):
        for i, lk in enumerate(lens):
            if lk == 0:
                out[layer, i] = 0
                continue
            ids = table[i, :-(-lk // PAGE)]
            kv = [(_e4m3(x[c][layer, ids]) * torch.exp2(x[c + "_exp"][layer, ids].double() - 127)[..., None, None])
                  .transpose(0, 1).reshape(hkv, -1, DIM)[:, :lk] for c in ("k", "v")]
            for h in range(hkv):
                q = x["q"][layer, i:i + 1, h * group:(h + 1) * group]
                out[layer, i, h * group:(h + 1) * group] = _attend64(q, kv[0][h], kv[1][h], False)[0]
    return out

"""The packed and paged operators in plain numpy, 64 bits, one step after another: what the GPU
tests compare with. Codes are e4m3 bytes, a page of a head is [64, 128], tables and counts int32."""
from __future__ import annotations

import numpy as np

DIM, PAGE = 128, 64


def _table():
    c = np.arange(256)
    e, m = (c >> 3) & 15, (c & 7).astype(np.float64)
    x = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7.0), m / 8 * 2.0 ** -6)
    x = np.where((c & 127) == 127, np.nan, x)
    return np.where(c >= 128, -x, x)


E4M3 = _table()
_POS = E4M3[:127]  # 0 .. 448, ascending


def encode(y: np.ndarray) -> np.ndarray:
    """e4m3 bytes nearest to y (ties to the even code; NaN where y is not finite)."""
    y = np.asarray(y, np.float64)
    a = np.abs(np.where(np.isfinite(y), y, 0.0))
    hi = np.clip(np.searchsorted(_POS, a), 1, 126)
    lo = hi - 1
    up, down = _POS[hi] - a, a - _POS[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo).astype(np.uint8)
    code = np.where(np.isfinite(y), code, 127).astype(np.uint8)
    return code | (np.signbit(y).astype(np.uint8) << 7)


def scale_byte(amax: float) -> int:
    """The least x >= 0 with amax <= 448 * 2^(x - 127)."""
    x = 0
    while amax > 448.0 * 2.0 ** (x - 127):
        x += 1
    return x


class Pool:
    """Host side of a pool: k, v [layers, pages, hkv, 64, 128] codes, k_exp, v_exp scale bytes."""

    def __init__(self, layers, pages, hkv, rng=None):
        shape = (layers, pages, hkv)
        draw = (lambda s, n: rng.integers(0, n, s).astype(np.uint8)) if rng is not None else \
               (lambda s, n: np.zeros(s, np.uint8))
        self.k, self.v = draw((*shape, PAGE, DIM), 256), draw((*shape, PAGE, DIM), 256)
        self.k_exp, self.v_exp = draw(shape, 200), draw(shape, 200)
        self.layers, self.pages, self.hkv = shape

    def arrays(self):
        return self.k, self.v, self.k_exp, self.v_exp


def store(pool: Pool, layer, k, v, cu, pos, table):
    """k, v [rows, hkv, 128] f32 into the pages, in place."""
    width = table.shape[1]
    for i in range(len(pos)):
        p, src, end = int(pos[i]), int(cu[i]), int(cu[i + 1])
        if p < 0:
            continue
        while src < end and p < width * PAGE:
            slot = p % PAGE
            take = min(PAGE - slot, end - src)
            page = int(table[i, p // PAGE])
            if 0 <= page < pool.pages:
                for rows, codes, exps in ((k, pool.k, pool.k_exp), (v, pool.v, pool.v_exp)):
                    for h in range(pool.hkv):
                        x = rows[src:src + take, h].astype(np.float64)
                        tile = codes[layer, page, h]
                        e = scale_byte(np.abs(x[np.isfinite(x)]).max(initial=0.0))
                        if slot:
                            old = int(exps[layer, page, h])
                            if e > old:
                                tile[:slot] = encode(E4M3[tile[:slot]] * 2.0 ** (old - e))
                            e = max(e, old)
                        tile[slot:slot + take] = encode(x * 2.0 ** (127 - e))
                        exps[layer, page, h] = e
            p, src = p + take, src + take


def rows_of(pool: Pool, layer, ids, lk):
    """K and V of a sequence in 64 bits: [lk, hkv, 128] each."""
    out = []
    for codes, exps in ((pool.k, pool.k_exp), (pool.v, pool.v_exp)):
        x = E4M3[codes[layer, ids]] * 2.0 ** (exps[layer, ids].astype(np.float64) - 127)[..., None, None]
        out.append(x.transpose(0, 2, 1, 3).reshape(-1, pool.hkv, DIM)[:lk])
    return out


def attend(q, k, v, causal):
    """q [t, hq, 128] over k, v [lk, hkv, 128]. Returns o, the weighted sum of |v| (what errors of the
    weights are relative to) and the largest sum of |q k| / sqrt(128) of each row (what errors
    of the scores are relative to), all [t, hq, 128] or [t, hq, 1]."""
    t, hq, _ = q.shape
    lk, hkv, _ = k.shape
    o, av = np.zeros((t, hq, DIM)), np.zeros((t, hq, DIM))
    top = np.zeros((t, hq, 1))
    if lk == 0:
        return o, av, top
    hidden = np.arange(lk)[None] > np.arange(t)[:, None] if causal else np.zeros((t, lk), bool)
    for h in range(hq):
        kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        qh = q[:, h].astype(np.float64)
        with np.errstate(over="ignore", invalid="ignore"):
            s = np.where(hidden, -np.inf, qh @ kh.T / np.sqrt(DIM))
            a = np.where(hidden, 0.0, np.abs(qh) @ np.abs(kh).T / np.sqrt(DIM))
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            o[:, h], av[:, h] = p @ vh, p @ np.abs(vh)
        top[:, h, 0] = a.max(-1)
    return o, av, top


def fork(parent, table, lens, ref):
    n, pages = len(parent), len(ref)
    table2, lens2, ref2 = np.full_like(table, -1), np.zeros_like(lens), ref.copy()
    for i in range(n):
        if 0 <= parent[i] < n:
            table2[i], lens2[i] = table[parent[i]], lens[parent[i]]
    for t, d in ((table, -1), (table2, 1)):
        ids = t[(t >= 0) & (t < pages)]
        np.add.at(ref2, ids, d)
    return table2, lens2, ref2


def reserve(pool, add, table, lens, ref):
    """One claim after another. Returns table, ref, status; pool is changed in place."""
    n, width = table.shape
    claims = []
    for i in range(n):
        if add[i] > 0:
            if max(lens[i], 0) + add[i] > width * PAGE:
                return table.copy(), ref.copy(), np.array([0, -1], np.int32)
            for b in range(lens[i] // PAGE, -(-(lens[i] + add[i]) // PAGE)):
                claims.append((i, b))
    held = {}
    for i, b in claims:
        held.setdefault(int(table[i, b]), []).append((i, b))
    takes = []
    for c in claims:
        e = int(table[c])
        if e < 0 or not (len(held[e]) >= ref[e] and held[e][0] == c):
            takes.append(c)
    free = np.flatnonzero(ref <= 0)
    if len(takes) > len(free):
        return table.copy(), ref.copy(), np.array([0, len(takes) - len(free)], np.int32)
    table2, ref2 = table.copy(), ref.copy()
    for (i, b), page in zip(takes, free):
        e = int(table[i, b])
        ref2[page] = 1
        table2[i, b] = page
        if e >= 0:
            ref2[e] -= 1
            live = lens[i] - b * PAGE
            if live > 0:
                for codes, exps in ((pool.k, pool.k_exp), (pool.v, pool.v_exp)):
                    codes[:, page, :, :live] = codes[:, e, :, :live]
                    exps[:, page] = exps[:, e]
    return table2, ref2, np.array([len(takes), 0], np.int32)


def compact(pool, table, ref):
    live = int((ref > 0).sum())
    src = [p for p in range(len(ref)) if ref[p] > 0 and p >= live]
    dst = [p for p in range(live) if ref[p] <= 0]
    to, ref2 = np.arange(len(ref), dtype=np.int32), ref.copy()
    for s, d in zip(src, dst):
        to[s], ref2[d], ref2[s] = d, ref[s], 0
        for a in pool.arrays():
            a[:, d] = a[:, s]
    table2 = np.where((table >= 0) & (table < len(ref)), to[np.clip(table, 0, len(ref) - 1)], table)
    return table2.astype(np.int32), ref2, live

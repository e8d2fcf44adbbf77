"""The maps of a step's rows, rotary axes and attention of new rows over the paged cache in plain
numpy, 64 bits: what the GPU tests compare with."""
from __future__ import annotations

import numpy as np

import paged_ref as ref

DIM, PAGE = ref.DIM, ref.PAGE


def raised(x, top):
    """Bounds clamped to [0, top] and raised to the largest before them."""
    return np.maximum.accumulate(np.clip(np.asarray(x, np.int64), 0, top))


def rows(add, lens, table, pages, tokens):
    """cu, lk, seq, pos, slot, one row after another."""
    n, width = table.shape
    cu, lk = np.zeros(n + 1, np.int32), np.zeros(n, np.int32)
    seq, pos, slot = (np.full(tokens, -1, np.int32) for _ in range(3))
    t = 0
    for i in range(n):
        cu[i] = t
        if lens[i] >= 0:
            for j in range(min(max(int(add[i]), 0), tokens - t)):
                p = int(lens[i]) + j
                seq[t], pos[t] = i, min(p, 2 ** 31 - 1)
                if p // PAGE < width and 0 <= table[i, p // PAGE] < pages:
                    slot[t] = table[i, p // PAGE] * PAGE + p % PAGE
                t += 1
        lk[i] = min(max(int(lens[i]), 0) + t - int(cu[i]), 2 ** 31 - 1)
    cu[n] = t
    return cu, lk, seq, pos, slot


def shared(table, lens, group, pages):
    out = []
    bounds = np.clip(group, 0, len(lens))
    for a, b in zip(bounds, bounds[1:]):
        live = [i for i in range(a, b) if lens[i] > 0]
        c = 0
        if len(live) > 1:
            lead = table[live[0]]
            while c < table.shape[1] and 0 <= lead[c] < pages and \
                    all(table[i, c] == lead[c] and lens[i] >= (c + 1) * PAGE for i in live):
                c += 1
        out.append(c * PAGE)
    return np.array(out, np.int32)


def rope(x, cos, sin, of, pos):
    """x [rows, heads, dim] in 64 bits; pos [axes, rows]; rows at a negative position as they are."""
    half = x.shape[-1] // 2
    y = x.astype(np.float64)
    for t in range(len(x)):
        if (pos[:, t] < 0).any():
            continue
        if (pos[:, t] >= len(cos)).any():
            y[t] = np.nan
            continue
        c = np.array([cos[pos[of[i], t], i] for i in range(half)], np.float64)
        s = np.array([sin[pos[of[i], t], i] for i in range(half)], np.float64)
        a, b = y[t, :, :half].copy(), y[t, :, half:].copy()
        y[t, :, :half], y[t, :, half:] = a * c - b * s, b * c + a * s
    return y


def attend(q, k, v, held):
    """q [t, hq, 128], row r at position held + r, over k, v [held + t, hkv, 128]. Returns o, the weighted sum
    of |v|, and the largest sum of |q k| / sqrt(128) of each row, as paged_ref.attend does. Values that a
    row does not see never reach it."""
    t, hq, _ = q.shape
    hkv = k.shape[1]
    o, av, top = np.zeros((t, hq, DIM)), np.zeros((t, hq, DIM)), np.zeros((t, hq, 1))
    finite = np.isfinite(v).all()
    for h in range(hq):
        kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        qh = q[:, h].astype(np.float64)
        with np.errstate(over="ignore", invalid="ignore"):
            hidden = np.arange(held + t)[None] > np.arange(held, held + t)[:, None]
            s = np.where(hidden, -np.inf, qh @ kh.T / np.sqrt(DIM))
            a = np.where(hidden, 0.0, np.abs(qh) @ np.abs(kh).T / np.sqrt(DIM))
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            if finite:
                o[:, h], av[:, h] = p @ vh, p @ np.abs(vh)
            else:
                for r in range(t):
                    o[r, h], av[r, h] = p[r, :held + r + 1] @ vh[:held + r + 1], p[r, :held + r + 1] @ np.abs(vh[:held + r + 1])
        top[:, h, 0] = a.max(-1)
    return o, av, top

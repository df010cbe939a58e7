"""Plain numpy statements, in 64 bits, of the paged cache's operators: what their tests check against."""

from __future__ import annotations

import numpy as np


def extend(tables, lengths, free, count, page, counts, tokens):
    """Slots, positions, sequences and served, and the tables, lengths and count afterwards."""
    tables, lengths = tables.copy(), lengths.copy()
    out = np.full((3, tokens), -1)
    served = np.zeros(len(lengths), bool)
    at = needed = taken = 0
    for s, c in enumerate(np.maximum(counts, 0)):
        held = int(lengths[s])
        grown = held + int(c)
        fits = grown <= tables.shape[1] * page and at + c <= tokens
        need = -(-grown // page) + -held // page if fits else 0
        needed += need
        served[s] = fits and (need == 0 or needed <= count)
        if served[s]:
            for j in range(need):
                tables[s, -(-held // page) + j] = free[count - 1 - taken]
                taken += 1
            for i in range(c):
                p = held + i
                out[:, at + i] = tables[s, p // page] * page + p % page, p, s
            lengths[s] = grown
        at += c
    return (*out, served, tables, lengths, count - taken)


def shrink(tables, lengths, free, count, page, to):
    """The lengths, the stack and its count afterwards."""
    new = np.minimum(lengths, np.maximum(to, 0))
    back = [tables[s, j] for s in range(len(new)) for j in range(-(-new[s] // page), -(-lengths[s] // page))]
    free = free.copy()
    free[count : count + len(back)] = back[::-1]
    return new, free, count + len(back)


def rotate(x, positions, frequencies, interleaved=False, magnitude=1.0):
    """``x`` [N, heads, D], each pair as a complex number times magnitude e^(i position frequency)."""
    y = x.astype(np.float64).copy()
    h = len(frequencies)
    turn = magnitude * np.exp(1j * positions[:, None].astype(np.float64) * frequencies)[:, None]
    one, two = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if interleaved else (slice(0, h), slice(h, 2 * h))
    z = (y[..., one] + 1j * y[..., two]) * turn
    y[..., one], y[..., two] = z.real, z.imag
    return y


def attend(q, keys, values, lengths, prefix=None, scale=None):
    """``q`` [S, T, H, D]; ``keys[s]`` and ``values[s]`` [n, Hkv, D], a sequence's prefix (``prefix[s]`` positions) and
    its own after it. Outputs, the same with |v| for v, and the largest scale sum |q k| of each row."""
    S, T, H, D = q.shape
    scale = D**-0.5 if scale is None else scale
    out, mass, size = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:3])
    for s in range(S):
        pre, G = 0 if prefix is None else int(prefix[s]), H // keys[s].shape[1]
        for t in range(T):
            last = int(lengths[s]) - T + t + 1
            if last <= 0:
                continue
            n = pre + last
            for h in range(H):
                x, k, v = q[s, t, h].astype(np.float64), keys[s][:n, h // G].astype(np.float64), values[s][:n, h // G].astype(np.float64)
                z = scale * (k @ x)
                if not np.any(z > -np.inf) and not np.any(np.isnan(z)):
                    continue
                e = np.exp(z - np.max(z))
                e = np.where(z == -np.inf, 0.0, e)
                seen = e != 0  # (what has no weight adds nothing, whatever it holds)
                out[s, t, h] = e[seen] @ v[seen] / e.sum()
                mass[s, t, h] = e[seen] @ np.abs(v[seen]) / e.sum()
                size[s, t, h] = np.max(scale * (np.abs(k) @ np.abs(x)))
    return out, mass, size

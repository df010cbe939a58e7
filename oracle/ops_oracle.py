"""Plain numpy statements, in 64 bits, of beam search's selection, the states' reordering and the distillation
loss: what the tests of those operators check against."""

from __future__ import annotations

import numpy as np


def beam_select(logits, scores, n, finished=None, pad_id=0, keep_slots=False):
    """``logits`` [B, W, V], ``scores`` [B, W]. Returns scores fp64, beams and tokens int64, [B, n] each."""
    B, W, V = logits.shape
    out = np.full((B, n), -np.inf), np.full((B, n), -1), np.full((B, n), -1)
    for b in range(B):
        cand = []  # (score, beam, logit, id, token)
        for w in range(W):
            s = float(scores[b, w])
            if not np.isfinite(s):
                continue
            if finished is not None and finished[b, w]:
                cand.append((s, w, 0.0, 0, pad_id))
                continue
            x = logits[b, w].astype(np.float64)
            m = np.max(x)  # (NaN for a row with one)
            if not np.isfinite(m):
                continue
            logs = np.log(np.sum(np.exp(x - m)))
            order = np.lexsort((np.arange(V), -x))[:n]
            cand += [((x[v] - m) - logs + s, w, x[v], int(v), int(v)) for v in order if x[v] > -np.inf]
        cand.sort(key=lambda c: (-c[0], c[1], -c[2], c[3]))
        cand = cand[:n]
        place = list(range(n))
        if keep_slots:
            firsts = {}
            for i, c in enumerate(cand):
                firsts.setdefault(c[1], i)
            rest = [k for k in range(n) if k not in firsts]
            for i in range(len(cand)):
                place[i] = cand[i][1] if firsts[cand[i][1]] == i else rest.pop(0)
        for i, c in enumerate(cand):
            out[0][b, place[i]], out[1][b, place[i]], out[2][b, place[i]] = c[0], c[1], c[4]
    return out


def reorder(state, parents, lengths=None):
    """``state`` [B, W, L, ...] as it becomes: slot w of request b holds the first ``lengths[b]`` positions of slot
    ``parents[b, w]`` (all of them without lengths); a parent outside [0, W) changes nothing."""
    new = state.copy()
    B, W = parents.shape
    for b in range(B):
        n = state.shape[2] if lengths is None else min(max(int(lengths[b]), 0), state.shape[2])
        for w in range(W):
            if 0 <= parents[b, w] < W:
                new[b, w, :n] = state[b, parents[b, w], :n]
    return new


def _log_softmax(x):
    """(The largest is taken off first: beside values of 1e38 a log of the sum would be lost.)"""
    if not np.any(x > -np.inf) and not np.any(np.isnan(x)):
        return x
    d = x - np.max(x)
    return d - np.log(np.sum(np.exp(d)))


def distill(student, ids, teacher, weights, temperature=1.0, tail=False):
    """Losses [T] and gradients [T, V], row by row from log-softmax."""
    T, V = student.shape
    loss, grad = np.zeros(T), np.zeros((T, V))
    for t in range(T):
        w = 1.0 if weights is None else float(weights[t])
        if w == 0.0:
            continue
        z = student[t].astype(np.float64) / temperature
        there = (ids[t] >= 0) & (ids[t] < V)
        at = ids[t][there].astype(np.int64)
        a = teacher[t][there].astype(np.float64)
        if not tail:
            a = a / temperature
            if not np.any(a > -np.inf):
                continue
            a = _log_softmax(a)
        p = np.exp(a)
        logq = _log_softmax(z)
        q = np.exp(logq)
        hot = p > 0
        total = np.sum(p[hot] * (a[hot] - logq[at][hot]))
        rest = max(0.0, 1.0 - np.sum(p)) if tail else 0.0
        g = q * (np.sum(p) + rest)
        others = np.ones(V, bool)
        others[at] = False
        if rest > 0.0:
            with np.errstate(divide="ignore"):
                log_rest = np.max(logq[others], initial=-np.inf)
                if log_rest > -np.inf:
                    log_rest += np.log(np.sum(np.exp(logq[others] - log_rest)))
            total += rest * (np.log(rest) - log_rest)
            if log_rest > -np.inf:
                g[others] -= rest * np.exp(_log_softmax(z[others]))
        g[at] -= p
        loss[t], grad[t] = w * total, w / temperature * g
    return loss, grad

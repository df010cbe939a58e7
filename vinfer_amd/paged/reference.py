"""The ``reference`` paged-cache backend: plain torch, sequence by sequence."""

from __future__ import annotations

import math

import torch

from vinfer_amd.paged.base import (
    PAGED,
    AttentionPlan,
    Extension,
    PageTables,
    Rotary,
    check_attend,
    check_extend,
    check_plan,
    check_rotate,
    check_shrink,
)
from vinfer_amd.registry import BackendContext


def _ceil(n: int, page: int) -> int:
    return -(-n // page)


@PAGED.register("reference")
class ReferencePaged:
    def __init__(self, ctx: BackendContext) -> None:
        self.ctx = ctx

    def extend(self, pages: PageTables, counts: torch.Tensor, tokens: int) -> Extension:
        check_extend(pages, counts, tokens)
        page, wide = pages.page_size, pages.tables.shape[1]
        cap = min(wide * page, (1 << 31) - 1)
        tables, free = pages.tables.tolist(), pages.free.tolist()
        left = min(max(int(pages.free_count), 0), len(free))
        lengths = [min(max(n, 0), cap) for n in pages.lengths.tolist()]
        new_lengths, served, out = pages.lengths.tolist(), [], [[-1] * tokens for _ in range(3)]
        at = needed = 0
        enough = left
        for s, c in enumerate(counts.tolist()):
            c = max(c, 0)
            fits = lengths[s] + c <= cap and at + c <= tokens
            need = _ceil(lengths[s] + c, page) - _ceil(lengths[s], page) if fits else 0
            needed += need
            ok = fits and (need == 0 or needed <= enough)
            if ok and c:
                for i in range(need):
                    left -= 1
                    tables[s][_ceil(lengths[s], page) + i] = free[left]
                for i in range(c):
                    p = lengths[s] + i
                    out[0][at + i], out[1][at + i], out[2][at + i] = tables[s][p // page] * page + p % page, p, s
                new_lengths[s] = lengths[s] + c
            served.append(ok)
            at += c
        dev = pages.tables.device
        mk = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        pages.tables.copy_(mk(tables).reshape(pages.tables.shape))
        pages.lengths.copy_(mk(new_lengths))
        pages.free_count.fill_(left)
        return Extension(*map(mk, out), torch.tensor(served, dtype=torch.bool, device=dev))

    def shrink(self, pages: PageTables, lengths: torch.Tensor) -> None:
        check_shrink(pages, lengths)
        page, cap = pages.page_size, min(pages.tables.shape[1] * pages.page_size, (1 << 31) - 1)
        tables, free = pages.tables.tolist(), pages.free.tolist()
        count = min(max(int(pages.free_count), 0), len(free))
        back, new = [], []
        for s, (n, to) in enumerate(zip(pages.lengths.tolist(), lengths.tolist())):
            n = min(max(n, 0), cap)
            new.append(min(n, max(to, 0)))
            back += tables[s][_ceil(new[-1], page) : _ceil(n, page)]
        for i, p in enumerate(reversed(back)):
            if count + i < len(free):
                free[count + i] = p
        dev = pages.tables.device
        pages.free.copy_(torch.tensor(free, dtype=torch.int32, device=dev))
        pages.lengths.copy_(torch.tensor(new, dtype=torch.int32, device=dev))
        pages.free_count.fill_(min(count + len(back), len(free)))

    def rotate_store(self, q, k, v, positions, slots, k_pages, v_pages, rotary: Rotary) -> torch.Tensor:
        check_rotate(q, k, v, positions, slots, k_pages, v_pages, rotary)
        angle = positions.double()[:, None] * rotary.frequencies
        cos, sin = (rotary.magnitude * f(angle)[:, None] for f in (torch.cos, torch.sin))
        half = rotary.frequencies.shape[0]

        def turn(x):
            wide = x.double()
            out = wide.clone()
            one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if rotary.interleaved \
                else (slice(0, half), slice(half, 2 * half))
            x1, x2 = wide[..., one], wide[..., two]
            out[..., one] = x1 * cos - x2 * sin
            out[..., two] = x2 * cos + x1 * sin
            return out.to(x.dtype)

        page = k_pages.shape[1]
        stored = (positions >= 0) & (slots >= 0) & (slots < k_pages.shape[0] * page)
        at = slots[stored].long()
        k_pages[at // page, at % page] = turn(k)[stored]
        v_pages[at // page, at % page] = v[stored]
        return torch.where((positions >= 0)[:, None, None], turn(q), 0)

    def plan(self, lengths, *, queries, heads, kv_heads, head_dim, page_size, max_pages, prefix_lengths=None,
             max_prefix_pages=0, group_starts=None) -> AttentionPlan:
        check_plan(lengths, queries, heads, kv_heads, head_dim, page_size, max_pages, prefix_lengths, max_prefix_pages,
                   group_starts)
        S = lengths.shape[0]
        own = [min(max(n, 0), max_pages * page_size) for n in lengths.tolist()]
        group = [-1] * S
        prefixes = []
        if prefix_lengths is not None:
            prefixes = [min(max(n, 0), max_prefix_pages * page_size) for n in prefix_lengths.tolist()]
            starts = group_starts.tolist()
            for g in range(len(prefixes)):
                for s in range(max(starts[g], 0), min(starts[g + 1], S)):
                    group[s] = g
        return AttentionPlan(S, len(prefixes), queries, heads, kv_heads, head_dim, page_size, max_pages, max_prefix_pages,
                             lengths.device, (own, group, prefixes))

    def attend(self, q, k_pages, v_pages, tables, plan: AttentionPlan, *, prefix_tables=None, scale=None) -> torch.Tensor:
        check_attend(q, k_pages, v_pages, tables, plan, prefix_tables, scale)
        own, group, prefixes = plan.data
        T, D = plan.queries, plan.head_dim
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)

        def read(pages, table, n):  # [kv_heads, n, D], fp64
            ids = table[: _ceil(n, plan.page_size)].long().clamp(0, pages.shape[0] - 1)
            return pages[ids].flatten(0, 1)[:n].double().transpose(0, 1)

        for s in range(plan.sequences):
            n, g = own[s], group[s]
            pre = prefixes[g] if g >= 0 else 0
            for t in range(max(0, T - n), T):
                last = n - T + t + 1
                k, v = (read(pages, tables[s], last) for pages in (k_pages, v_pages))
                if pre:
                    k, v = (torch.cat([read(pages, prefix_tables[g], pre), x], 1) for pages, x in ((k_pages, k), (v_pages, v)))
                x = q[s, t].double().view(plan.kv_heads, -1, D) * (D**-0.5 if scale is None else scale)
                z = torch.matmul(x, k.transpose(1, 2).contiguous())
                z = z - z.amax(2, keepdim=True).clamp(min=-1e300)  # (a row of -inf alone stays one)
                e = torch.exp(z)
                total = e.sum(2, keepdim=True)
                y = torch.where(total == 0, 0.0, torch.matmul(e, v.contiguous()) / total)
                out[s, t] = y.reshape(plan.heads, D).to(q.dtype)
        return out


__all__ = ["ReferencePaged"]

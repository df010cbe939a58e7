"""The ``hip`` paged-cache backend: gfx950 kernels behind the C ABI of libvpaged.so.

Registered for device type ``"cuda"`` (ROCm PyTorch reports HIP devices as ``cuda``) and the dtypes bf16 and
fp16. Every call enqueues its work on torch's current stream of its tensors' device and returns without
synchronising; outputs, plans and workspaces are torch's, so calls may be captured into HIP graphs.
"""

from __future__ import annotations

import ctypes

import torch

from vinfer_amd import _vpaged
from vinfer_amd.paged.base import (
    DTYPES,
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


def _on_gpu(device) -> None:
    if device.type != "cuda":
        raise ValueError(f"the hip paged cache needs its tensors on a GPU, got {device}")


def _dtype(t) -> int:
    if t.dtype not in DTYPES:
        raise ValueError(f"the hip paged cache supports bf16 and fp16, got {t.dtype}")
    return DTYPES[t.dtype]


class _Planned:
    """A plan's memory, and the argument block that its layers share."""

    def __init__(self, shape, memory, stream, workspace: int) -> None:
        self.shape, self.memory, self.stream, self.workspace = shape, memory, stream, workspace


@PAGED.register("hip", devices={"cuda"}, dtypes=set(DTYPES), supports=lambda ctx: _vpaged.unsupported(ctx.device))
class HipPaged:
    def __init__(self, ctx: BackendContext) -> None:
        self.ctx = ctx
        self._lib = _vpaged.load()
        self._need: dict[tuple, tuple] = {}  # a shape's block, and its plan's and workspace's bytes

    @staticmethod
    def _tables(pages: PageTables) -> _vpaged.VpagedTables:
        _on_gpu(pages.tables.device)
        S, M = pages.tables.shape
        return _vpaged.VpagedTables(pages.tables.data_ptr(), pages.lengths.data_ptr(), pages.free.data_ptr(),
                                    pages.free_count.data_ptr(), S, M, pages.free.shape[0], pages.page_size)

    def extend(self, pages: PageTables, counts: torch.Tensor, tokens: int) -> Extension:
        check_extend(pages, counts, tokens)
        dev = pages.tables.device
        t = self._tables(pages)
        counts = counts.contiguous()
        out = torch.empty(3, tokens, dtype=torch.int32, device=dev)
        served = torch.empty(counts.shape, dtype=torch.bool, device=dev)
        at, need = out.data_ptr(), self._lib.vpaged_extend_workspace_bytes(t.sequences, tokens)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _vpaged.call(self._lib.vpaged_extend, dev, ctypes.byref(t), counts.data_ptr(), tokens, at, at + 4 * tokens, at + 8 * tokens,
                     served.data_ptr(), ws.data_ptr() if need else None, need)
        return Extension(*out.unbind(0), served)

    def shrink(self, pages: PageTables, lengths: torch.Tensor) -> None:
        check_shrink(pages, lengths)
        lengths = lengths.contiguous()
        _vpaged.call(self._lib.vpaged_shrink, pages.tables.device, ctypes.byref(self._tables(pages)), lengths.data_ptr())

    def rotate_store(self, q, k, v, positions, slots, k_pages, v_pages, rotary: Rotary) -> torch.Tensor:
        check_rotate(q, k, v, positions, slots, k_pages, v_pages, rotary)
        dev, dtype = q.device, _dtype(q)
        _on_gpu(dev)
        N, heads, D = q.shape
        positions, slots = positions.contiguous(), slots.contiguous()
        out = torch.empty(N, heads, D, dtype=q.dtype, device=dev)
        (qn, qh, _), (kn, kh, _), (vn, vh, _), (pn, pp, ph, _) = q.stride(), k.stride(), v.stride(), k_pages.stride()
        f = rotary.frequencies
        a = _vpaged.VpagedRotateArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), qn, kn, vn, qh, kh, vh, out.data_ptr(),
                                     k_pages.data_ptr(), v_pages.data_ptr(), pn, pp, ph, positions.data_ptr(),
                                     slots.data_ptr(), f.data_ptr(), rotary.magnitude, dtype, N, heads, k.shape[1], D,
                                     2 * f.shape[0], rotary.interleaved, k_pages.shape[0], k_pages.shape[1])
        _vpaged.call(self._lib.vpaged_rotate_store, dev, ctypes.byref(a))
        return out

    def plan(self, lengths, *, queries, heads, kv_heads, head_dim, page_size, max_pages, prefix_lengths=None,
             max_prefix_pages=0, group_starts=None) -> AttentionPlan:
        check_plan(lengths, queries, heads, kv_heads, head_dim, page_size, max_pages, prefix_lengths, max_prefix_pages,
                   group_starts)
        dev = lengths.device
        _on_gpu(dev)
        S, B = lengths.shape[0], 0 if prefix_lengths is None else prefix_lengths.shape[0]
        if not B:
            max_prefix_pages = 0
        key = S, B, queries, heads, kv_heads, head_dim, page_size, max_pages, max_prefix_pages
        known = self._need.get(key)
        if known is None:
            shape = _vpaged.VpagedShape(DTYPES[self.ctx.dtype], *key)
            known = shape, self._lib.vpaged_plan_bytes(shape), self._lib.vpaged_attend_workspace_bytes(shape)
            if not known[1]:
                raise ValueError(f"a shape of more tiles or rows than 32 bits number: {key}")
            if len(self._need) > 4096:
                self._need.clear()
            self._need[key] = known
        shape, need, workspace = known
        memory = torch.empty(need, dtype=torch.uint8, device=dev)  # (torch aligns to 512 bytes)
        lengths = lengths.contiguous()
        if B:
            prefix_lengths, group_starts = prefix_lengths.contiguous(), group_starts.contiguous()
        _vpaged.call(self._lib.vpaged_plan, dev, ctypes.byref(shape), lengths.data_ptr(), prefix_lengths.data_ptr() if B else None,
                     group_starts.data_ptr() if B else None, memory.data_ptr(), need)
        return AttentionPlan(S, B, queries, heads, kv_heads, head_dim, page_size, max_pages, max_prefix_pages, dev,
                             _Planned(shape, memory, torch._C._cuda_getCurrentRawStream(dev.index), workspace))

    def attend(self, q, k_pages, v_pages, tables, plan: AttentionPlan, *, prefix_tables=None, scale=None) -> torch.Tensor:
        check_attend(q, k_pages, v_pages, tables, plan, prefix_tables, scale)
        dev, data = q.device, plan.data
        if q.dtype != self.ctx.dtype:
            raise ValueError(f"this backend was made for {self.ctx.dtype}, got {q.dtype}")
        sn, st, sh, _ = q.stride()
        if (sn | st | sh) & 7 or q.data_ptr() & 15:
            q = q.contiguous()
            sn, st, sh, _ = q.stride()
        pn, pp, ph, _ = k_pages.stride()
        if (pn | pp | ph) & 7 or (k_pages.data_ptr() | v_pages.data_ptr()) & 15:
            raise ValueError("the cache must be 16-byte aligned, with strides of multiples of 8 elements")
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        if torch._C._cuda_getCurrentRawStream(dev.index) != data.stream:
            data.memory.record_stream(torch.cuda.current_stream(dev))
        ws = torch.empty(data.workspace, dtype=torch.uint8, device=dev)
        pre, pre_stride = (prefix_tables.data_ptr(), prefix_tables.stride(0)) if plan.groups else (None, 0)
        a = _vpaged.VpagedAttendArgs(data.shape, k_pages.shape[0], plan.head_dim**-0.5 if scale is None else scale,
                                     q.data_ptr(), sn, st, sh, k_pages.data_ptr(), v_pages.data_ptr(), pn, pp, ph,
                                     tables.data_ptr(), pre, tables.stride(0), pre_stride, out.data_ptr(),
                                     data.memory.data_ptr(), ws.data_ptr(), data.workspace)
        _vpaged.call(self._lib.vpaged_attend, dev, ctypes.byref(a))
        return out


__all__ = ["HipPaged"]

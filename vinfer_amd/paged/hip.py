"""The ``hip`` paged-cache backend: gfx950 kernels behind the C ABI of libvpaged.so.

Registered for device type ``"cuda"`` (ROCm PyTorch reports HIP devices as ``cuda``) and the dtypes bf16 and
fp16. Every call enqueues its work on torch's current stream of its tensors' device and returns without
synchronising; outputs, plans and workspaces are torch's, so calls may be captured into HIP graphs.

A decode step makes these calls for few tokens, where their checks would take longer than their kernels: what a call
says of shapes, layouts, types and devices is checked once, and what the library needs of it kept by all that was
checked.
"""

from __future__ import annotations

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
    differentiated,
)
from vinfer_amd.registry import BackendContext

_KNOWN = 4096  # calls of unlike shapes that a backend keeps in mind


def _on_gpu(device) -> None:
    if device.type != "cuda":
        raise ValueError(f"the hip paged cache needs its tensors on a GPU, got {device}")


def _strides(t, n: int) -> tuple[int, ...]:
    """The first n strides, 0 in dimensions of one element (torch keeps any number there)."""
    return tuple(st if size > 1 else 0 for st, size in zip(t.stride()[:n], t.shape))


class _Planned:
    """A plan's memory and stream, its shape (any type's: the kernels that make it know none), and its layers' workspace."""

    def __init__(self, shape, memory, stream, workspace) -> None:
        self.shape, self.memory, self.stream, self.workspace = shape, memory, stream, workspace


@PAGED.register("hip", devices={"cuda"}, dtypes=set(DTYPES), supports=lambda ctx: _vpaged.unsupported(ctx.device))
class HipPaged:
    def __init__(self, ctx: BackendContext) -> None:
        self.ctx = ctx
        self._lib = _vpaged.load()
        self._known: dict[tuple, tuple] = {}

    def _keep(self, key, value):
        if len(self._known) >= _KNOWN:
            self._known.clear()
        self._known[key] = value
        return value

    def _check_dtype(self, t) -> None:
        if t.dtype != self.ctx.dtype:
            raise ValueError(f"this backend was made for {self.ctx.dtype}, got {t.dtype}")

    @staticmethod
    def _tables(pages: PageTables) -> bytes:
        t, free = pages.tables, pages.free
        S, M = t.shape
        return _vpaged.PACK_TABLES.pack(t.data_ptr(), pages.lengths.data_ptr(), free.data_ptr(), pages.free_count.data_ptr(),
                                        S, M, free.shape[0], pages.page_size)

    def extend(self, pages: PageTables, counts: torch.Tensor, tokens: int) -> Extension:
        check_extend(pages, counts, tokens)
        dev = counts.device
        _on_gpu(dev)
        counts = counts.contiguous()
        slots, positions, sequences = counts.new_empty(tokens), counts.new_empty(tokens), counts.new_empty(tokens)
        served = counts.new_empty(counts.shape, dtype=torch.bool)
        ws, need = None, self._lib.vpaged_extend_workspace_bytes(counts.shape[0], tokens)
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=dev)  # (torch aligns to 512 bytes)
        _vpaged.call(self._lib.vpaged_extend, dev, self._tables(pages), counts.data_ptr(), tokens, slots.data_ptr(),
                     positions.data_ptr(), sequences.data_ptr(), served.data_ptr(), ws.data_ptr() if need else None, need)
        return Extension(slots, positions, sequences, served)

    def shrink(self, pages: PageTables, lengths: torch.Tensor) -> None:
        check_shrink(pages, lengths)
        dev = lengths.device
        _on_gpu(dev)
        lengths = lengths.contiguous()
        _vpaged.call(self._lib.vpaged_shrink, dev, self._tables(pages), lengths.data_ptr())

    def rotate_store(self, q, k, v, positions, slots, k_pages, v_pages, rotary: Rotary) -> torch.Tensor:
        f = rotary.frequencies
        key = ("rotate", torch.is_grad_enabled(), q.requires_grad, k.requires_grad, v.requires_grad, k_pages.requires_grad,
               v_pages.requires_grad, f.requires_grad, rotary.interleaved, rotary.magnitude, f.shape, q.shape, k.shape, v.shape,
               positions.shape, slots.shape, k_pages.shape, v_pages.shape, q.stride(), k.stride(), v.stride(), k_pages.stride(),
               v_pages.stride(), q.dtype, k.dtype, v.dtype, positions.dtype, slots.dtype, k_pages.dtype, v_pages.dtype,
               q.get_device(), k.get_device(), v.get_device(), positions.get_device(), slots.get_device(), k_pages.get_device(),
               v_pages.get_device(), f.get_device())
        known = self._known.get(key)
        if known is None or differentiated():
            check_rotate(q, k, v, positions, slots, k_pages, v_pages, rotary)
            _on_gpu(q.device)
            self._check_dtype(q)
            N, heads, D = q.shape
            known = self._keep(key, (
                q.device, (N, heads, D), tuple(x for t in (q, k, v) for x in t.stride()[:1]) + tuple(t.stride(1) for t in (q, k, v)),
                k_pages.stride()[:3], (rotary.magnitude, DTYPES[q.dtype], N, heads, k.shape[1], D, 2 * f.shape[0],
                                       int(rotary.interleaved), k_pages.shape[0], k_pages.shape[1])))
        dev, shape, strides, page_strides, rest = known
        positions, slots = positions.contiguous(), slots.contiguous()
        out = q.new_empty(shape)
        a = _vpaged.PACK_ROTATE.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), *strides, out.data_ptr(), k_pages.data_ptr(),
                                     v_pages.data_ptr(), *page_strides, positions.data_ptr(), slots.data_ptr(), f.data_ptr(), *rest)
        _vpaged.call(self._lib.vpaged_rotate_store, dev, a)
        return out

    def plan(self, lengths, *, queries, heads, kv_heads, head_dim, page_size, max_pages, prefix_lengths=None,
             max_prefix_pages=0, group_starts=None) -> AttentionPlan:
        groups = prefix_lengths is not None and group_starts is not None
        key = ("plan", queries, heads, kv_heads, head_dim, page_size, max_pages, max_prefix_pages, lengths.shape, lengths.dtype,
               lengths.get_device(), *((prefix_lengths.shape, prefix_lengths.dtype, prefix_lengths.get_device(), group_starts.shape,
                                        group_starts.dtype, group_starts.get_device()) if groups else ()))
        known = self._known.get(key)
        if known is None or groups != (prefix_lengths is not None or group_starts is not None):
            check_plan(lengths, queries, heads, kv_heads, head_dim, page_size, max_pages, prefix_lengths, max_prefix_pages,
                       group_starts)
            _on_gpu(lengths.device)
            S, B = lengths.shape[0], prefix_lengths.shape[0] if groups else 0
            shape = S, B, queries, heads, kv_heads, head_dim, page_size, max_pages, max_prefix_pages if B else 0
            block = _vpaged.PACK_SHAPE.pack(DTYPES[self.ctx.dtype], *shape)
            need = self._lib.vpaged_plan_bytes(block)
            if not need:
                raise ValueError(f"a shape of more tiles or rows than 32 bits number: {S} sequences of {queries} x {heads} queries "
                                 f"on {max_pages} pages, {B} prefixes of {max_prefix_pages}, of {page_size} positions")
            known = self._keep(key, (lengths.device, shape, block, need, self._lib.vpaged_attend_workspace_bytes(block)))
        dev, shape, block, need, workspace = known
        memory = torch.empty(need, dtype=torch.uint8, device=dev)
        lengths = lengths.contiguous()
        pre = starts = None
        if groups:
            prefix_lengths, group_starts = prefix_lengths.contiguous(), group_starts.contiguous()
            pre, starts = prefix_lengths.data_ptr(), group_starts.data_ptr()
        _vpaged.call(self._lib.vpaged_plan, dev, block, lengths.data_ptr(), pre, starts, memory.data_ptr(), need)
        return AttentionPlan(*shape, dev, _Planned(shape, memory, torch._C._cuda_getCurrentRawStream(dev.index), workspace))

    def attend(self, q, k_pages, v_pages, tables, plan: AttentionPlan, *, prefix_tables=None, scale=None) -> torch.Tensor:
        data, pre = plan.data, prefix_tables
        if not isinstance(data, _Planned):
            raise ValueError("the plan is another backend's")
        key = ("attend", data.shape, scale, torch.is_grad_enabled(), q.requires_grad, k_pages.requires_grad, v_pages.requires_grad,
               q.shape, k_pages.shape, v_pages.shape, tables.shape, q.stride(), k_pages.stride(), v_pages.stride(), tables.stride(),
               q.dtype, k_pages.dtype, v_pages.dtype, tables.dtype, q.get_device(), k_pages.get_device(), v_pages.get_device(),
               tables.get_device(), plan.device.index,
               *((pre.shape, pre.stride(), pre.dtype, pre.get_device()) if pre is not None else ()))
        known = self._known.get(key)
        if known is None or differentiated():
            check_attend(q, k_pages, v_pages, tables, plan, pre, scale)
            self._check_dtype(q)
            strides = _strides(k_pages, 3)
            if any(x & 7 for x in strides) or strides[0] >= 1 << 31 or strides[1] * max(plan.page_size, 16) >= 1 << 30:
                raise ValueError(f"the cache's strides must be multiples of 8 elements, pages less than 2^31 elements apart and "
                                 f"a page's positions within 2^30, got {strides}")
            q_strides = _strides(q, 3)
            known = self._keep(key, (q.device, any(x & 7 for x in q_strides), q_strides, strides,
                                     (DTYPES[q.dtype], *data.shape, k_pages.shape[0], plan.head_dim**-0.5 if scale is None else scale),
                                     (tables.stride(0), pre.stride(0) if plan.groups else 0)))
        dev, odd, q_strides, strides, first, table_strides = known
        kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
        if (kp | vp) & 15:
            raise ValueError("the cache must be 16-byte aligned")
        if odd or q.data_ptr() & 15:
            q = q.clone(memory_format=torch.contiguous_format)  # (contiguous() keeps what lies at an odd address)
            q_strides = _strides(q, 3)
        out = q.new_empty(q.shape)
        ws = torch.empty(data.workspace, dtype=torch.uint8, device=dev)
        memory = data.memory
        if torch._C._cuda_getCurrentRawStream(dev.index) != data.stream:
            memory.record_stream(torch.cuda.current_stream(dev))
        a = _vpaged.PACK_ATTEND.pack(*first, q.data_ptr(), *q_strides, kp, vp, *strides, tables.data_ptr(),
                                     pre.data_ptr() if plan.groups else 0, *table_strides, out.data_ptr(), memory.data_ptr(),
                                     ws.data_ptr(), data.workspace)
        _vpaged.call(self._lib.vpaged_attend, dev, a)
        return out


__all__ = ["HipPaged"]

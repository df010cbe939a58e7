"""The ``hip`` distillation backend: gfx950 kernels behind the C ABI of libvops.so.

Registered for device type ``"cuda"`` (ROCm PyTorch reports HIP devices as ``cuda``) and the dtypes bf16 and
fp32. Every call enqueues its work on torch's current stream of the student's device and returns without
synchronising; outputs and workspaces are torch's, so calls may be captured into HIP graphs.
"""

from __future__ import annotations

import ctypes

import torch

from vinfer_amd import _vops
from vinfer_amd.distill.base import DISTILL, DTYPES, check, check_states
from vinfer_amd.registry import BackendContext


@DISTILL.register("hip", devices={"cuda"}, dtypes=set(DTYPES), supports=lambda ctx: _vops.unsupported(ctx.device))
class HipDistill:
    def __init__(self, ctx: BackendContext) -> None:
        self.ctx = ctx
        self._lib = _vops.load()
        self._need: dict[tuple, int] = {}  # workspace bytes by sizes

    def _args(self, student, ids, weights, temperature, tail):
        if student.device.type != "cuda":
            raise ValueError(f"hip distillation needs logits on a GPU, got {student.device}")
        T, V = student.shape
        ids = ids.contiguous()
        a = _vops.VopsDistillArgs()
        a.student, a.dtype = student.data_ptr(), DTYPES[student.dtype]
        a.rows, a.vocab, a.entries = T, V, ids.shape[1]
        a.row_stride = student.stride(0) if T > 1 else V
        a.ids = ids.data_ptr()
        if weights is not None:
            weights = weights.contiguous()
            a.weights = weights.data_ptr()
        a.temperature = temperature
        a.flags = _vops.VOPS_DISTILL_TAIL if tail else 0
        return a, (ids, weights)

    def _run(self, student, ids, teacher, weights, temperature, tail, grad, states):
        check(student, ids, teacher, weights, temperature)
        a, keep = self._args(student, ids, weights, temperature, tail)
        dev = student.device
        teacher = teacher.contiguous()
        a.teacher = teacher.data_ptr()
        loss = torch.empty(a.rows, dtype=torch.float32, device=dev)
        a.out_loss = loss.data_ptr()
        out = None
        if grad:
            out = torch.empty(a.rows, a.vocab, dtype=student.dtype, device=dev)
            a.out_grad, a.grad_stride = out.data_ptr(), a.vocab
        if states:
            out = torch.empty(a.rows, 2 + a.entries, dtype=torch.float32, device=dev)
            a.states = out.data_ptr()
        sizes = a.dtype, a.rows, a.vocab, a.entries
        need = self._need.get(sizes)
        if need is None:
            need = self._need[sizes] = self._lib.vops_distill_workspace_bytes(*sizes)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)  # (torch aligns to 512 bytes)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _vops.call(self._lib.vops_distill, dev, ctypes.byref(a))
        del keep
        return loss, out

    def loss(self, student, ids, teacher, weights=None, *, temperature=1.0, tail=False):
        return self._run(student, ids, teacher, weights, temperature, tail, False, False)[0]

    def loss_and_grad(self, student, ids, teacher, weights=None, *, temperature=1.0, tail=False):
        return self._run(student, ids, teacher, weights, temperature, tail, True, False)

    def loss_and_states(self, student, ids, teacher, weights=None, *, temperature=1.0, tail=False):
        return self._run(student, ids, teacher, weights, temperature, tail, False, True)

    def grad(self, student, ids, states, weights=None, *, temperature=1.0):
        check(student, ids, None, weights, temperature)
        check_states(states, ids, student)
        a, keep = self._args(student, ids, weights, temperature, False)
        out = torch.empty(a.rows, a.vocab, dtype=student.dtype, device=student.device)
        a.out_grad, a.grad_stride, a.states = out.data_ptr(), a.vocab, states.data_ptr()
        _vops.call(self._lib.vops_distill_grad, student.device, ctypes.byref(a))
        del keep
        return out


__all__ = ["HipDistill"]

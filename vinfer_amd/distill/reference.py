"""The ``reference`` distillation backend: the definition in torch, in fp64, on any device."""

from __future__ import annotations

import torch

from vinfer_amd.distill.base import DISTILL, check, check_states
from vinfer_amd.registry import BackendContext


@DISTILL.register("reference")
class ReferenceDistill:
    def __init__(self, ctx: BackendContext) -> None:
        self.ctx = ctx

    @staticmethod
    def _rows(student, ids, teacher, temperature, tail):
        """Losses and the rows' states without their weights: the ids' gradients, then the largest of the other
        logits and their gradients' factor."""
        T, V = student.shape
        x = student.double()
        there = (ids >= 0) & (ids < V)
        at = torch.where(there, ids, 0).long()
        member = torch.zeros(T, V, dtype=torch.int32, device=x.device).scatter_add_(1, at, there.int()) > 0
        logp = teacher.double() if tail else teacher.double() / temperature
        logp = torch.where(there, logp, -torch.inf)
        none = (logp == -torch.inf).all(1, keepdim=True)
        if not tail:
            logp = logp - torch.where(none, 0.0, torch.logsumexp(logp, 1, keepdim=True))
        p = torch.exp(logp)
        rest = (1 - p.sum(1)).clamp(min=0) if tail else torch.zeros(T, dtype=torch.float64, device=x.device)
        mass = p.sum(1) + rest
        z = x / temperature
        logq = torch.log_softmax(z, 1)
        others = torch.where(member, -torch.inf, logq)
        log_rest = torch.logsumexp(others, 1)
        largest = others.amax(1)
        m = torch.where(member, -torch.inf, x).amax(1)
        # (no entry, or none that either side gives a probability: nothing to learn from, whatever the logits hold)
        empty = none[:, 0] & ((torch.gather(x, 1, at) == -torch.inf) | ~there).all(1) if tail else none[:, 0]
        logq = torch.gather(logq, 1, at)
        loss = torch.where(p != 0, p * (logp - logq), 0.0).sum(1)
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - log_rest), 0.0)
        # the others' gradient: exp((x - m) / temperature) times this
        factor = mass * torch.exp(largest) - torch.where(rest > 0, rest * torch.exp(largest - log_rest), 0.0)
        factor = torch.where(m == -torch.inf, 0.0, factor)
        listed = torch.where(there, torch.exp(logq) * mass[:, None] - p, 0.0)
        states = torch.cat([m[:, None], factor[:, None], listed], 1)
        return torch.where(empty, 0.0, loss), torch.where(empty[:, None], 0.0, states)

    def loss_and_states(self, student, ids, teacher, weights=None, *, temperature=1.0, tail=False):
        check(student, ids, teacher, weights, temperature)
        loss, states = self._rows(student, ids, teacher, temperature, tail)
        if weights is not None:
            loss = torch.where(weights == 0, 0.0, weights.double() * loss)
            states = torch.where(weights[:, None] == 0, 0.0, states)
        return loss.float(), states.float()

    def grad(self, student, ids, states, weights=None, *, temperature=1.0):
        check(student, ids, None, weights, temperature)
        check_states(states, ids, student)
        T, V = student.shape
        m, factor, listed = states[:, :1].double(), states[:, 1:2].double(), states[:, 2:].double()
        m = torch.where(m == -torch.inf, 0.0, m)
        w = torch.ones(T, 1, dtype=torch.float64, device=student.device) if weights is None else weights.double()[:, None]
        # (a factor of 0: nothing of the row's logits counts, which a row of weight 0 in the forward pass was not asked for; and
        # what is 0 there is 0 under any weight)
        g = torch.where(factor == 0, 0.0, torch.exp((student.double() - m) / temperature) * factor)
        there = (ids >= 0) & (ids < V)
        rows = torch.arange(T, device=ids.device)[:, None].expand_as(ids)
        g[rows[there], ids[there].long()] = listed[there]
        return torch.where((w == 0) | (g == 0), 0.0, w / temperature * g).to(student.dtype)

    def loss(self, student, ids, teacher, weights=None, *, temperature=1.0, tail=False):
        return self.loss_and_states(student, ids, teacher, weights, temperature=temperature, tail=tail)[0]

    def loss_and_grad(self, student, ids, teacher, weights=None, *, temperature=1.0, tail=False):
        loss, states = self.loss_and_states(student, ids, teacher, weights, temperature=temperature, tail=tail)
        return loss, self.grad(student, ids, states, weights, temperature=temperature)


__all__ = ["ReferenceDistill"]

"""A draft head distilled from its target's top log-probabilities, then both searched with beams.

    python -m vinfer_amd.examples.distill_and_search [--device cpu] [--steps N]

The target is a small recurrent model (a matrix a head) with random weights. The draft head is a low-rank map of the
target's hidden states, as a speculative loop's drafter is. Each step the target runs a batch of sequences, its top
log-probabilities are taken (``logprobs``), and the head learns them with ``distill_loss`` (``tail``: the rest of the
target's mass counts as a whole). The search moves the model's recurrent states in place as its beams change.
"""

from __future__ import annotations

import argparse

import torch

from vinfer_amd.distill import DISTILL, distill_loss
from vinfer_amd.registry import BackendContext
from vinfer_amd.runtime import beam_search
from vinfer_amd.sampler import SAMPLER, BeamState


class RecurrentLM:
    """logits = head(h + q S) with S <- decay S + k v' a head, from the token's embedding h."""

    def __init__(self, vocab: int, heads: int = 4, dim: int = 32, slots: int = 64, device="cpu", seed: int = 0) -> None:
        g = torch.Generator().manual_seed(seed)
        self.device = torch.device(device)
        self.heads, self.dim, width = heads, dim, heads * dim
        mk = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(self.device)  # noqa: E731
        self.emb = mk(vocab, width)
        self.qkv = mk(width, 3 * width, scale=width**-0.5)
        self.out = mk(width, vocab, scale=2.0 * width**-0.5)
        self.decay = 0.9
        self.state = torch.zeros(slots, heads, dim, dim, device=self.device)
        self.head = lambda hidden: hidden @ self.out  # (replaced to search with another head)

    def hidden(self, slots: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
        h = self.emb[tokens]
        q, k, v = (h @ self.qkv).view(-1, 3, self.heads, self.dim).unbind(1)
        s = self.decay * self.state[slots] + 0.5 * k[..., :, None] * v[..., None, :]
        self.state[slots] = s
        return h + 0.2 * (q[..., :, None] * s).sum(-2).reshape(h.shape)

    def decode(self, slots, tokens, positions):
        return self.head(self.hidden(slots, tokens))

    def prefill(self, slot, prompt_ids):
        at = torch.tensor([slot], device=self.device)
        self.state[at] = 0.0
        for t in prompt_ids:
            h = self.hidden(at, t.view(1))
        return self.head(h)[0]

    def beam_states(self, slots):
        return [BeamState(self.state[:slots])]


def train(target: RecurrentLM, sampler, distiller, *, steps: int, batch: int, length: int, rank: int, n_top: int,
          lr: float = 0.02, seed: int = 1):
    """The draft head's two matrices, and the mean loss of each step."""
    g = torch.Generator().manual_seed(seed)
    width, vocab = target.out.shape
    mk = lambda *s: torch.nn.Parameter((torch.randn(*s, generator=g) * s[0] ** -0.5).to(target.device))  # noqa: E731
    down, up = mk(width, rank), mk(rank, vocab)
    opt = torch.optim.Adam([down, up], lr=lr)
    slots = torch.arange(batch, device=target.device)
    losses = []
    for _ in range(steps):
        tokens = torch.randint(vocab, (batch, length), generator=g).to(target.device)
        target.state[slots] = 0.0
        hidden = torch.cat([target.hidden(slots, tokens[:, i]) for i in range(length)])
        _, ids, top = sampler.logprobs((hidden @ target.out).float(), n_top=n_top)
        weights = torch.full((hidden.shape[0],), 1.0 / hidden.shape[0], device=target.device)
        loss = distill_loss(hidden @ down @ up, ids, top, weights, tail=True, backend=distiller).sum()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    return down.detach(), up.detach(), losses


def main(argv=None) -> dict:
    p = argparse.ArgumentParser()
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--vocab", type=int, default=4096)
    p.add_argument("--width", type=int, default=4)
    a = p.parse_args(argv)
    dev = torch.device("cuda", torch.cuda.current_device()) if a.device == "cuda" else torch.device(a.device)
    ctx = BackendContext(dev, torch.float32)
    name = "hip" if dev.type == "cuda" else "reference"
    sampler, distiller = SAMPLER.resolve(name, ctx), DISTILL.resolve(name, ctx)
    target = RecurrentLM(a.vocab, device=dev)
    down, up, losses = train(target, sampler, distiller, steps=a.steps, batch=16, length=8, rank=64, n_top=20)
    print(f"distillation: {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps", flush=True)
    prompts = [[1, 2, 3], [7], [11, 5, 9, 4]]
    found = {"target": beam_search(target, sampler, prompts, width=a.width, max_tokens=8, eos_token_ids=[0])}
    target.head = lambda hidden: hidden @ down @ up
    found["draft"] = beam_search(target, sampler, prompts, width=a.width, max_tokens=8, eos_token_ids=[0])
    for who, results in found.items():
        for prompt, hyps in zip(prompts, results):
            print(f"{who} {prompt}: {hyps[0].tokens} at {hyps[0].score:.3f}", flush=True)
    return {"losses": losses, **found}


if __name__ == "__main__":
    main()

"""A small attention model searched with beams over its prompts' shared pages.

    python -m vinfer_amd.examples.shared_prompt_search [--device cpu] [--width N]

The model (random weights) keeps its keys and values in a ``SharedPromptCache``: a prompt once, each beam's continuation
by itself. ``beam_search`` moves the continuations as beams change; the prompts stay where they are.
"""

from __future__ import annotations

import argparse

import torch

from vinfer_amd.paged import PAGED, Rotary, rotary_frequencies
from vinfer_amd.registry import BackendContext
from vinfer_amd.runtime import SharedPromptCache, beam_search
from vinfer_amd.sampler import SAMPLER


class AttentionLM:
    """Layers of attention and a two-layer map beside it on a residual stream, RMS norms before each."""

    shared_prompts = True

    def __init__(self, vocab: int, *, layers: int = 2, heads: int = 4, kv_heads: int = 2, head_dim: int = 64, requests: int = 4,
                 beams: int = 4, max_prompt: int = 256, max_tokens: int = 64, dtype=torch.bfloat16, device="cpu", seed: int = 0) -> None:
        g = torch.Generator().manual_seed(seed)
        self.device = torch.device(device)
        width = heads * head_dim
        mk = lambda *s: (torch.randn(*s, generator=g) * s[0] ** -0.5).to(dtype).to(self.device)  # noqa: E731
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.emb = (torch.randn(vocab, width, generator=g)).to(dtype).to(self.device)
        self.layers = [(mk(width, (heads + 2 * kv_heads) * head_dim), mk(width, width), mk(width, 2 * width), mk(2 * width, width))
                       for _ in range(layers)]
        self.out = mk(width, vocab)
        name = "hip" if self.device.type == "cuda" else "reference"
        self.cache = SharedPromptCache(
            PAGED.resolve(name, BackendContext(self.device, dtype)), layers=layers, requests=requests, beams=beams, heads=heads,
            kv_heads=kv_heads, head_dim=head_dim, prompt_pages=requests * -(-max_prompt // 16), max_prompt=max_prompt,
            max_tokens=max_tokens, rotary=Rotary(rotary_frequencies(head_dim, device=self.device)), dtype=dtype, device=self.device)
        self.max_new_tokens = max_tokens

    def _hidden(self, step, tokens):
        x = self.emb[tokens]
        norm = lambda t: torch.nn.functional.rms_norm(t, t.shape[-1:])  # noqa: E731
        split = [n * self.head_dim for n in (self.heads, self.kv_heads, self.kv_heads)]
        for i, (qkv, out, up, down) in enumerate(self.layers):
            q, k, v = (t.unflatten(1, (-1, self.head_dim)) for t in (norm(x) @ qkv).split(split, 1))
            x = x + step.attend(i, q, k, v).flatten(1) @ out
            x = x + torch.relu(norm(x) @ up) @ down
        return norm(x)

    def prefill(self, slot, prompt_ids):
        return (self._hidden(self.cache.prefill(slot, prompt_ids.shape[0]), prompt_ids)[-1:] @ self.out)[0]

    def decode(self, slots, tokens, positions):
        return self._hidden(self.cache.decode(slots, positions), tokens) @ self.out

    def release(self, slot):
        self.cache.release(slot)

    def beam_states(self, slots):
        return self.cache.beam_states()


def main(argv=None) -> list:
    p = argparse.ArgumentParser()
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    p.add_argument("--vocab", type=int, default=4096)
    p.add_argument("--width", type=int, default=4)
    p.add_argument("--tokens", type=int, default=12)
    a = p.parse_args(argv)
    dev = torch.device("cuda", torch.cuda.current_device()) if a.device == "cuda" else torch.device(a.device)
    prompts = [list(range(1, 40)), [7], [11, 5, 9, 4]]
    model = AttentionLM(a.vocab, requests=len(prompts), beams=a.width, max_tokens=a.tokens, device=dev)
    sampler = SAMPLER.resolve("hip" if dev.type == "cuda" else "reference", BackendContext(dev, torch.bfloat16))
    found = beam_search(model, sampler, prompts, width=a.width, max_tokens=a.tokens, eos_token_ids=[0])
    for prompt, hyps in zip(prompts, found):
        print(f"{len(prompt)} tokens: {hyps[0].tokens} at {hyps[0].score:.3f}", flush=True)
    return found


if __name__ == "__main__":
    main()

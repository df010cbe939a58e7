"""Beam search over a decode model (``runtime.beam_search``) against a search that recomputes every beam from its
prompt in fp64, and the distillation example."""

from __future__ import annotations

import math

import pytest
import torch

from vinfer_amd.examples.distill_and_search import RecurrentLM, main
from vinfer_amd.registry import BackendContext
from vinfer_amd.runtime import beam_search
from vinfer_amd.sampler import SAMPLER

DEVICES = [torch.device("cpu"), pytest.param(torch.device("cuda", 0), marks=pytest.mark.gpu)]


def backend(device):
    return SAMPLER.resolve("hip" if device.type == "cuda" else "reference", BackendContext(device, torch.float32))


def plain_search(model: RecurrentLM, prompt, width, max_tokens, eos):
    """Every step from the prompt: no states to move, no kernels."""
    def logprobs(ids):
        s = torch.zeros(model.heads, model.dim, model.dim, dtype=torch.float64)
        for t in ids:
            h = model.emb[t].double()
            q, k, v = (h @ model.qkv.double()).view(3, model.heads, model.dim).unbind(0)
            s = model.decay * s + 0.5 * k[:, :, None] * v[:, None, :]
        return torch.log_softmax((h + 0.2 * (q[:, :, None] * s).sum(1).reshape(-1)) @ model.out.double(), 0)

    beams = [([], 0.0, False)]
    for _ in range(max_tokens):
        cand = []
        for ids, score, done in beams:
            if done:
                cand.append((score, ids, True))
            else:
                lp = logprobs(list(prompt) + ids)
                top = torch.topk(lp, min(width, lp.numel()))
                cand += [(score + float(v), ids + [int(t)], int(t) in eos) for v, t in zip(*top)]
        cand.sort(key=lambda c: -c[0])
        beams = [(ids, score, done) for score, ids, done in cand[:width]]
        if all(done for _, _, done in beams):
            break
    return beams


@pytest.mark.parametrize("eos", [(), tuple(range(30))], ids=["open", "ends"])
@pytest.mark.parametrize("width", [1, 3, 8])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_the_search_finds_what_a_search_from_the_prompts_finds(device, width, eos):
    model = RecurrentLM(211, heads=2, dim=8, slots=40, seed=3)
    prompts = [[5], [9, 17, 4], [100, 3]]
    want = [plain_search(model, p, width, 9, eos) for p in prompts]
    moved = RecurrentLM(211, heads=2, dim=8, slots=40, device=device, seed=3)
    got = beam_search(moved, backend(device), prompts, width=width, max_tokens=9, eos_token_ids=eos, length_penalty=0.0,
                      check_every=2)
    for w, g in zip(want, got):
        assert [h.tokens for h in g] == [ids for ids, _, _ in w]
        assert [h.finished for h in g] == [done for _, _, done in w]
        for h, (_, score, _) in zip(g, w):
            # nine sums of fp32 log-probabilities of size up to 10 from fp32 logits (products of up to 32 terms)
            assert math.isclose(h.score, score, abs_tol=9 * 64 * 10 * 2.0**-24)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_fewer_continuations_than_beams(device):
    model = RecurrentLM(3, heads=1, dim=4, slots=16, device=device, seed=1)
    got = beam_search(model, backend(device), [[1]], width=8, max_tokens=1)
    assert sorted(h.tokens for h in got[0]) == [[0], [1], [2]]
    assert math.isclose(sum(math.exp(h.score) for h in got[0]), 1.0, abs_tol=1e-5)


def test_empty_prompts_are_refused():
    model = RecurrentLM(7, heads=1, dim=4, slots=8)
    for prompts in ([], [[1], []]):
        with pytest.raises(ValueError, match="prompt"):
            beam_search(model, backend(torch.device("cpu")), prompts, width=2, max_tokens=3)
    with pytest.raises(ValueError, match="positive"):
        beam_search(model, backend(torch.device("cpu")), [[1]], width=2, max_tokens=0)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_the_example_learns_and_searches(device, capsys):
    found = main(["--device", device.type, "--steps", "25", "--vocab", "600"])
    assert found["losses"][-1] < 0.8 * found["losses"][0]
    assert all(len(h) == 4 for h in found["target"] + found["draft"])
    assert "distillation:" in capsys.readouterr().out

"""The paged cache's operators together: tables, rotation and storing, attention and the reordering of beams, as a
model's steps make them (``runtime.SharedPromptCache``), searches over it, and the decode loop."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_oracle
from vinfer_amd.examples.shared_prompt_search import AttentionLM, main
from vinfer_amd.paged import PAGED, PageTables, Rotary, rotary_frequencies
from vinfer_amd.registry import BackendContext
from vinfer_amd.runtime import BatchDecoder, NoRoom, SharedPromptCache, SpeculativeDecoder, beam_search
from vinfer_amd.sampler import SAMPLER
from vinfer_amd.sampling import SamplingParams

GPU = torch.device("cuda", 0)
DEVICES = [torch.device("cpu"), pytest.param(GPU, marks=pytest.mark.gpu)]
BF16 = torch.bfloat16


def resolve(registry, device, dtype=BF16):
    return registry.resolve("hip" if device.type == "cuda" else "reference", BackendContext(device, dtype))


def make_cache(device, requests, beams, *, layers=2, heads=6, kv_heads=2, D=72, dtype=BF16, max_prompt=300, max_tokens=40):
    return SharedPromptCache(resolve(PAGED, device, dtype), layers=layers, requests=requests, beams=beams, heads=heads,
                             kv_heads=kv_heads, head_dim=D, prompt_pages=40, max_prompt=max_prompt, max_tokens=max_tokens,
                             rotary=Rotary(rotary_frequencies(D // 2 // 2 * 2, device=device)), dtype=dtype, device=device)


class Mirror:
    """What every sequence holds, token by token: keys turned in 64 bits, values as they are."""

    def __init__(self, cache):
        self.f = cache.rotary.frequencies.cpu().numpy()
        self.prompts, self.own = {}, {}

    def turned(self, x, position):
        return paged_oracle.rotate(x.double().cpu().numpy()[None], np.array([position]), self.f)[0]


def check_attend(step, layer, q, k, v, held, lengths, prefix):
    """The step's outputs against softmaxes over ``held`` (a sequence's turned keys and values)."""
    got = step.attend(layer, q, k, v).double().cpu().numpy()
    S, T = step.plan.sequences, step.plan.queries
    f = step.cache.rotary.frequencies.cpu().numpy()
    turned = paged_oracle.rotate(q.double().cpu().numpy(), step.positions.cpu().numpy(), f).reshape(S, T, *q.shape[1:])
    out, mass, size = paged_oracle.attend(turned, [np.stack(h[0]) for h in held], [np.stack(h[1]) for h in held], lengths, prefix)
    # queries and keys are rounded after they are turned (half a step each of |q k|), weights and the output once
    step_ = 2.0**-8
    weight = step_ + 2 * step_ * size.reshape(S, T, -1, 1) * 2 + 2.0**-12
    bound = step_ * np.abs(out) + 1.1 * np.expm1(weight) * 2 * mass + 2.0**-20
    assert np.all(np.abs(got.reshape(out.shape) - out) <= bound)
    assert np.mean(np.abs(got.reshape(out.shape) - out)) <= 2 * step_ * np.mean(mass)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_a_search_s_steps(device):
    B, W, layers, tokens = 3, 4, 2, 21
    cache = make_cache(device, B, W)
    g = torch.Generator().manual_seed(1)
    rng = np.random.default_rng(1)
    reorder = resolve(SAMPLER, device).prepare_reorder(cache.beam_states(), B, W)

    def qkv(n):
        return [torch.randn(n, h, 72, generator=g).to(BF16).to(device) for h in (6, 2, 2)]

    mirror = Mirror(cache)
    prompts = [37, 1, 260]
    held = {}  # (layer, request): (keys, values)
    for b, n in enumerate(prompts):
        step = cache.prefill(b * W, n)
        for i in range(layers):
            q, k, v = qkv(n)
            held[i, b] = [mirror.turned(k[t], t) for t in range(n)], [v[t].double().cpu().numpy() for t in range(n)]
            check_attend(step, i, q, k, v, [held[i, b]], [n], None)
    own = {(i, s): ([], []) for i in range(layers) for s in range(B * W)}
    lengths = torch.tensor(prompts, dtype=torch.int32, device=device)
    reorder.launch(torch.zeros(B, W, dtype=torch.int32, device=device), torch.zeros_like(lengths))
    slots = torch.arange(B * W, device=device)
    for t in range(tokens):
        step = cache.decode(slots, (lengths + t).repeat_interleave(W).long())
        for i in range(layers):
            q, k, v = qkv(B * W)
            for s in range(B * W):
                own[i, s][0].append(mirror.turned(k[s], prompts[s // W] + t))
                own[i, s][1].append(v[s].double().cpu().numpy())
            both = [[held[i, s // W][j] + own[i, s][j] for j in range(2)] for s in range(B * W)]
            check_attend(step, i, q, k, v, both, [t + 1] * (B * W), [prompts[s // W] for s in range(B * W)])
        parents = rng.integers(0, W, (B, W))
        reorder.launch(torch.tensor(parents, dtype=torch.int32, device=device), torch.full_like(lengths, t + 1))
        own = {(i, s): tuple(list(x) for x in own[i, s // W * W + int(parents[s // W, s % W])]) for i, s in own}


def plain_search(model, prompt, width, tokens):
    """Every step from the prompt, all of it in the model's own arithmetic but its cache."""
    def logprobs(ids):
        x = model.emb[torch.tensor(ids)].double()
        f = model.cache.rotary.frequencies.cpu().numpy()
        pos = np.arange(len(ids))
        norm = lambda t: t / torch.sqrt((t * t).mean(-1, keepdim=True) + torch.finfo(torch.float32).eps)  # noqa: E731
        for qkv, out, up, down in model.layers:
            split = [n * model.head_dim for n in (model.heads, model.kv_heads, model.kv_heads)]
            q, k, v = (t.unflatten(1, (-1, model.head_dim)).numpy() for t in (norm(x) @ qkv.double()).split(split, 1))
            q, k = (paged_oracle.rotate(t, pos, f) for t in (q, k))
            y, _, _ = paged_oracle.attend(q[None], [k], [v], [len(ids)])
            x = x + torch.from_numpy(y[0]).flatten(1) @ out.double()
            x = x + torch.relu(norm(x) @ up.double()) @ down.double()
        return torch.log_softmax(norm(x)[-1] @ model.out.double(), 0)

    beams = [([], 0.0)]
    for _ in range(tokens):
        cand = []
        for ids, score in beams:
            lp = logprobs(list(prompt) + ids)
            top = torch.topk(lp, width)
            cand += [(score + float(v), ids + [int(t)]) for v, t in zip(*top)]
        cand.sort(key=lambda c: -c[0])
        beams = [(ids, score) for score, ids in cand[:width]]
    return beams


def test_the_search_finds_what_a_search_from_the_prompts_finds():
    prompts = [[5, 3, 8, 1, 1, 2], [9], list(range(20))]
    model = AttentionLM(61, heads=2, kv_heads=1, head_dim=16, requests=3, beams=3, max_tokens=6, dtype=torch.float32, seed=4)
    found = beam_search(model, resolve(SAMPLER, torch.device("cpu"), torch.float32), prompts, width=3, max_tokens=6, length_penalty=0.0)
    for p, hyps in zip(prompts, found):
        want = plain_search(model, p, 3, 6)
        assert [h.tokens for h in hyps] == [ids for ids, _ in want]
        # six sums of fp32 log-probabilities of size up to 10 behind two layers of products of up to 64 terms
        np.testing.assert_allclose([h.score for h in hyps], [s for _, s in want], atol=6 * 64 * 40 * 2.0**-24)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_the_decode_loop_over_single_slots(device):
    # slots that come and go: a sequence's tokens do not depend on what else is in the batch
    sampler = resolve(SAMPLER, device)
    params = SamplingParams(temperature=0.0, max_tokens=7)
    prompts = [[1, 2, 3], [4] * 17, [9, 9], [30, 20], [5]]

    def run(together):
        model = AttentionLM(97, requests=3, beams=1, max_tokens=8, device=device, seed=2)
        out = {}
        for batch in ([prompts] if together else [[p] for p in prompts]):
            loop = BatchDecoder(model, sampler, num_slots=3, max_seq_len=64)
            ids = [loop.submit(p, params) for p in batch]
            tokens = {i: [] for i in ids}
            while loop.busy:
                for rid, step in loop.step():
                    tokens[rid].append(step.token_id)
            for p, i in zip(batch, ids):
                out[tuple(p)] = tokens[i]
        assert int(model.cache.prompts.free_count) == model.cache.prompt_pages  # (every page came back)
        return out

    assert run(True) == run(False)


@pytest.mark.gpu
def test_a_captured_step():
    B, W = 2, 3
    cache = make_cache(GPU, B, W)
    g = torch.Generator().manual_seed(3)
    qkv = lambda n: [torch.randn(n, h, 72, generator=g).to(BF16).to(GPU) for h in (6, 2, 2)]  # noqa: E731
    for b, n in enumerate((100, 18)):
        cache.prefill(b * W, n).attend(0, *qkv(n))
    slots = torch.arange(B * W, device=GPU)
    positions = torch.tensor([100] * W + [18] * W, device=GPU)
    q, k, v = qkv(B * W)
    cache.decode(slots, positions).attend(0, q, k, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.decode(slots, positions).attend(0, q, k, v)
    for t in range(5):
        for x, y in zip((q, k, v), qkv(B * W)):
            x.copy_(y)
        want = cache.decode(slots, positions).attend(0, q, k, v)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        positions += 1


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_pages_run_out_and_come_back(device):
    cache = make_cache(device, 3, 2)
    cache.prefill(0, 300)  # 19 pages of 40
    cache.prefill(2, 300)
    with pytest.raises(RuntimeError, match="no pages"):
        cache.prefill(4, 33)
    assert cache.prompts.lengths.tolist() == [300, 300, 0]
    cache.prefill(4, 32)
    cache.release(1)
    cache.prefill(4, 300)
    assert cache.prompts.lengths.tolist() == [0, 300, 300]
    for bad in (lambda: cache.prefill(6, 1), lambda: cache.prefill(0, 0), lambda: cache.prefill(0, 301),
                lambda: cache.decode(torch.arange(4, device=device), torch.zeros(4, device=device))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_a_drafted_step_and_what_is_refused_of_it(device):
    # five drafted tokens a sequence, some refused: the next step's tokens take their places
    b = resolve(PAGED, device)
    S, T, D = 3, 5, 64
    pages = PageTables.empty(S, 20, 60, 8, device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    k_pages, v_pages = (torch.zeros(60, 8, 2, D, dtype=BF16, device=device) for _ in range(2))
    rotary = Rotary(rotary_frequencies(D, device=device), interleaved=True)
    f = rotary.frequencies.cpu().numpy()
    g = torch.Generator().manual_seed(5)
    held = [([], []) for _ in range(S)]
    for step, accepted in enumerate(([5, 1, 3], [0, 5, 2], [4, 4, 5], [1, 2, 3])):
        before = pages.lengths.tolist()
        e = b.extend(pages, i32([T] * S), S * T)
        q, k, v = (torch.randn(S * T, h, D, generator=g).to(BF16).to(device) for h in (4, 2, 2))
        turned = b.rotate_store(q, k, v, e.positions, e.slots, k_pages, v_pages, rotary)
        plan = b.plan(pages.lengths, queries=T, heads=4, kv_heads=2, head_dim=D, page_size=8, max_pages=20)
        got = b.attend(turned.view(S, T, 4, D), k_pages, v_pages, pages.tables, plan).double().cpu().numpy()
        stored = k_pages.flatten(0, 1).double().cpu().numpy()
        at = e.slots.cpu().numpy().reshape(S, T)
        want_k = paged_oracle.rotate(k.double().cpu().numpy(), e.positions.cpu().numpy(), f, interleaved=True)
        assert np.all(np.abs(stored[at.reshape(-1)] - want_k) <= 2.0**-8 * np.abs(want_k) + 2.0**-19)
        for s in range(S):
            held[s][0].extend(stored[at[s]])
            held[s][1].extend(v.view(S, T, 2, D)[s].double().cpu().numpy())
        out, mass, size = paged_oracle.attend(turned.double().cpu().numpy().reshape(S, T, 4, D), [np.stack(h[0]) for h in held],
                                              [np.stack(h[1]) for h in held], [n + T for n in before])
        assert np.all(np.abs(got - out) <= 2.0**-8 * (np.abs(out) + 1.05 * mass) + 2.0**-20)
        keep = [n + a for n, a in zip(before, accepted)]
        b.shrink(pages, i32(keep))
        held = [(h[0][:n], h[1][:n]) for h, n in zip(held, keep)]
        assert pages.lengths.tolist() == keep
        assert int(pages.free_count) == 60 - sum(-(-n // 8) for n in keep)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_the_example_searches(device, capsys):
    found = main(["--device", device.type, "--vocab", "500", "--tokens", "5"])
    assert all(len(h) == 4 and all(len(x.tokens) <= 5 for x in h) for h in found)
    assert "39 tokens:" in capsys.readouterr().out


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_a_search_longer_than_the_cache_is_refused(device):
    # (pages of 16: the room is what was asked for, not what its pages hold)
    sampler = resolve(SAMPLER, device)
    search = lambda room, tokens: beam_search(  # noqa: E731
        AttentionLM(97, requests=2, beams=2, max_tokens=room, device=device, seed=3), sampler, [[1, 2, 3], [7]], width=2, max_tokens=tokens)
    for room, tokens in ((4, 10), (4, 6), (16, 18)):
        with pytest.raises(ValueError, match="room for"):
            search(room, tokens)
    for room, tokens in ((4, 5), (1, 2), (1, 1)):  # (the last token is not decoded)
        assert [[h.tokens for h in x] for x in search(room, tokens)] == [[h.tokens for h in x] for x in search(40, tokens)]


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_a_search_of_another_width_is_refused(device):
    # as many slots, but another request's: slot 4 is the third request of two beams, the second of four
    sampler = resolve(SAMPLER, device)
    for requests, beams, width in ((4, 2, 4), (4, 2, 1), (2, 4, 2), (4, 1, 2)):
        model = AttentionLM(97, requests=requests, beams=beams, device=device, seed=3)
        with pytest.raises(ValueError, match=f"for {beams} beams"):
            beam_search(model, sampler, [[1, 2, 3]] * (requests * beams // width), width=width, max_tokens=3)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_the_decode_loop_refuses_requests_past_the_cache(device):
    sampler = resolve(SAMPLER, device)

    def run(room, tokens):
        loop = BatchDecoder(AttentionLM(97, requests=1, beams=1, max_tokens=room, device=device, seed=2), sampler, num_slots=1, max_seq_len=64)
        loop.submit([1, 2, 3], SamplingParams(temperature=0.0, max_tokens=tokens))
        return [s.token_id for s in loop.run()[0]]

    with pytest.raises(ValueError, match="room for 4"):
        run(4, 6)
    assert run(4, 5) == run(40, 5)
    model, other = (AttentionLM(97, requests=1, beams=1, max_tokens=n, device=device) for n in (8, 40))
    for target, draft in ((model, other), (other, model)):
        loop = SpeculativeDecoder(target, sampler, draft_model=draft, num_draft=3, num_slots=1, max_seq_len=64)
        with pytest.raises(ValueError, match="room for 8"):
            loop.submit([1, 2, 3], SamplingParams(temperature=0.0, max_tokens=7))
        loop.submit([1, 2, 3], SamplingParams(temperature=0.0, max_tokens=6))


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_a_prompt_that_cannot_be_planned_holds_nothing(device, monkeypatch):
    with pytest.raises(ValueError, match="max_prompt must be at most 65536"):
        make_cache(device, 1, 1, max_prompt=65537)
    make_cache(device, 1, 1, max_prompt=65536)
    cache = make_cache(device, 2, 2)
    cache.prefill(0, 100)

    def refused(*a, **k):
        raise ValueError("a shape of more tiles")

    with monkeypatch.context() as m:
        m.setattr(cache.backend, "plan", refused)
        with pytest.raises(ValueError, match="more tiles"):
            cache.prefill(2, 300)
    assert cache.prompts.lengths.tolist() == [100, 0] and int(cache.prompts.free_count) == 40 - 7
    cache.prefill(2, 300)
    assert cache.prompts.lengths.tolist() == [100, 300] and int(cache.prompts.free_count) == 40 - 7 - 19


@pytest.mark.parametrize("graphs", [False, pytest.param(True, marks=pytest.mark.gpu)], ids=["eager", "graphs"])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_the_decode_loop_waits_for_pages(device, graphs):
    # prompts of two pages each, three or six pages free: a prompt waits until others end, and no token changes
    if graphs and device.type == "cpu":
        pytest.skip("graphs need a GPU")
    sampler = resolve(SAMPLER, device)
    prompts = [list(range(1 + i, 20 + i)) for i in range(5)]

    def run(free):
        model = AttentionLM(97, requests=3, beams=1, max_prompt=32, max_tokens=12, device=device, seed=2)
        model.cache.prompts.free_count.fill_(free)  # (the others: held elsewhere)
        loop = BatchDecoder(model, sampler, num_slots=3, max_seq_len=64, graphs=graphs, graph_after=1)
        ids = [loop.submit(p, SamplingParams(temperature=0.0, max_tokens=5 + i % 3 * 3)) for i, p in enumerate(prompts)]
        done = loop.run()
        assert int(model.cache.prompts.free_count) == free and loop._free == [2, 1, 0]
        return [[s.token_id for s in done[i]] for i in ids]

    want = run(6)
    assert [len(x) for x in want] == [5, 8, 11, 5, 8]
    assert run(3) == want and run(2) == want
    model = AttentionLM(97, requests=3, beams=1, max_prompt=64, device=device, seed=2)
    model.cache.prompts.free_count.fill_(2)
    loop = BatchDecoder(model, sampler, num_slots=3, max_seq_len=64, graphs=graphs)
    loop.submit([1] * 40, SamplingParams(temperature=0.0, max_tokens=2))
    rid = loop.submit([1], SamplingParams(temperature=0.0, max_tokens=2))
    with pytest.raises(NoRoom, match="no pages"):  # (none is running whose end would make room)
        loop.step()
    assert len(loop.run()[rid]) == 2 and loop._free == [2, 1, 0]


def test_a_prefill_that_raises_costs_the_others_nothing():
    sampler = resolve(SAMPLER, torch.device("cpu"))

    class Failing(AttentionLM):
        def prefill(self, slot, prompt_ids):
            if int(prompt_ids[0]) == 96:
                raise OSError("the prompt cannot be read")
            return super().prefill(slot, prompt_ids)

    def run(prompts):
        loop = BatchDecoder(Failing(97, requests=3, beams=1, max_tokens=12, seed=2), sampler, num_slots=3, max_seq_len=64)
        ids = [loop.submit(p, SamplingParams(temperature=0.0, max_tokens=4)) for p in prompts]
        done, errors = {}, 0
        for _ in range(40):
            if not loop.busy:
                break
            try:
                for rid, s in loop.step():
                    done.setdefault(rid, []).append(s.token_id)
            except OSError:
                errors += 1
        assert not loop.busy and loop._free == [2, 1, 0]
        return [done.get(i) for i in ids], errors

    fine, errors = run([[1, 2], [3], [5, 6, 7]])
    assert errors == 0
    assert run([[1, 2], [96], [3], [96, 1], [5, 6, 7]]) == ([fine[0], None, fine[1], None, fine[2]], 2)

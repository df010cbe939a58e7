"""Beam search and distillation over vocabulary-wide logits: the operators' work as their users have it done.

Three operators, each in its plain form (elementary torch operations) and, where ``own`` is true, through the
framework's public calls:

- the selection of a beam search (``beam_select`` of a sampler backend): the best continuations of each
  request over its beams and the whole vocabulary;
- the reordering of the beams' states that follows it, in place (``prepare_reorder`` of a sampler backend);
- the distillation loss on a teacher's top logits, with its gradient (``vinfer_amd.distill``).
"""

from __future__ import annotations

import functools
import math

import torch

own = False

DEV = torch.device("cuda", 0)
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}
PAD = 0  # the token of a finished beam


# ---- cases ------------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # One request searched with four beams: a step's latency is all there is.
        _beam("beam_one", 1, 4, 151936, 4, keep=True),
        # A few requests at an odd vocabulary in fp32, some beams finished, half of the vocabulary masked by
        # a grammar; twice as many continuations as beams, as a caller asks that sorts the ended ones out.
        _beam("beam_masked_fp32", 7, 5, 50257, 10, dtype="fp32", finished=2, masked=0.5),
        # A batch of requests of an offline translation or rescoring job.
        _beam("beam_batch", 64, 4, 151936, 8),
        # Wide beams over the largest vocabulary in use.
        _beam("beam_wide", 24, 16, 262144, 16, keep=True),
        # One request's states: each layer's recurrent state, and the token histories up to the present token.
        _states("states_one", 1, 4, "recurrent", 24, heads=16, dim=64, length=1024),
        # A key and a value cache with the layers stacked, requests of very different lengths (one has none), odd
        # sizes, the beams in the order of their scores.
        _states("states_ragged", 6, 5, "stacked", 4, heads=3, dim=72, length=1023, ranked=True),
        # A batch's caches, one pair of tensors a layer, half of the beams replaced.
        _states("states_kv", 16, 4, "layers", 4, heads=8, dim=128, length=4096),
        # Many beams' recurrent states (a matrix a head), ranked: nearly every beam moves.
        _states("states_wide", 16, 8, "recurrent", 4, heads=32, dim=128, length=512, ranked=True),
        # A draft model's step on few tokens: the rows that a small fine-tuning step holds.
        _distill("distill_few", 16, 151936, 20, tail=True),
        # fp32 logits of an odd vocabulary, softened, ragged teacher entries, an eighth of the rows padding.
        _distill("distill_odd_fp32", 1000, 50257, 33, dtype="fp32", temperature=2.0, ragged=True, pad=8),
        # The loss alone, over an evaluation set's batch.
        _distill("distill_eval", 2048, 151936, 64, grad=False, tail=True),
        # A training step's tokens: loss and gradient, two rows in sixteen padding.
        _distill("distill_step", 4096, 151936, 64, pad=8),
    ]


def _beam(name, B, W, V, n, dtype="bf16", keep=False, finished=0, masked=0.0, first=False):
    return {"name": name, "kind": "beam", "B": B, "W": W, "V": V, "n": n, "dtype": dtype, "keep": keep,
            "finished": finished, "masked": masked, "first": first}


def _states(name, B, W, form, layers, heads, dim, length, ranked=False):
    return {"name": name, "kind": "states", "B": B, "W": W, "form": form, "layers": layers, "heads": heads,
            "dim": dim, "length": length, "ranked": ranked}


def _distill(name, T, V, K, dtype="bf16", temperature=1.0, tail=False, ragged=False, pad=0, grad=True):
    return {"name": name, "kind": "distill", "T": T, "V": V, "K": K, "dtype": dtype, "temperature": temperature,
            "tail": tail, "ragged": ragged, "pad": pad, "grad": grad}


def draw(rng) -> dict:
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    kind = rng.choice(("beam", "states", "distill"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    V = rng.choice((log(1000, 262144), 32000, 50257, 128256, 151936, 262144))
    if kind == "beam":
        W = rng.randint(1, 16)
        keep = rng.random() < 0.5
        n = W if keep else rng.randint(1, 2 * W)
        rows = max(1, min(400, int(2e8 / (V * SIZE[dtype]))))
        B = max(1, log(1, max(2, rows)) // W)
        c = _beam("", B, W, V, n, dtype, keep, rng.choice((0, 0, 1)) if W > 1 else 0, rng.choice((0.0, 0.0, 0.3, 0.9)),
                  rng.random() < 0.2)
    elif kind == "states":
        form = rng.choice(("recurrent", "stacked", "layers"))
        W = rng.randint(2, 12)
        heads, dim = rng.choice((1, 2, 4, 8, 16)), rng.choice((64, 72, 80, 128, 192))
        length = log(16, 4096)
        layer = heads * dim * (4 * dim if form == "recurrent" else 4 * length)  # one slot's bytes
        layers = rng.randint(1, max(1, min(16, int(1e9 / (W * layer)))))
        B = log(1, max(1, min(64, int(1e9 / (W * layers * layer)))))
        c = _states("", B, W, form, layers, heads, dim, length, rng.random() < 0.5)
    else:
        T = log(1, max(2, min(4096, int(8e8 / (V * SIZE[dtype])))))
        c = _distill("", T, V, rng.randint(1, 100), dtype, rng.choice((1.0, 1.0, 0.7, 3.0)), rng.random() < 0.5,
                     rng.random() < 0.5, rng.choice((0, 3, 8)), rng.random() < 0.8)
    del c["name"]
    return c


def work(case) -> dict:
    if case["kind"] == "beam":
        rows = case["B"] * (1 if case["first"] else case["W"] - case["finished"])
        n = rows * case["V"]
        # each live beam's logits once, its scores, the selection
        return {"bytes": n * SIZE[case["dtype"]] + 5 * case["B"] * case["W"] + 12 * case["B"] * case["n"], "flops": 4 * n}
    if case["kind"] == "states":
        B, W = case["B"], case["W"]
        # Slots written and distinct slots read, by the parents that prepare() makes: ranked, each of the better
        # half is the parent of two (one slot in W stays by chance); else the other half is replaced.
        half = (W + 1) // 2
        moved, read = (W - 1, half) if case["ranked"] else (W // 2, min(W // 2, half))
        per = sum(_slot_bytes(case, n) for n in _lengths(case))  # one slot of each request
        return {"bytes": (moved + read) * per + 4 * B * W, "flops": 0}
    live = case["T"] - (case["T"] // case["pad"] if case["pad"] else 0)
    n = live * case["V"]
    e = SIZE[case["dtype"]]
    return {"bytes": n * e + (case["T"] * case["V"] * e if case["grad"] else 0) + 8 * case["T"] * (case["K"] + 1),
            "flops": (8 if case["grad"] else 4) * n}


def _slot_bytes(case, n):
    per_layer = 4 * case["heads"] * case["dim"] ** 2 if case["form"] == "recurrent" else 4 * case["heads"] * case["dim"] * n
    return case["layers"] * per_layer + 4 * n


def _lengths(case) -> list[int]:
    """The requests' valid positions: spread from the whole length down, the fourth request's none."""
    L, B = case["length"], case["B"]
    return [0 if b % 16 == 3 else max(1, L - (b * 37 * L // 101) % L) for b in range(B)]


# ---- inputs -----------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case, **{"beam": _prepare_beam, "states": _prepare_states, "distill": _prepare_distill}[case["kind"]](case, g)}
    return s


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _prepare_beam(case, g):
    B, W, V = case["B"], case["W"], case["V"]
    rows = 1 if case["first"] else W
    x = torch.randn(B, rows, V, generator=g, device=DEV)
    # flat and certain rows both: a language model's rows are anything between
    x *= (1.0 + 3.0 * _rand(g, B, rows, 1))
    x.scatter_add_(2, torch.randint(V, (B, rows, 1), generator=g, device=DEV), 12.0 * _rand(g, B, rows, 1))
    if case["masked"]:  # a grammar allows the same tokens in each of a request's beams
        x.masked_fill_(_rand(g, B, 1, V) < case["masked"], -math.inf)
    x = x.to(DTYPES[case["dtype"]])
    scores = torch.sort(-3.0 - 2.0 * _rand(g, B, W), dim=1, descending=True).values
    finished = torch.zeros(B, W, dtype=torch.bool, device=DEV)
    if case["first"]:  # the first step: every beam has the prompt's row, and one of them is live
        x = x.expand(B, W, V)
        scores[:, 1:] = -math.inf
    elif case["finished"]:
        finished.scatter_(1, torch.argsort(_rand(g, B, W), dim=1)[:, : case["finished"]], True)
    return {"logits": x, "scores": scores, "finished": finished}


def _parents(case, g):
    B, W = case["B"], case["W"]
    relabel = torch.argsort(_rand(g, B, W), dim=1)  # which beams are the better ones
    half = (W + 1) // 2
    if case["ranked"]:  # each of the better half has two children, in any order
        p = torch.gather(relabel, 1, torch.argsort(_rand(g, B, W), dim=1) // 2)
    else:  # the better half stay, each of the others becomes another of the better half
        p = torch.empty_like(relabel)
        rank = torch.arange(W, device=DEV)
        p.scatter_(1, relabel, torch.gather(relabel, 1, torch.where(rank < half, rank, rank - half).expand(B, W)))
    return p.to(torch.int32)


def _prepare_states(case, g):
    B, W, heads, dim, L = case["B"], case["W"], case["heads"], case["dim"], case["length"]
    n = B * W
    if case["form"] == "recurrent":  # a layer's matrix a head, fp32, no length
        tensors = [(torch.randn(n, heads, dim, dim, generator=g, device=DEV), 0, None) for _ in range(case["layers"])]
    elif case["form"] == "stacked":  # keys and values, the layers in one tensor, positions inside the heads
        tensors = [(torch.randn(case["layers"], n, heads, L, dim, generator=g, device=DEV, dtype=torch.bfloat16), 1, 3)
                   for _ in range(2)]
    else:  # keys and values of each layer, positions outside the heads
        tensors = [(torch.randn(n, L, heads, dim, generator=g, device=DEV, dtype=torch.bfloat16), 0, 1)
                   for _ in range(2 * case["layers"])]
    tensors.append((torch.randint(100000, (n, L), generator=g, device=DEV, dtype=torch.int32), 0, 1))  # token histories
    return {"states": tensors, "parents": _parents(case, g),
            "lengths": torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)}


def _prepare_distill(case, g):
    T, V, K = case["T"], case["V"], case["K"]
    dtype = DTYPES[case["dtype"]]
    x = torch.empty(T, V, dtype=dtype, device=DEV)
    for i in range(0, T, 256):  # (pieces: the noise is made in 32 bits)
        x[i : i + 256] = 2.0 * torch.randn(min(256, T - i), V, generator=g, device=DEV)
    # the teacher's entries lie anywhere, and the student knows them in part
    at = torch.arange(K, device=DEV) * (V // K) + torch.randint(V // K, (T, K), generator=g, device=DEV)
    ids = torch.gather(at, 1, torch.argsort(_rand(g, T, K), dim=1))
    teacher = torch.sort(6.0 + 3.0 * torch.randn(T, K, generator=g, device=DEV), dim=1, descending=True).values
    x.scatter_(1, ids, (teacher + 2.0 * torch.randn(T, K, generator=g, device=DEV)).to(dtype))
    if case["tail"]:  # the teacher's log-probabilities: the rest of its vocabulary has a share too
        rest = torch.log(torch.tensor(float(V), device=DEV)) + _rand(g, T, 1)
        teacher = teacher - torch.logsumexp(torch.cat([teacher, rest], 1), 1, keepdim=True)
    if case["ragged"]:  # rows with fewer entries, down to one
        ids = torch.where(torch.arange(K, device=DEV) < torch.randint(1, K + 1, (T, 1), generator=g, device=DEV), ids, -1)
    weights = torch.full((T,), 1.0 / T, device=DEV)
    if case["pad"]:  # (exactly T // pad rows)
        weights[torch.argsort(_rand(g, T))[: T // case["pad"]]] = 0.0
    return {"student": x, "ids": ids.to(torch.int32), "teacher": teacher, "weights": weights}


# ---- one pass ---------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _backend(family, dtype):
    from vinfer_amd.registry import BackendContext

    if family == "distill":
        from vinfer_amd.distill import DISTILL as registry
    else:
        from vinfer_amd.sampler import SAMPLER as registry
    return registry.resolve("hip", BackendContext(DEV, DTYPES[dtype]))


def run(state):
    case = state["case"]
    if case["kind"] == "beam":
        return _run_beam(case, state)
    if case["kind"] == "states":
        return _run_states(case, state)
    return _run_distill(case, state)


def _run_beam(case, s):
    if own:
        scores, beams, tokens = _backend("sampler", case["dtype"]).beam_select(
            s["logits"], s["scores"], case["n"], finished=s["finished"], pad_id=PAD, keep_slots=case["keep"])
        return {"scores": scores, "beams": beams, "tokens": tokens}
    B, W, V, n = case["B"], case["W"], case["V"], case["n"]
    # The first step's beams but one are dead and read nothing (all have the same row).
    rows = 1 if case["first"] else W
    x = s["logits"][:, :rows]
    # each beam's n best by its logits, the lower id first among equals: unique whole keys (ordered bits, id)
    k = min(n, V)
    bits = (x + 0.0).float().view(torch.int32)  # (-0 counts as 0)
    keys = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64) << 32
    keys += (V - 1) - torch.arange(V, device=DEV)
    top = torch.topk(keys, k, dim=2).values
    ids = (V - 1) - (top & 0xFFFFFFFF)
    # log-probabilities and scores in 64 bits: beams are compared across their rows
    xd = x.double()
    m = xd.amax(2, keepdim=True)
    lse = m + torch.log(torch.exp(xd - m).sum(2, keepdim=True))
    score = s["scores"][:, :rows, None].double()
    cand = torch.gather(xd, 2, ids) - lse + score
    cand = torch.where(cand.isnan(), -math.inf, cand)  # (a row without a finite logit has no candidates)
    fin = s["finished"][:, :rows, None]
    alone = torch.arange(k, device=DEV) == 0
    cand = torch.where(fin, torch.where(alone, score, -math.inf), cand)
    ids = torch.where(fin, PAD, ids)
    beams = torch.arange(rows, device=DEV)[:, None].expand(B, rows, k)
    best, at = torch.sort(cand.reshape(B, rows * k), dim=1, descending=True, stable=True)
    none = best == -math.inf
    tokens = torch.where(none, -1, torch.gather(ids.reshape(B, -1), 1, at))
    beams = torch.where(none, -1, torch.gather(beams.reshape(B, -1), 1, at))
    # where there are fewer candidates than asked for, the rest is empty
    short = max(0, n - rows * k)
    pad = lambda t, v: torch.nn.functional.pad(t[:, :n], (0, short), value=v)  # noqa: E731
    best, beams, tokens = pad(best, -math.inf), pad(beams, -1), pad(tokens, -1)
    if case["keep"]:
        # a parent's best child takes its place; the others take the free places in their order
        i = torch.arange(n, device=DEV)
        same = (beams[:, :, None] == beams[:, None, :]) & (i[:, None] > i)  # an earlier child of the same parent
        stays = (beams >= 0) & ~same.any(2)
        taken = torch.zeros(B, n, dtype=torch.int64, device=DEV)
        taken.scatter_add_(1, beams.clamp(min=0), stays.long())
        free = torch.argsort(taken, dim=1, stable=True)  # free places first, ascending
        order = torch.cumsum(~stays, 1) - 1
        place = torch.where(stays, beams, torch.gather(free, 1, order.clamp(min=0)))
        put = lambda t: torch.empty_like(t).scatter_(1, place, t)  # noqa: E731
        best, beams, tokens = put(best), put(beams), put(tokens)
    return {"scores": best.float(), "beams": beams.to(torch.int32), "tokens": tokens.to(torch.int32)}


def _run_states(case, s):
    tensors = s["states"]
    if own:
        if "plan" not in s:
            from vinfer_amd.sampler import BeamState

            s["plan"] = _backend("sampler", "bf16").prepare_reorder(
                [BeamState(t, slot_dim, length_dim) for t, slot_dim, length_dim in tensors], case["B"], case["W"])
        s["plan"].launch(s["parents"], s["lengths"])
        return [t for t, _, _ in tensors]
    B, W = case["B"], case["W"]
    source = (torch.arange(B, device=DEV)[:, None] * W + s["parents"]).reshape(-1)
    lengths = s["lengths"].repeat_interleave(W)
    for t, slot_dim, length_dim in tensors:
        new = t.index_select(slot_dim, source)
        if length_dim is None:
            t.copy_(new)
            continue
        shape = [1] * t.dim()
        shape[slot_dim], shape[length_dim] = B * W, t.shape[length_dim]
        inside = torch.arange(t.shape[length_dim], device=DEV) < lengths[:, None]
        t.copy_(torch.where(inside.view(shape), new, t))
    return [t for t, _, _ in tensors]


def _run_distill(case, s):
    x, ids, teacher, weights = s["student"], s["ids"], s["teacher"], s["weights"]
    if own:
        d = _backend("distill", case["dtype"])
        if not case["grad"]:
            return {"loss": d.loss(x, ids, teacher, weights, temperature=case["temperature"], tail=case["tail"])}
        loss, grad = d.loss_and_grad(x, ids, teacher, weights, temperature=case["temperature"], tail=case["tail"])
        return {"loss": loss, "grad": grad}
    t = case["temperature"]
    there = ids >= 0
    at = ids.clamp(min=0).long()
    # the teacher's probabilities, and the share of the ids that it does not list
    if case["tail"]:
        logp = torch.where(there, teacher, -math.inf)
    else:
        logp = torch.log_softmax(torch.where(there, teacher / t, -math.inf), 1)
    p = torch.exp(logp)
    rest = (1 - p.double().sum(1)).clamp(min=0).float() if case["tail"] else torch.zeros_like(weights)
    z = x.float() / t
    z -= z.amax(1, keepdim=True)
    logq = torch.gather(z, 1, at)
    e = torch.exp_(z)
    listed_e = torch.where(there, torch.gather(e, 1, at), 0.0)
    if case["tail"]:  # the mass outside the list by itself: 1 - Q loses it where Q is near 1
        hit = torch.where(there, at, at[:, :1])  # (the first entry is always there)
        outside = e.scatter(1, hit, 0.0).sum(1)
        total = outside + listed_e.sum(1)
    else:
        total = e.sum(1)
    logq = logq - torch.log(total)[:, None]
    loss = torch.where(there, torch.special.xlogy(p, p) - p * logq, 0.0).sum(1)
    if case["tail"]:
        q_rest = outside / total
        loss = loss + torch.special.xlogy(rest, rest) - torch.special.xlogy(rest, q_rest)
    loss = torch.where(weights == 0, 0.0, weights * loss)
    if not case["grad"]:
        return {"loss": loss}
    mass = p.sum(1) + rest
    scale = (weights / t)[:, None]
    q = e.div_(total[:, None])
    if case["tail"]:
        listed_q = torch.where(there, torch.gather(q, 1, at), 0.0)
        grad = q * ((mass - rest / q_rest)[:, None] * scale)
        value = (listed_q * mass[:, None] - p) * scale
        grad.scatter_(1, hit, torch.where(there, value, value[:, :1]))
    else:
        grad = q.mul_(mass[:, None] * scale)
        grad.scatter_add_(1, at, torch.where(there, -p * scale, 0.0))
    return {"loss": loss, "grad": grad.to(x.dtype)}


# ---- the definitions, in 64 bits --------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"beam": _exact_beam, "states": _exact_states, "distill": _exact_distill}[case["kind"]](case, s)


def _exact_beam(case, s):
    """Request by request: every candidate's score, all of them sorted."""
    B, W, V, n = case["B"], case["W"], case["V"], case["n"]
    out = {"scores": torch.full((B, n), -math.inf, dtype=torch.float64), "beams": torch.full((B, n), -1, dtype=torch.int32),
           "tokens": torch.full((B, n), -1, dtype=torch.int32)}
    for b in range(B):
        lp = torch.log_softmax(s["logits"][b].double(), 1) + s["scores"][b].double()[:, None]
        lp[lp.isnan()] = -math.inf  # (a row without a finite logit has no candidates)
        for w in torch.nonzero(s["finished"][b]).flatten().tolist():
            lp[w] = -math.inf
            lp[w, PAD] = s["scores"][b, w].double()
        best, at = torch.sort(lp.flatten(), descending=True, stable=True)
        chosen = [(v, i // V, i % V) for v, i in zip(best[:n].tolist(), at[:n].tolist()) if v > -math.inf]
        places = list(range(n))
        if case["keep"]:
            where: dict[int, int] = {}  # the place of each parent's best child
            for i, (_, w, _) in enumerate(chosen):
                where.setdefault(w, i)
            stay = {i: w for w, i in where.items()}
            free = [k for k in range(n) if k not in where]
            places = [stay[i] if i in stay else free.pop(0) for i in range(n)]
        for i, (v, w, t) in enumerate(chosen):
            out["scores"][b, places[i]], out["beams"][b, places[i]], out["tokens"][b, places[i]] = v, w, t
    return out


def _exact_states(case, s):
    """Copies have no rounding: slot by slot from a copy of what was there."""
    W = case["W"]
    parents, lengths = s["parents"].tolist(), s["lengths"].tolist()
    for t, slot_dim, length_dim in s["states"]:
        old = t.clone()
        for b, row in enumerate(parents):
            for w, p in enumerate(row):
                dst, src = t.select(slot_dim, b * W + w), old.select(slot_dim, b * W + p)
                if length_dim is not None:
                    d = length_dim - (length_dim > slot_dim)
                    dst, src = dst.narrow(d, 0, lengths[b]), src.narrow(d, 0, lengths[b])
                dst.copy_(src)
    return [t for t, _, _ in s["states"]]


def _exact_distill(case, s):
    """From log-softmax over the whole row, a few rows at a time."""
    t = case["temperature"]
    losses, grads = [], []
    for i in range(0, case["T"], 64):
        x, ids = s["student"][i : i + 64].double(), s["ids"][i : i + 64].long()
        w, there = s["weights"][i : i + 64].double(), s["ids"][i : i + 64] >= 0
        # the target's distribution over the vocabulary, the unlisted rest apart
        teacher = s["teacher"][i : i + 64].double()
        target = torch.zeros_like(x)
        p = torch.exp(teacher) if case["tail"] else torch.exp(teacher / t)
        p = torch.where(there, p, 0.0)
        if not case["tail"]:
            p = p / p.sum(1, keepdim=True)
        target.scatter_add_(1, ids.clamp(min=0), p)
        member = torch.zeros_like(x).scatter_add_(1, ids.clamp(min=0), there.double()) > 0
        logq = torch.log_softmax(x / t, 1)
        q = torch.exp(logq)
        loss = (torch.special.xlogy(target, target) - target * logq).sum(1)
        grad = q * target.sum(1, keepdim=True) - target
        if case["tail"]:
            rest = (1 - target.sum(1)).clamp(min=0)
            q_rest = torch.where(member, 0.0, q).sum(1)
            loss = loss + torch.special.xlogy(rest, rest) - rest * torch.log(q_rest)
            # d(-rest log q_rest)/dz_j = rest q_j - (rest q_j / q_rest outside the list)
            grad = grad + rest[:, None] * q - torch.where(member, 0.0, q * (rest / q_rest)[:, None])
        losses.append(w * loss)
        if case["grad"]:
            grads.append((w / t)[:, None] * grad)
            if case["dtype"] == "bf16":  # (64 bits of the largest gradient would not fit beside the rest)
                grads[-1] = grads[-1].float()
    loss = torch.cat(losses)
    return {"loss": loss, "grad": torch.cat(grads)} if case["grad"] else {"loss": loss}

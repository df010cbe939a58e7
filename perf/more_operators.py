"""A paged cache that sequences share, and the attention that reads it: the operators' work as their users have it done.

Three operators, each in its plain form (elementary torch operations) and, where ``own`` is true, through the
framework's public calls (``vinfer_amd.paged``):

- the page tables of growing sequences, built on the GPU from their lengths (``extend``, and ``shrink``, which takes
  back what a step did not keep);
- the rotation of queries and keys by their positions, and the keys' and values' way into their pages
  (``rotate_store``);
- the attention of sequences in groups that share a prefix, read once for a whole group (``plan`` for a step,
  ``attend`` for each layer).
"""

from __future__ import annotations

import functools
import math

import torch

own = False

DEV = torch.device("cuda", 0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # One request's beams take a step: the call's latency is all there is.
        _tables("tables_one", 4, 2000, "step"),
        # A batch's verification step: each sequence five drafted tokens, some sequences pausing, all taken back.
        _tables("tables_drafts", 256, 8000, "drafts", idle=8),
        # Prompts of very different lengths join; small pages; the last ones find no room.
        _tables("tables_prompts", 96, 6000, "prompts", page=16, tight=True),
        # One request's beams: four tokens of a model of 32 query and 8 key heads.
        _rotate("rotate_one", 4, 32, 8, 128),
        # Part of an odd head, interleaved, far positions of a stretched context, some tokens padding.
        _rotate("rotate_odd", 1003, 9, 3, 72, dtype="fp16", dim=36, interleaved=True, scaling=8.0, far=700000, pad=16),
        # A prompt's tokens.
        _rotate("rotate_prompt", 16384, 32, 8, 128, scaling=4.0, far=100000),
        # One request's four beams on their prompt, two layers.
        _attend("attend_one", 1, 4, 1, 32, 8, 128, 1000, 40, layers=2),
        # Groups of any size, three query heads a key head, sequences and prefixes of no length, drafted tokens.
        _attend("attend_odd", 9, 5, 3, 9, 3, 72, 1500, 300, dtype="fp16", ragged=True, layers=2),
        # A batch of requests searched with four beams each.
        _attend("attend_beams", 64, 4, 1, 32, 8, 128, 8192, 200, layers=2),
        # Every sequence of a batch behind one long system prompt: the prefix is a matrix product.
        _attend("attend_system", 1, 192, 1, 32, 8, 128, 32768, 1024),
        # A few sequences of their own, long, with four drafted tokens to verify; a large page.
        _attend("attend_long", 4, 1, 5, 64, 8, 128, 0, 100000, page=64),
        # Pieces of four requests' prompts behind what they share.
        _attend("attend_prompts", 1, 4, 384, 16, 4, 256, 4000, 2000, page=32),
    ]


def _tables(name, S, length, kind, page=16, idle=0, tight=False):
    return {"name": name, "kind": "tables", "S": S, "length": length, "step": kind, "page": page, "idle": idle, "tight": tight}


def _rotate(name, N, heads, kv_heads, head_dim, dtype="bf16", dim=None, interleaved=False, scaling=1.0, far=8192, pad=0,
            page=16):
    return {"name": name, "kind": "rotate", "N": N, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": dtype, "dim": dim or head_dim, "interleaved": interleaved, "scaling": scaling, "far": far, "pad": pad,
            "page": page}


def _attend(name, B, W, T, heads, kv_heads, head_dim, prefix, length, dtype="bf16", ragged=False, page=16, layers=1):
    return {"name": name, "kind": "attend", "B": B, "W": W, "T": T, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "prefix": prefix, "length": length, "dtype": dtype, "ragged": ragged, "page": page,
            "layers": layers}


def draw(rng) -> dict:
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))  # noqa: E731
    kind = rng.choice(("tables", "rotate", "attend", "attend"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    page = rng.choice((8, 16, 16, 32, 64, 128))
    if kind == "tables":
        step = rng.choice(("step", "drafts", "prompts"))
        S = log(1, 128 if step == "prompts" else 2048)
        length = log(20, min(16000, 4_000_000 // S))
        c = _tables("", S, length, step, page, rng.choice((0, 0, 8)), rng.random() < 0.3)
    elif kind == "rotate":
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 7, 8))
        D = rng.choice((64, 72, 80, 128, 128, 192, 256))
        N = log(1, min(16384, 100_000_000 // (D * (heads + 2 * kv_heads))))
        c = _rotate("", N, heads, kv_heads, D, dtype, rng.choice((None, D // 2, D // 4)), rng.random() < 0.5,
                    rng.choice((1.0, 1.0, 4.0, 32.0)), log(N, 1_000_000), rng.choice((0, 0, 8)), page)
    else:
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        G = rng.choice((1, 2, 3, 4, 5, 8))
        D = rng.choice((64, 72, 80, 128, 128, 192, 256))
        T = rng.choice((1, 1, 1, 2, 4, 5, log(6, 300)))
        B, W, layers = log(1, 64), log(1, 64), rng.choice((1, 2))
        B = max(1, min(B, 400 // W, 8000 // (W * T)))
        # (a ragged batch has up to twice the sequences) what a position costs in bytes, and in a part's operations
        row, each = 8 * layers * kv_heads * D, 8 * layers * B * W * T * G * kv_heads * D
        ragged = rng.random() < 0.5
        prefix = min(rng.choice((0, log(1, 50000))), int(8e8 / (B * row)), int(5e10 / each))
        length = min(T + log(1, 8000), max(T, int(8e8 / (B * W * row))), max(T, int(5e10 / each)))
        c = _attend("", B, W, T, kv_heads * G, kv_heads, D, prefix, length, dtype, ragged, page, layers)
    del c["name"]
    return c


def _spread(n, top, low, empty=True):
    """n lengths from ``top`` down, the fourth of each sixteen none."""
    return [0 if empty and i % 16 == 3 else max(low, top - (i * 37 * top // 101) % max(1, top)) for i in range(n)]


def _sizes(case):
    """What a tables case asks for: each sequence's length before, its new tokens, and their total."""
    S = case["S"]
    if case["step"] == "prompts":  # every second sequence is new
        lengths = [0 if i % 2 else n for i, n in enumerate(_spread(S, case["length"] // 2, 1))]
        counts = [n if i % 2 else 0 for i, n in enumerate(_spread(S, case["length"], 1, empty=False))]
    else:
        lengths = _spread(S, case["length"], 1)
        counts = [5 if case["step"] == "drafts" else 1] * S
    if case["idle"]:
        counts = [0 if i % case["idle"] == 5 else n for i, n in enumerate(counts)]
    return lengths, counts, max(1, sum(counts))


def _groups(case):
    """The groups' sequence counts (ragged: others than W, one of them none where there are enough)."""
    B, W = case["B"], case["W"]
    if not case["ragged"] or B == 1:
        return [W] * B
    return [0 if g == 2 else 1 + (W * (g + 1) * 5 // 7) % (2 * W) for g in range(B)]


def _keys(case):
    """Prefix length of each group and own length of each sequence (new tokens included)."""
    prefixes = _spread(case["B"], case["prefix"], 1, case["ragged"]) if case["prefix"] else [0] * case["B"]
    return prefixes, _spread(sum(_groups(case)), case["length"], min(case["T"], case["length"]), case["ragged"])


def work(case) -> dict:
    if case["kind"] == "tables":
        lengths, counts, N = _sizes(case)
        page = case["page"]
        pages = sum(-(-(n + c) // page) - -(-n // page) for n, c in zip(lengths, counts))
        # lengths and counts; the pages taken and entered, and given back; each token's slot, position and sequence
        return {"bytes": 24 * case["S"] + 16 * pages + 12 * N, "flops": 4 * N}
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "rotate":
        N = case["N"] - (case["N"] // case["pad"] if case["pad"] else 0)
        n = N * (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        return {"bytes": 2 * n * size + 8 * case["N"], "flops": 3 * N * (case["heads"] + case["kv_heads"]) * case["dim"]}
    groups, (prefixes, lengths) = _groups(case), _keys(case)
    T, D = case["T"], case["head_dim"]
    keys = sum(p for p, w in zip(prefixes, groups) if w) + sum(lengths)
    pairs = sum(p * w * T for p, w in zip(prefixes, groups))  # (query, key) pairs a head
    pairs += sum(sum(max(0, n - T + t + 1) for t in range(T)) for n in lengths)
    each = 2 * keys * case["kv_heads"] * D + 2 * sum(groups) * T * case["heads"] * D
    return {"bytes": case["layers"] * each * size, "flops": case["layers"] * 4 * pairs * case["heads"] * D}


# ---- inputs -----------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    make = {"tables": _prepare_tables, "rotate": _prepare_rotate, "attend": _prepare_attend}[case["kind"]]
    return {"case": case, **make(case, g)}


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _shuffled(g, n):
    return torch.argsort(_rand(g, n)).to(torch.int32)


def _paged(g, lengths, page, wide, shuffled, first):
    """Tables of ``wide`` pages for sequences of these lengths, from ``shuffled[first:]``; the next page unused."""
    tables = torch.zeros(len(lengths), wide, dtype=torch.int32, device=DEV)
    have = (torch.tensor(lengths, device=DEV) + page - 1) // page
    inside = torch.arange(wide, device=DEV) < have[:, None]
    n = sum(-(-x // page) for x in lengths)
    tables[inside] = shuffled[first : first + n]
    return tables, first + n


def _prepare_tables(case, g):
    lengths, counts, N = _sizes(case)
    page = case["page"]
    used = sum(-(-n // page) for n in lengths)
    need = sum(-(-(n + c) // page) - -(-n // page) for n, c in zip(lengths, counts))
    pages = used + (need * 7 // 8 if case["tight"] else need + 64)
    wide = max(-(-(n + c) // page) for n, c in zip(lengths, counts)) + 3
    shuffled = _shuffled(g, pages)
    tables, at = _paged(g, lengths, page, wide, shuffled, 0)
    free = torch.zeros(pages, dtype=torch.int32, device=DEV)
    free[: pages - at] = shuffled[at:]
    return {"tables": tables, "lengths": _int(lengths), "before": _int(lengths), "counts": _int(counts), "free": free,
            "free_count": _int([pages - at]), "N": N}


def _prepare_rotate(case, g):
    N, heads, kv_heads, D, page = case["N"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    # queries, keys and values come out of one product
    fused = _randn(g, N, (heads + 2 * kv_heads) * D, dtype=dtype)
    q, k, v = (t.unflatten(1, (-1, D)) for t in fused.split([heads * D, kv_heads * D, kv_heads * D], 1))
    # a prompt's positions run on; a batch's lie anywhere
    if N > 2048:
        positions = torch.arange(N, device=DEV) + case["far"] - N
    else:
        positions = (_rand(g, N) * case["far"]).long()
    pages = -(-N // page) + 5
    slots = (_shuffled(g, pages)[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)[:N]
    if case["pad"]:
        out = torch.argsort(_rand(g, N))[: N // case["pad"]]
        positions[out], slots[out] = -1, -1
    # rotations slower than half a turn over the trained length are stretched, the fast ones stay
    dim, base, stretch, trained = case["dim"], 500000.0, case["scaling"], 8192
    freq = base ** -(torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim)
    keep = ((trained * freq / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
    freq = (1 - keep) * freq / stretch + keep * freq
    return {"q": q, "k": k, "v": v, "positions": positions.to(torch.int32), "slots": slots.to(torch.int32),
            "frequencies": freq, "magnitude": 0.1 * math.log(stretch) + 1.0,
            "k_pages": torch.zeros(pages, page, kv_heads, D, dtype=dtype, device=DEV),
            "v_pages": torch.zeros(pages, page, kv_heads, D, dtype=dtype, device=DEV)}


def _prepare_attend(case, g):
    T, heads, kv_heads, D, page = case["T"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    groups, (prefixes, lengths) = _groups(case), _keys(case)
    S = sum(groups)
    pages = sum(-(-n // page) for n in prefixes + lengths) + 3
    shuffled = _shuffled(g, pages)
    prefix_tables, at = _paged(g, prefixes, page, -(-max(prefixes) // page) + 1, shuffled, 0)
    tables, at = _paged(g, lengths, page, -(-max(lengths) // page) + 1, shuffled, at)
    starts = [0]
    for w in groups:
        starts.append(starts[-1] + w)
    cache = [[_randn(g, pages, page, kv_heads, D, dtype=dtype) for _ in range(2)] for _ in range(case["layers"])]
    # heads that look at everything, and heads that look at few keys
    sharp = 0.5 + 3.0 * _rand(g, 1, 1, heads, 1)
    q = [(_randn(g, S, T, heads, D) * sharp).to(dtype) for _ in range(case["layers"])]
    return {"q": q, "cache": cache, "tables": tables, "prefix_tables": prefix_tables, "lengths": _int(lengths),
            "prefix_lengths": _int(prefixes), "starts": _int(starts), "widest": max(groups)}


# ---- one pass ---------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _backend(dtype):
    from vinfer_amd.paged import PAGED
    from vinfer_amd.registry import BackendContext

    return PAGED.resolve("hip", BackendContext(DEV, DTYPES[dtype]))


def run(state):
    case = state["case"]
    return {"tables": _run_tables, "rotate": _run_rotate, "attend": _run_attend}[case["kind"]](case, state)


def _run_tables(case, s):
    """A step's pages, and all of it taken back (a draft that is refused, a request that is cancelled)."""
    if own:
        if "pages" not in s:
            from vinfer_amd.paged import PageTables

            s["pages"] = PageTables(s["tables"], s["lengths"], s["free"], s["free_count"], case["page"])
        b = _backend("bf16")
        e = b.extend(s["pages"], s["counts"], s["N"])
        b.shrink(s["pages"], s["before"])
        slots, positions, sequences, served = e.slots, e.positions, e.sequences, e.served
    else:
        slots, positions, sequences, served = _extend(case, s)
        _shrink(case, s)
    return {"slots": slots, "positions": positions, "sequences": sequences, "served": served, "tables": s["tables"],
            "lengths": s["lengths"], "free": s["free"], "free_count": s["free_count"]}


def _extend(case, s):
    page, tables, lengths, free, N = case["page"], s["tables"], s["lengths"].long(), s["free"], s["N"]
    wide = tables.shape[1]
    counts = s["counts"].long().clamp(min=0)
    have = (lengths + page - 1) // page
    need = (lengths + counts + page - 1) // page - have
    ends = torch.cumsum(counts, 0)
    fits = (have + need <= wide) & (ends <= N)
    need = torch.where(fits, need, 0)
    upto = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (upto <= s["free_count"]))
    # the i-th page that the call takes is the i-th from the stack's top
    column = torch.arange(wide, device=DEV)
    new = served[:, None] & (column >= have[:, None]) & (column < (have + need)[:, None])
    taken = (upto - need)[:, None] + column - have[:, None]
    at = (s["free_count"] - 1 - taken).clamp(0, free.shape[0] - 1)
    tables.copy_(torch.where(new, free[at], tables))
    i = torch.arange(N, device=DEV)
    sequence = torch.searchsorted(ends, i, right=True).clamp(max=lengths.shape[0] - 1)
    position = lengths[sequence] + i - (ends - counts)[sequence]
    valid = (i < ends[-1]) & served[sequence]
    slot = tables[sequence, (position // page).clamp(0, wide - 1)].long() * page + position % page
    s["lengths"].add_(torch.where(served, counts, 0))
    s["free_count"].sub_(torch.where(served, need, 0).sum())
    whole = lambda t: torch.where(valid, t, -1).to(torch.int32)  # noqa: E731
    return whole(slot), whole(position), whole(sequence), served


def _shrink(case, s):
    page, tables, free = case["page"], s["tables"], s["free"]
    new = torch.minimum(s["lengths"], s["before"].clamp(min=0)).long()
    have, keep = (s["lengths"].long() + page - 1) // page, (new + page - 1) // page
    drop = have - keep
    upto = torch.cumsum(drop, 0)
    column = torch.arange(tables.shape[1], device=DEV)
    back = (column >= keep[:, None]) & (column < have[:, None])
    at = s["free_count"] + upto[-1] - 1 - ((upto - drop)[:, None] + column - keep[:, None])
    free[at[back]] = tables[back]
    s["free_count"].add_(upto[-1])
    s["lengths"].copy_(new)


def _run_rotate(case, s):
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        if "rotary" not in s:
            from vinfer_amd.paged import Rotary

            s["rotary"] = Rotary(s["frequencies"], interleaved=case["interleaved"], magnitude=s["magnitude"])
        out = _backend(case["dtype"]).rotate_store(q, k, v, s["positions"], s["slots"], s["k_pages"], s["v_pages"],
                                                   s["rotary"])
        return {"q": out, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    angle = s["positions"].double()[:, None] * s["frequencies"]  # (far positions need 64 bits)
    cos, sin = ((f(angle) * s["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))

    def turn(x):
        d = case["dim"]
        a, rest = x[..., :d].float(), x[..., d:]
        if case["interleaved"]:
            x1, x2 = a[..., 0::2], a[..., 1::2]
            y = torch.stack([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1).flatten(-2)
        else:
            x1, x2 = a[..., : d // 2], a[..., d // 2 :]
            y = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
        return torch.cat([y.to(x.dtype), rest], -1)

    used = s["slots"] >= 0
    at = s["slots"][used].long()
    s["k_pages"].flatten(0, 1)[at] = turn(k)[used]
    s["v_pages"].flatten(0, 1)[at] = v[used]
    return {"q": torch.where((s["positions"] >= 0)[:, None, None], turn(q), 0), "k_pages": s["k_pages"],
            "v_pages": s["v_pages"]}


def _run_attend(case, s):
    """A step's plan, and every layer's attention."""
    if own:
        b = _backend(case["dtype"])
        plan = b.plan(s["lengths"], queries=case["T"], heads=case["heads"], kv_heads=case["kv_heads"],
                      head_dim=case["head_dim"], page_size=case["page"], max_pages=s["tables"].shape[1],
                      prefix_lengths=s["prefix_lengths"], max_prefix_pages=s["prefix_tables"].shape[1],
                      group_starts=s["starts"])
        return [b.attend(q, k, v, s["tables"], plan, prefix_tables=s["prefix_tables"])
                for q, (k, v) in zip(s["q"], s["cache"])]
    return [_attention(case, s, q, k, v) for q, (k, v) in zip(s["q"], s["cache"])]


def _attention(case, s, q, k, v):
    T, Hkv, D, page = case["T"], case["kv_heads"], case["head_dim"], case["page"]
    G = case["heads"] // Hkv
    S, B, W = q.shape[0], case["B"], s["widest"]
    starts = s["starts"].long()

    def cached(pages, tables):  # [rows, Hkv, positions, D]
        return pages[tables.long()].flatten(1, 2).transpose(1, 2).float().contiguous()

    rows = (q.float() * D**-0.5).view(S, T, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hkv, T * G, D)
    # the sequence's own keys: a token sees those up to its own
    own_scores = torch.matmul(rows, cached(k, s["tables"]).transpose(2, 3).contiguous())
    L = own_scores.shape[-1]
    seen = torch.arange(L, device=DEV) < (s["lengths"][:, None] - T + 1 + torch.arange(T, device=DEV))[:, :, None]
    seen = seen.repeat_interleave(G, 1)[:, None]  # [S, 1, T G, L]
    own_scores = torch.where(seen, own_scores, -math.inf)
    # the groups' rows side by side: all of a group's sequences on its prefix
    place = starts[:-1, None] + torch.arange(W, device=DEV)
    there = place < starts[1:, None]
    grouped = rows[place.clamp(max=S - 1)].transpose(1, 2).reshape(B, Hkv, W * T * G, D)
    scores = torch.matmul(grouped, cached(k, s["prefix_tables"]).transpose(2, 3).contiguous())
    P = scores.shape[-1]
    scores = torch.where((torch.arange(P, device=DEV) < s["prefix_lengths"][:, None])[:, None, None], scores, -math.inf)
    # a row without own keys that it may see is not a token: it sees nothing at all
    alive = torch.arange(T, device=DEV) >= T - s["lengths"][:, None]
    # both parts' largest, first in the groups' order, then in the sequences'
    back = torch.empty(S, dtype=torch.int64, device=DEV)
    back[place[there]] = torch.arange(B * W, device=DEV).view(B, W)[there]

    def apart(t):  # [B, Hkv, W T G, n] -> [S, Hkv, T G, n]
        return t.view(B, Hkv, W, T * G, -1).transpose(1, 2).reshape(B * W, Hkv, T * G, -1)[back]

    most = torch.maximum(apart(scores.amax(3, keepdim=True)), own_scores.amax(3, keepdim=True))
    most = torch.where(most == -math.inf, 0.0, most)
    together = torch.zeros(B * W, Hkv, T * G, 1, device=DEV).index_copy_(0, back, most)
    together = together.view(B, W, Hkv, T * G, 1).transpose(1, 2).reshape(B, Hkv, W * T * G, 1)
    e, own_e = torch.exp(scores - together), torch.exp(own_scores - most)
    total = apart(e.sum(3, keepdim=True)) + own_e.sum(3, keepdim=True)
    value = apart(torch.matmul(e, cached(v, s["prefix_tables"]))) + torch.matmul(own_e, cached(v, s["tables"]))
    out = torch.where(total > 0, value / total, 0.0).view(S, Hkv, T, G, D).permute(0, 2, 1, 3, 4)
    return torch.where(alive[:, :, None, None, None], out, 0.0).reshape(S, T, Hkv * G, D).to(q.dtype)


# ---- the definitions, in 64 bits --------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "tables":  # (whole numbers)
        return None
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "attend": _exact_attend}[case["kind"]](case, s)


def _exact_rotate(case, s):
    """As products of complex numbers."""
    d = case["dim"]
    turn = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device=DEV),
                       s["positions"].double()[:, None, None] * s["frequencies"])

    def rotated(x):
        y = x.double().clone()
        pairs = y[..., :d].unflatten(-1, (d // 2, 2) if case["interleaved"] else (2, d // 2))
        if not case["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        y[..., :d] = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        return y

    q = rotated(s["q"])
    q[s["positions"] < 0] = 0.0
    k_pages, v_pages = (t.double().flatten(0, 1) for t in (s["k_pages"], s["v_pages"]))
    rows = torch.nonzero(s["slots"] >= 0).flatten()
    k_pages[s["slots"][rows].long()] = rotated(s["k"])[rows]
    v_pages[s["slots"][rows].long()] = s["v"].double()[rows]
    return {"q": q, "k_pages": k_pages.view(s["k_pages"].shape), "v_pages": v_pages.view(s["v_pages"].shape)}


def _exact_attend(case, s):
    """Sequence by sequence where they are short, a group's prefix with all of its sequences at once."""
    T, Hkv, D, page = case["T"], case["kv_heads"], case["head_dim"], case["page"]
    starts, prefixes, lengths = s["starts"].tolist(), s["prefix_lengths"].tolist(), s["lengths"].tolist()
    outs = []
    for q, (k_pages, v_pages) in zip(s["q"], s["cache"]):
        S, _, H, _ = q.shape
        G = H // Hkv
        out = torch.zeros(S, T, H, D, dtype=torch.float64, device=DEV)

        def read(pages, table, n):  # [Hkv, n, D]
            return pages[table[: -(-n // page)].long()].flatten(0, 1)[:n].double().transpose(0, 1)

        for b in range(case["B"]):
            lo, hi = starts[b], starts[b + 1]
            if lo == hi:
                continue
            x = q[lo:hi].double().view(hi - lo, T, Hkv, G, D).permute(2, 0, 1, 3, 4).reshape(Hkv, -1, D) / math.sqrt(D)
            pk, pv = (read(t, s["prefix_tables"][b], prefixes[b]) for t in (k_pages, v_pages))
            # the prefix's sums, and its rows' logs of them
            z = torch.bmm(x, pk.transpose(1, 2).contiguous())
            log_p = torch.logsumexp(z, 2) if prefixes[b] else torch.full_like(x[..., 0], -math.inf)
            o_p = torch.bmm(torch.softmax(z, 2), pv)
            del z
            log_p, o_p, x = (t.view(Hkv, hi - lo, T, G, *t.shape[2:]) for t in (log_p, o_p, x))
            for i in range(hi - lo):
                n = lengths[lo + i]
                if n == 0:
                    continue
                ok, ov = (read(t, s["tables"][lo + i], n) for t in (k_pages, v_pages))
                z = torch.bmm(x[:, i].reshape(Hkv, T * G, D), ok.transpose(1, 2).contiguous()).view(Hkv, T, G, n)
                hidden = torch.arange(n, device=DEV)[None, :] > (n - T + torch.arange(T, device=DEV))[:, None]
                z.masked_fill_(hidden[None, :, None], -math.inf)
                z = torch.cat([log_p[:, i, ..., None], z], -1)
                w = torch.nan_to_num(torch.softmax(z, -1))  # (rows before a short sequence's first token)
                o = w[..., :1] * o_p[:, i] + torch.bmm(w[..., 1:].reshape(Hkv, T * G, n), ov).view(Hkv, T, G, D)
                o[:, : max(0, T - n)] = 0.0
                out[lo + i] = o.permute(1, 0, 2, 3).reshape(T, H, D)
        outs.append(out)
    return outs

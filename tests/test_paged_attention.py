"""Attention of sequences behind shared prefixes (``plan``, ``attend``): the reference backend and the hip kernels
against softmaxes in 64 bits, a row at a time."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import paged_oracle
from vinfer_amd.paged import PAGED
from vinfer_amd.registry import BackendContext

GPU = torch.device("cuda", 0)
DEVICES = [torch.device("cpu"), pytest.param(GPU, marks=pytest.mark.gpu)]
BF16, F16 = torch.bfloat16, torch.float16


def backend(device, dtype):
    return PAGED.resolve("hip" if device.type == "cuda" else "reference", BackendContext(device, dtype))


class Case:
    """A cache of random pages, groups (sequences of each, prefix of each) and the sequences' own lengths."""

    def __init__(self, device, dtype, groups, lengths, *, T=1, heads=4, kv_heads=2, D=64, page=16, order="places", seed=0,
                 spread=1.0, extra=1):
        rng = np.random.default_rng(seed)
        self.device, self.dtype, self.page = device, dtype, page
        self.T, self.heads, self.kv_heads, self.D = T, heads, kv_heads, D
        self.lengths, self.prefixes = list(lengths), [p for _, p in groups] if groups else None
        S = len(self.lengths)
        self.starts = np.cumsum([0] + [n for n, _ in groups]) if groups else None
        held = self.lengths + (self.prefixes or [])
        need = [-(-n // page) for n in held]
        P = sum(need) + 2
        order_of = rng.permutation(P)
        M, MP = max(need[:S], default=0) + extra, max(need[S:], default=0) + extra
        tables = rng.integers(-3, P + 3, (len(held), max(M, MP)))  # (behind a sequence's pages: anything)
        at = 0
        for i, n in enumerate(need):
            tables[i, :n] = order_of[at : at + n]
            at += n
        i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=device)  # noqa: E731
        self.tables, self.prefix_tables = i32(tables)[:S, :M], i32(tables)[S:, :MP]
        shape = (P, kv_heads, page, D) if order == "heads" else (P, page, kv_heads, D)
        self.cache = [torch.tensor(rng.standard_normal(shape) * spread, dtype=torch.float32).to(dtype).to(device) for _ in range(2)]
        if order == "heads":
            self.cache = [t.transpose(1, 2) for t in self.cache]
        self.q = torch.tensor(rng.standard_normal((S, T, heads, D)) * spread, dtype=torch.float32).to(dtype).to(device)
        self.lengths_t = i32(self.lengths)
        self.groups = {}
        if groups:
            self.groups = dict(prefix_lengths=i32(self.prefixes), max_prefix_pages=MP, group_starts=i32(self.starts))

    def plan(self, b):
        return b.plan(self.lengths_t, queries=self.T, heads=self.heads, kv_heads=self.kv_heads, head_dim=self.D,
                      page_size=self.page, max_pages=self.tables.shape[1], **self.groups)

    def attend(self, b, plan=None, scale=None):
        return b.attend(self.q, *self.cache, self.tables, plan or self.plan(b), scale=scale,
                        prefix_tables=self.prefix_tables if self.groups else None)

    def want(self, scale=None):
        S = len(self.lengths)
        k, v = (t.double().cpu().numpy().reshape(-1, self.kv_heads, self.D) for t in self.cache)
        tables, prefix_tables = self.tables.cpu().numpy(), self.prefix_tables.cpu().numpy()
        pre, keys, values = [0] * S, [], []

        def slots(row, n):
            p = np.arange(n)
            return row[p // self.page].astype(np.int64) * self.page + p % self.page

        for s, n in enumerate(self.lengths):
            at = slots(tables[s], n)
            if self.groups:
                g = int(np.searchsorted(self.starts, s, side="right")) - 1
                pre[s] = self.prefixes[g]
                at = np.concatenate([slots(prefix_tables[g], pre[s]), at])
            keys.append(k[at])
            values.append(v[at])
        return paged_oracle.attend(self.q.double().cpu().numpy(), keys, values, self.lengths, pre, scale)

    def check(self, scale=None, b=None):
        got = self.attend(b or backend(self.device, self.dtype), scale=scale).double().cpu().numpy()
        out, mass, size = self.want(scale)
        n = max(self.lengths + [0]) + max(self.prefixes or [0])
        step = torch.finfo(self.dtype).eps / 2
        # The output's rounding; each weight's (fp16: half of 2^-24 at least, beside a sum of at least 2^-1, so that n of
        # them add n 2^-25 times the largest value at most); scores' products summed in fp32, twice (weights and their
        # sum); n weights and products summed in fp32, twice.
        weight = step + 4 * (self.D + 16) * 2.0**-24 * size[..., None] + 2 * (n + 64) * 2.0**-24
        tiny = n * 2.0**-24 * 8 * 2.0**-10 if self.dtype == F16 else 0.0
        off = np.abs(got - out)
        bound = step * np.abs(out) + weight * mass * 1.01 + tiny + 2.0**-25
        assert np.isfinite(got).all()
        assert np.all(off <= bound), (np.max(off - bound), np.argwhere(off > bound)[:5])
        return got


@pytest.mark.parametrize("D", [8, 64, 72, 80, 96, 128, 160, 192, 256])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_heads(device, dtype, D):
    Case(device, dtype, [(2, 70), (1, 33)], [5, 130, 64], D=D, heads=6, kv_heads=2, seed=D).check()


@pytest.mark.parametrize("heads", [(1, 1), (8, 1), (5, 5), (9, 3), (40, 2), (33, 1)], ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_shared_key_heads(device, heads):
    Case(device, BF16, [(3, 100), (2, 40)], [1, 17, 65, 129, 3], heads=heads[0], kv_heads=heads[1], T=2, seed=heads[0]).check()


@pytest.mark.parametrize("page", [1, 2, 16, 64, 256, 4096])
@pytest.mark.parametrize("order", ["places", "heads"])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_pages(device, order, page):
    Case(device, BF16, [(2, 200), (1, 63), (1, 65)], [1, 64, 66, 150], page=page, order=order, seed=page).check()


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_lengths_of_zero_and_one(device):
    # groups without sequences, without a prefix, sequences without keys of their own: these give 0
    c = Case(device, BF16, [(0, 50), (2, 0), (3, 1), (0, 0), (1, 64)], [0, 1, 0, 1, 2, 0], seed=1)
    got = c.check()
    assert (got[[0, 2, 5]] == 0).all()
    c = Case(device, BF16, None, [0, 0], seed=2)
    assert (c.check() == 0).all()
    assert Case(device, BF16, None, [], seed=2).check().shape == (0, 1, 4, 64)


@pytest.mark.parametrize("T", [2, 5, 33, 70])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_new_tokens(device, T):
    # causal among the new tokens; sequences shorter than them (padded on the left) have none before their first
    lengths = [T, T + 1, 3, 0, T - 1, 64, 200]
    got = Case(device, BF16, [(3, 31), (4, 0)], lengths, T=T, seed=T).check()
    for s, n in enumerate(lengths):
        assert (got[s, : max(0, T - n)] == 0).all()
    Case(device, F16, None, lengths, T=T, heads=3, kv_heads=1, D=128, seed=T).check()


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_many_rows_of_a_group(device):
    # rows past a workgroup's, in groups of unlike sizes
    rng = np.random.default_rng(5)
    Case(device, BF16, [(45, 130), (1, 500), (20, 64)], rng.integers(0, 40, 66).tolist(), heads=8, kv_heads=2, seed=6).check()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_long_keys_in_several_workgroups(D):
    # one sequence's keys over the whole chip; a prefix and long own keys
    Case(GPU, BF16, None, [20011], T=3, heads=8, kv_heads=4, D=D, seed=D).check()
    Case(GPU, F16, [(3, 9001), (2, 777)], [1200, 0, 3001, 64, 1], heads=4, kv_heads=4, D=D, page=32, seed=D).check()


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_sharp_scores_and_a_scale(device):
    # weights that differ by e^100 and more: maxima that move from tile to tile
    Case(device, BF16, [(2, 300)], [100, 259], spread=4.0, D=128, seed=3).check()
    Case(device, F16, [(2, 300)], [100, 259], D=32, seed=4).check(scale=2.5)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_what_lies_behind_the_lengths_is_not_seen(device):
    c = Case(device, BF16, [(2, 37)], [9, 30], seed=8)
    want = c.check()
    held = set()
    for tables, lengths in ((c.tables, c.lengths), (c.prefix_tables, c.prefixes)):
        for row, n in zip(tables.tolist(), lengths):
            held |= {row[p // c.page] * c.page + p % c.page for p in range(n)}
    other = torch.tensor([i for i in range(c.cache[0].shape[0] * c.page) if i not in held], device=device)
    for bad in (math.nan, math.inf, -math.inf):
        for t in c.cache:
            t.view(-1, *t.shape[2:])[other] = bad
        got = c.attend(backend(device, BF16)).double().cpu().numpy()
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_keys_of_minus_infinity_and_rows_without_weight(device):
    c = Case(device, BF16, None, [70, 3], heads=1, kv_heads=1, seed=9)
    k = c.cache[0]
    q0 = c.q.clone().abs_()
    c.q.copy_(q0)
    row = c.tables.tolist()
    for p in (0, 5, 69):
        k[row[0][p // 16], p % 16] = -math.inf  # (weights of 0)
    for p in range(3):
        k[row[1][0], p] = -math.inf  # (no weight at all: 0)
    got = c.attend(backend(device, BF16)).double().cpu().numpy()
    keep = [p for p in range(70) if p not in (0, 5, 69)]
    at = np.array([row[0][p // 16] * 16 + p % 16 for p in keep])
    kk, vv = (t.double().cpu().numpy().reshape(-1, 1, 64)[at] for t in c.cache)
    out, mass, _ = paged_oracle.attend(c.q[:1].double().cpu().numpy(), [kk], [vv], [67])
    assert np.all(np.abs(got[0] - out[0]) <= 2.0**-8 * (np.abs(out[0]) + 1.02 * mass[0]) + 2.0**-16)
    assert (got[1] == 0).all()


@pytest.mark.gpu
def test_the_same_bits_every_time_in_graphs_and_on_other_streams():
    rng = np.random.default_rng(11)
    c = Case(GPU, BF16, [(30, 700), (3, 4000)], rng.integers(0, 300, 33).tolist(), heads=8, kv_heads=2, D=128, seed=11)
    b = backend(GPU, BF16)
    plan = c.plan(b)
    want = c.attend(b, plan)
    for _ in range(3):
        assert torch.equal(c.attend(b), want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:  # two calls at once, of one plan
        with torch.cuda.stream(s):
            outs += [c.attend(b, plan) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for s in streams:
        with torch.cuda.stream(s):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                graphs.append((g, c.attend(b)))
    c2 = Case(GPU, BF16, [(30, 650), (3, 3000)], rng.integers(0, 300, 33).tolist(), heads=8, kv_heads=2, D=128, seed=11)
    for lengths, prefixes in ((c.lengths_t.clone(), c.groups["prefix_lengths"].clone()),
                              (c.lengths_t // 2, c.groups["prefix_lengths"] - 50), (c2.lengths_t * 0 + 1, c2.groups["prefix_lengths"])):
        c.lengths_t.copy_(lengths)  # (a plan that is captured is made anew from what the lengths have become)
        c.groups["prefix_lengths"].copy_(prefixes)
        now = c.attend(b)
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, now) for _, o in graphs)


@pytest.mark.gpu
def test_queries_of_other_layouts():
    c = Case(GPU, BF16, [(3, 50)], [9, 20, 70], T=2, heads=4, kv_heads=2, seed=12)
    b = backend(GPU, BF16)
    want = c.attend(b)
    S, T, H, D = c.q.shape
    wide = torch.zeros(S, T, H + 4, D + 8, dtype=BF16, device=GPU)
    wide[:, :, :H, 8:].copy_(c.q)
    odd = torch.zeros(S, T, H, D + 3, dtype=BF16, device=GPU)
    odd[..., 1 : D + 1].copy_(c.q)
    turned = c.q.transpose(1, 2).contiguous().transpose(1, 2)
    for q in (wide[:, :, :H, 8:], odd[..., 1 : D + 1], turned):
        c.q = q
        assert torch.equal(c.attend(b), want)


def test_refusals():
    b = backend(torch.device("cpu"), BF16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    good = dict(lengths=i32(2), queries=1, heads=4, kv_heads=2, head_dim=64, page_size=16, max_pages=3)
    for bad, match in (({"queries": 0}, "queries"), ({"heads": 3}, "multiple"), ({"head_dim": 60}, "head_dim"),
                       ({"head_dim": 264}, "head_dim"), ({"page_size": 24}, "power of two"), ({"max_pages": 0}, "max_pages"),
                       ({"lengths": torch.zeros(2)}, "lengths"), ({"lengths": i32(2, 1)}, "lengths"), ({"kv_heads": 0}, "kv_heads"),
                       ({"prefix_lengths": i32(1)}, "together"), ({"group_starts": i32(1)}, "together"),
                       ({"prefix_lengths": i32(1), "group_starts": i32(1), "max_prefix_pages": 2}, "group_starts"),
                       ({"prefix_lengths": i32(1), "group_starts": i32(2)}, "max_prefix_pages")):
        with pytest.raises(ValueError, match=match):
            b.plan(**{**good, **bad})
    plan = b.plan(**good, prefix_lengths=i32(1), group_starts=i32(2), max_prefix_pages=2)
    mk = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt)  # noqa: E731
    call = dict(q=mk(2, 1, 4, 64), k_pages=mk(5, 16, 2, 64), v_pages=mk(5, 16, 2, 64), tables=i32(2, 3), plan=plan,
                prefix_tables=i32(1, 2))
    b.attend(**call)
    for bad, match in (({"q": mk(2, 4, 64)}, "q must be"), ({"q": mk(2, 1, 64, 4).transpose(2, 3)}, "unit stride"),
                       ({"q": mk(2, 1, 4, 64).requires_grad_()}, "gradient"), ({"k_pages": mk(5, 16, 2, 64, dt=F16)}, "k_pages"),
                       ({"k_pages": mk(5, 8, 2, 64), "v_pages": mk(5, 8, 2, 64)}, "positions"),
                       ({"k_pages": mk(0, 16, 2, 64), "v_pages": mk(0, 16, 2, 64)}, "pages"),
                       ({"tables": i32(2, 4)}, "tables"), ({"tables": i32(3, 2).T}, "tables"), ({"prefix_tables": None}, "prefix_tables"),
                       ({"prefix_tables": i32(1, 3)}, "prefix_tables"), ({"scale": 0.0}, "scale"), ({"scale": math.nan}, "scale")):
        with pytest.raises(ValueError, match=match):
            b.attend(**{**call, **bad})


@pytest.mark.gpu
def test_a_plan_of_another_backend_is_refused():
    c = Case(torch.device("cpu"), BF16, None, [9], seed=13)
    plan = c.plan(backend(c.device, BF16))
    with pytest.raises(ValueError, match="another backend"):
        c.attend(backend(GPU, BF16), plan)


@pytest.mark.gpu
def test_a_cache_past_32_bits():
    # pages whose bytes lie past 2^32 from the first one's, as keys and as a place to store them
    P, page, D = 300000, 16, 256
    cache = [torch.empty(P, page, 2, D, dtype=BF16, device=GPU) for _ in range(2)]  # 4.9 GB each
    tables = torch.tensor([[P - 1, 5, P - 7, 262144]], dtype=torch.int32, device=GPU)
    g = torch.Generator().manual_seed(1)
    small = [torch.randn(4, page, 2, D, generator=g).to(BF16) for _ in range(2)]
    for t, x in zip(cache, small):
        t[tables[0].long()] = x.to(GPU)
    q = torch.randn(1, 1, 4, D, generator=g).to(BF16)
    b = backend(GPU, BF16)
    plan = b.plan(torch.tensor([61], dtype=torch.int32, device=GPU), queries=1, heads=4, kv_heads=2, head_dim=D, page_size=page, max_pages=4)
    got = b.attend(q.to(GPU), *cache, tables, plan)
    near = [torch.zeros(4, page, 2, D, dtype=BF16, device=GPU) for _ in range(2)]
    for t, x in zip(near, small):
        t.copy_(x)
    want = b.attend(q.to(GPU), *near, torch.arange(4, dtype=torch.int32, device=GPU)[None], plan)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_more_rows_than_a_grid_s_dimension_has_threads():
    # 2^26 rows of outputs, all but the last two tokens' of each sequence without a token
    S, T, H, D, lengths = 16, 65536, 64, 8, [2, 1] * 8
    g = torch.Generator().manual_seed(21)
    one, k, v = (torch.randn(*s, generator=g).to(BF16).to(GPU) for s in ((S, 1, H, D), (S, 16, H, D), (S, 16, H, D)))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=GPU)  # noqa: E731
    b = backend(GPU, BF16)
    plan = b.plan(i32(lengths), queries=T, heads=H, kv_heads=H, head_dim=D, page_size=16, max_pages=1)
    torch.full((S, T, H, D), math.nan, dtype=BF16, device=GPU)  # (what the outputs' memory held)
    got = b.attend(one.expand(S, T, H, D), k, v, i32(range(S))[:, None], plan)
    x, kk, vv = one[:, 0].double(), k[:, :2].double(), v[:, :2].double()
    z = (x[:, None] * kk).sum(3) * D**-0.5  # [S, keys, H]
    first, both = vv[:, 0], (torch.softmax(z, 1)[..., None] * vv).sum(1)
    n = torch.tensor(lengths, device=GPU)[:, None, None]
    # one or two weights and the output rounded, each by half a step
    near = lambda a, want: bool(((a.double() - want).abs() <= 2.0**-8 * (want.abs() + 1.02 * vv.abs().amax(1)) + 2.0**-20).all())  # noqa: E731
    assert near(got[:, T - 1], torch.where(n == 2, both, first))
    assert near(got[:, T - 2], torch.where(n == 2, first, 0.0))
    for s in range(S):
        assert int(torch.count_nonzero(got[s, : T - 2])) == 0


@pytest.mark.gpu
def test_queries_and_caches_whose_layout_torch_calls_contiguous():
    # rows at odd addresses, and odd strides of dimensions of one element
    b = backend(GPU, BF16)
    for lengths, T, D, page, kv_heads, extra in (([9, 20, 70], 2, 64, 16, 2, 1), ([33], 3, 72, 64, 1, 0)):
        c = Case(GPU, BF16, None, lengths, T=T, heads=4, kv_heads=kv_heads, D=D, page=page, extra=extra, seed=14)
        want = c.attend(b)
        n, shape, q = c.q.numel(), c.q.shape, c.q
        for skip in (1, 4):
            c.q = torch.zeros(n + skip, dtype=BF16, device=GPU)[skip:].view(shape).copy_(q)
            assert c.q.is_contiguous() and c.q.data_ptr() % 16
            assert torch.equal(c.attend(b), want)
        if len(lengths) > 1:
            continue
        for odd in (n + 1, 3):
            c.q = torch.zeros(n, dtype=BF16, device=GPU).as_strided(shape, (odd, *q.stride()[1:])).copy_(q)
            assert c.q.is_contiguous()
            assert torch.equal(c.attend(b), want)
        # one page, one key head
        table = c.tables[:, :1].clone()
        held = [t[int(table[0, 0])] for t in c.cache]
        c.tables = torch.zeros_like(table)
        for odd in (1, 5):
            c.cache = [torch.zeros(page * D, dtype=BF16, device=GPU).as_strided((1, page, 1, D), (odd, D, odd, 1)).copy_(t[None]) for t in held]
            assert torch.equal(c.attend(b), want)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_derivatives_are_refused(device):
    c = Case(device, BF16, None, [9, 20], seed=15)
    b = backend(device, BF16)
    plan = c.plan(b)
    want = c.attend(b, plan)  # (what was checked once is checked again where a tensor asks for more)
    tensors = {"q": c.q, "k_pages": c.cache[0], "v_pages": c.cache[1]}
    call = lambda t: b.attend(t["q"], t["k_pages"], t["v_pages"], c.tables, plan)  # noqa: E731
    for name, t in tensors.items():
        asking = {**tensors, name: t.clone().requires_grad_()}
        with pytest.raises(ValueError, match=f"{name} requires a gradient"):
            call(asking)
        with torch.no_grad():
            assert torch.equal(call(asking), want)
        with torch.autograd.forward_ad.dual_level():
            assert torch.equal(call(tensors), want)
            with pytest.raises(ValueError, match=f"{name} has a tangent"):
                call({**tensors, name: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))})


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_scores_far_from_zero(device, dtype):
    # scores n 2^b, n whole numbers of 8 bits: where one is the largest its value comes out, where two are their mean. (All
    # other weights are e^(-2^b) at most; a score times log2 e is off by up to 2^(b - 18) where it is rounded.)
    for b, sign, groups, lengths, T, page in ((25, 1, None, [1, 200, 77], 1, 16), (30, -1, None, [130, 5], 2, 16), (30, 1, [(3, 300), (1, 0)], [1, 70, 3, 9], 1, 16),
                                             (34, -1, [(45, 90)], [3] * 45, 1, 8), (28, -1, None, [9000], 1, 64)):
        half = min(b // 2, 14) if dtype == F16 else b // 2
        if dtype == F16 and b - half > 7:  # (255 2^7 is what fp16 holds of a key; the rest is the scale's)
            up = 7
        else:
            up = b - half
        c = Case(device, dtype, groups, lengths, T=T, heads=2, kv_heads=1, D=64, page=page, seed=b)
        k, v = c.cache
        rng = np.random.default_rng(b)
        n = torch.tensor(rng.integers(128, 255, k.shape[:2]), dtype=torch.float64)
        for s in range(len(lengths)):  # one or two own keys of each sequence are the largest
            row = c.tables[s].tolist()
            at = list(range(lengths[s]))[: 2 - s % 2]
            for p in at:
                n[row[p // page], p % page] = 255 if sign > 0 else 127
        k.zero_()
        k[..., 0, 0] = (sign * n * 2.0**up).to(dtype).to(device)
        c.q.zero_()
        c.q[..., 0] = 2.0**half
        got = c.attend(backend(device, dtype), scale=2.0 ** (b - half - up)).double().cpu()
        for s in range(len(lengths)):
            row = c.tables[s].tolist()
            for t in range(T):
                last = lengths[s] - T + t + 1
                at = list(range(min(last, 2 - s % 2)))
                want = torch.stack([v[row[p // page], p % page, 0] for p in at]).double().cpu().mean(0)
                off = (got[s, t] - want).abs()
                assert bool((off <= torch.finfo(dtype).eps / 2 * want.abs() * 1.01 + 2.0**-24).all()), (b, s, t, off.max())


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_scales_that_fp32_does_not_hold_are_refused(device):
    c = Case(device, BF16, None, [1, 3], seed=16)
    b = backend(device, BF16)
    for scale in (1e300, 2.0**127, 2.0**64 * 1.01, 2.0**-127, 1e-300):
        with pytest.raises(ValueError, match="scale"):
            c.attend(b, scale=scale)
    one = torch.stack([c.cache[1][int(t[0]), 0] for t in c.tables.cpu()]).repeat_interleave(2, 1)  # (a single key's value)
    assert torch.equal(c.attend(b, scale=2.0**64)[0, 0], one[0])
    got = c.attend(b, scale=2.0**-126)[1, 0].double().cpu()  # (equal weights)
    v = torch.stack([c.cache[1][int(c.tables[1, 0]), p] for p in range(3)]).repeat_interleave(2, 1).double().cpu()
    assert bool(((got - v.mean(0)).abs() <= 2.0**-8 * (v.mean(0).abs() + 1.02 * v.abs().mean(0)) + 2.0**-20).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["alone", "many groups", "wide", "prompts"])
def test_more_sequences_than_a_plan_s_threads(kind):
    # past 1024 sequences and groups a plan goes round, past 2048 segments and 2047 groups it searches in memory
    rng = np.random.default_rng(22)
    if kind == "alone":
        S, groups, shape = 2500, None, {}
    elif kind == "many groups":  # of no, one and several sequences
        sizes = [(0, 1, 1, 3, 1)[i % 5] for i in range(2200)]
        groups, S, shape = [(n, int(rng.integers(0, 60))) for n in sizes], sum(sizes), {}
    elif kind == "wide":  # more than 32 rows a group and a sequence
        groups, S, shape = [(1 + i % 2, int(rng.integers(0, 90))) for i in range(900)], 1350, dict(heads=33, kv_heads=1)
    else:  # several segments a sequence
        S, groups, shape = 300, [(300, 70)], dict(T=40, heads=8, kv_heads=1, page=64)
    assert groups is None or sum(n for n, _ in groups) == S
    Case(GPU, BF16, groups, rng.integers(0, 80, S).tolist(), **{**dict(heads=2, kv_heads=2, D=8), **shape}, seed=22).check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
def test_many_weights_far_below_the_largest(dtype):
    # one key of weight 1, the others' 2^-17, 2^-20 and 2^-25: numbers that fp16 holds below its smallest normal one, 2^-14
    # (2^-25 rounds to 0)
    n, D = 30000, 64
    c = Case(GPU, dtype, None, [n], heads=2, kv_heads=1, D=D, seed=23)
    k, v = c.cache
    page_of = c.tables[0].long()
    v.abs_()
    c.q.fill_(1.0)
    for low, mass in ((17, n * 2.0**-17), (20, n * 2.0**-20), (25, n * 2.0**-25)):
        k.zero_()
        k[page_of[0], 0, 0, 0] = low  # (scale ln 2: powers of 2)
        got = c.attend(backend(GPU, dtype), scale=math.log(2.0)).double()[0, 0]
        flat = v[page_of].flatten(0, 1)[:n, 0].double()
        first, rest = flat[0], flat[1:].sum(0) * 2.0**-low
        want = (first + rest) / (1.0 + (n - 1) * 2.0**-low)
        # a score of `low` and its product with log2 e in fp32, each a few steps; the first weight 1 to 2^-20, the others one
        # rounding (fp16: up to 2^-25 each); sums of n in fp32
        step = torch.finfo(dtype).eps / 2
        lost = (n - 1) * 2.0**-25 if dtype == F16 and low > 20 else 0.0
        off = (got - want).abs()
        bound = step * want + (step + 2.0**-18 + n * 2.0**-24) * mass * 8 + lost * (want + flat.max(0).values) + 2.0**-18 * want
        assert bool((off <= bound).all()), (low, float((off - bound).max()))

"""Page tables of the paged cache (``extend``, ``shrink``): the reference backend and the hip kernels against a plain
loop over the sequences, entry by entry. Whole numbers have no tolerance."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_oracle
from vinfer_amd.paged import PAGED, PageTables
from vinfer_amd.registry import BackendContext

GPU = torch.device("cuda", 0)
DEVICES = [torch.device("cpu"), pytest.param(GPU, marks=pytest.mark.gpu)]


def backend(device):
    return PAGED.resolve("hip" if device.type == "cuda" else "reference", BackendContext(device, torch.bfloat16))


def words(x, device):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)


def state(pages: PageTables):
    return tuple(t.cpu().numpy().astype(np.int64) for t in (pages.tables, pages.lengths, pages.free, pages.free_count))


def make(device, lengths, M, pages, page, seed=0):
    """Tables of sequences of these lengths whose pages lie anywhere."""
    rng = np.random.default_rng(seed)
    order = rng.permutation(pages)
    tables = rng.integers(0, pages, (len(lengths), M))  # (what lies behind a sequence's pages is anything)
    at = 0
    for s, n in enumerate(lengths):
        need = -(-n // page)
        tables[s, :need] = order[at : at + need]
        at += need
    free = np.concatenate([order[at:], np.full(at, -7)])
    return PageTables(words(tables, device).reshape(len(lengths), M), words(lengths, device), words(free, device),
                      words([pages - at], device), page)


def check_extend(device, pages, counts, tokens):
    tables, lengths, free, count = state(pages)
    want = paged_oracle.extend(tables, lengths, free, int(count[0]), pages.page_size, np.asarray(counts, np.int64), tokens)
    e = backend(device).extend(pages, words(counts, device), tokens)
    got = *(t.cpu().numpy() for t in (e.slots, e.positions, e.sequences, e.served)), *state(pages)
    for name, g, w in zip(("slots", "positions", "sequences", "served", "tables", "lengths"), got, want):
        np.testing.assert_array_equal(g, w, err_msg=name)
    assert int(got[7][0]) == want[6]
    np.testing.assert_array_equal(got[6], free)  # (the stack itself stays)
    return e


def check_shrink(device, pages, to):
    tables, lengths, free, count = state(pages)
    want = paged_oracle.shrink(tables, lengths, free, int(count[0]), pages.page_size, np.asarray(to, np.int64))
    backend(device).shrink(pages, words(to, device))
    got = state(pages)
    np.testing.assert_array_equal(got[0], tables)
    np.testing.assert_array_equal(got[1], want[0])
    np.testing.assert_array_equal(got[2][: want[2]], want[1][: want[2]])
    assert int(got[3][0]) == want[2]


@pytest.mark.parametrize("S", [1, 3, 64, 1024, 1025, 2500])
@pytest.mark.parametrize("page", [1, 8, 64])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_steps(device, page, S):
    rng = np.random.default_rng(S + page)
    M = 12
    lengths = rng.integers(0, M * page // 2 + 1, S)
    pages = make(device, lengths, M, S * M + 5, page, S)
    for counts in (np.ones(S, int), rng.integers(-2, 4 * page, S), np.zeros(S, int)):
        before = state(pages)
        tokens = int(np.maximum(counts, 0).sum())
        check_extend(device, pages, counts, tokens + 3)
        check_shrink(device, pages, before[1])
        for a, b in zip(state(pages)[1:], before[1:]):
            np.testing.assert_array_equal(a, b)  # (laid back as it was)
        check_extend(device, pages, counts, tokens)
        check_shrink(device, pages, rng.integers(-3, M * page, S))


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_what_does_not_fit_is_not_served(device):
    # tables too short, tokens past the call's, pages run out: whole sequences, the others as if those were not there
    pages = make(device, [5, 30, 0, 32, 1, 9], 4, 14, 8)
    e = check_extend(device, pages, [3, 3, 0, 1, 60, 4], 11)
    assert e.served.tolist() == [True, False, True, False, False, False]
    pages = make(device, [8, 8, 8, 8, 7], 4, 8, 8)
    e = check_extend(device, pages, [9, 1, 2, 0, 1], 13)  # three pages are free, the second takes the last
    assert e.served.tolist() == [True, True, False, True, True]
    assert int(pages.free_count) == 0
    e = check_extend(device, pages, [0, 0, 1, 0, 0], 4)
    assert e.served.tolist() == [True, True, False, True, True] and e.slots.tolist() == [-1] * 4


@pytest.mark.parametrize("tokens", [8192, 8193, 40000])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_prompts(device, tokens):
    # both routes: one workgroup for all tokens, and tokens over the chip
    counts = np.array([0, 7000, 1, 0, 31000, 0, 5])
    if tokens < 40000:
        counts[4] = tokens - 7000 - 1 - 5 - 100
    pages = make(device, [3, 17, 0, 0, 900, 5, 64], 2100, 2500, 16)
    check_extend(device, pages, counts, tokens)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_nothing(device):
    pages = PageTables.empty(0, 3, 4, 16, device)
    e = backend(device).extend(pages, words([], device), 0)
    backend(device).shrink(pages, words([], device))
    assert e.slots.shape == (0,) and e.served.shape == (0,)
    pages = PageTables.empty(2, 1, 1, 4096, device)
    check_extend(device, pages, [0, 4096], 4096)
    check_shrink(device, pages, [5, 0])


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_states_from_outside_are_taken_as_the_nearest(device):
    pages = PageTables.empty(2, 2, 6, 4, device)
    pages.lengths.copy_(words([-5, 100], device))
    pages.free_count.fill_(99)
    e = backend(device).extend(pages, words([1, 1], device), 2)
    assert e.served.tolist() == [True, False] and e.positions.tolist() == [0, -1] and int(pages.free_count) == 5
    pages.lengths.copy_(words([1, 100], device))
    pages.free_count.fill_(-3)
    backend(device).shrink(pages, words([0, 0], device))
    assert pages.lengths.tolist() == [0, 0] and int(pages.free_count) == 3


def test_refusals():
    mk = lambda *s, dt=torch.int32: torch.zeros(*s, dtype=dt)  # noqa: E731
    good = dict(tables=mk(2, 3), lengths=mk(2), free=mk(4), free_count=mk(1), page_size=16)
    b = backend(torch.device("cpu"))
    p = PageTables(**good)
    for bad, match in (({"tables": mk(2, 3, dt=torch.int64)}, "tables"), ({"tables": mk(3, 2).T}, "tables"),
                       ({"lengths": mk(3)}, "lengths"), ({"free": mk(0)}, "pages"), ({"free_count": mk(2)}, "free_count"),
                       ({"tables": mk(2, 0)}, "page"), ({"page_size": 12}, "power of two"), ({"page_size": 8192}, "power of two"),
                       ({"page_size": 0}, "power of two")):
        with pytest.raises(ValueError, match=match):
            PageTables(**{**good, **bad})
    with pytest.raises(ValueError, match="counts"):
        b.extend(p, mk(3), 4)
    with pytest.raises(ValueError, match="counts"):
        b.extend(p, mk(2, dt=torch.int64), 4)
    with pytest.raises(ValueError, match="tokens"):
        b.extend(p, mk(2), -1)
    with pytest.raises(ValueError, match="tokens"):
        b.extend(PageTables.empty(0, 1, 1, 16, "cpu"), mk(0), 1)
    with pytest.raises(ValueError, match="lengths"):
        b.shrink(p, mk(1))


@pytest.mark.gpu
def test_a_captured_step_on_another_stream():
    S, page = 300, 16
    rng = np.random.default_rng(1)
    lengths = rng.integers(0, 100, S)
    pages, plain = (make(GPU, lengths, 40, S * 12, page) for _ in range(2))
    counts = words(rng.integers(0, 5, S), GPU)
    n = int(counts.sum())
    b = backend(GPU)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.extend(pages, counts, n)
        b.shrink(pages, words(lengths, GPU))
        back = words(lengths, GPU) + 1
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            e = b.extend(pages, counts, n)
            b.shrink(pages, back)
    for _ in range(3):
        want = b.extend(plain, counts, n)
        b.shrink(plain, back)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in ((e.slots, want.slots), (e.positions, want.positions), (e.served, want.served),
                     (pages.lengths, plain.lengths), (pages.free_count, plain.free_count)):
            assert torch.equal(x, y)

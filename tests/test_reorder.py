"""The reordering of a beam search's states (``prepare_reorder``): the reference backend and the hip kernel
against a copy of the old states, element by element. Copies have no tolerance."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import ops_oracle
from vinfer_amd import _vops
from vinfer_amd.registry import BackendContext
from vinfer_amd.sampler import SAMPLER, BeamState
from vinfer_amd.sampler.beams import describe

DEVICES = [torch.device("cpu"), pytest.param(torch.device("cuda", 0), marks=pytest.mark.gpu)]
GPU = torch.device("cuda", 0)


def backend(device):
    return SAMPLER.resolve("hip" if device.type == "cuda" else "reference", BackendContext(device, torch.bfloat16))


def fill(t, seed):
    g = torch.Generator().manual_seed(seed)
    t.copy_(torch.randint(0, 120, t.shape, generator=g).to(t.dtype))
    return t


def host(t):
    t = t.cpu()
    return t.float() if t.dtype == torch.bfloat16 else t  # (fill's values are exact in either)


def make_states(B, W, L, heads, dim, dtype, device):
    """Tensors of every layout that a model keeps: (state, slot dimension, length dimension)."""
    n, mk = B * W, lambda *s, dt=dtype: torch.empty(*s, dtype=dt, device=device)
    wide = mk(n, L, heads, 2 * dim)
    pool = mk(n, 2, L, heads, dim)
    return [
        (mk(n, heads, dim, dim, dt=torch.float32), 0, None),  # a recurrent state
        (mk(2, n, heads, L, dim), 1, 3),  # layers stacked, positions inside the heads
        (mk(n, L, heads, dim), 0, 1),
        (mk(n, heads, dim, L), 0, 3),  # keys transposed
        (mk(L, n, heads * dim), 1, 0),  # positions outermost
        (wide[..., :dim], 0, 1),  # a slice: heads apart
        (pool[:, 0], 0, 1),  # keys and values of one buffer
        (pool[:, 1], 0, 1),
        (mk(n, L, dt=torch.int32), 0, 1),  # token histories
        (mk(n, 3, dt=torch.uint8), 0, None),
        (mk(n, dt=torch.int64), 0, None),
        (mk(2, n, 3, L, 5, dt=torch.uint8), 1, 3),
        (torch.empty(n, L + 1, 7, dtype=torch.uint8, device=device)[:, 1:], 0, 1),  # an odd first byte
    ]


def check(device, states, B, W, parents, lengths, prepared=None):
    for i, (t, _, _) in enumerate(states):
        fill(t, i)
    want = []
    for t, slot, length in states:
        v = host(t).movedim(slot, 0)
        if length is not None:
            v = v.movedim(length + (length < slot), 1)
        else:
            v = v.unsqueeze(1)
        a = v.numpy().reshape(B, W, *v.shape[1:])
        want.append(ops_oracle.reorder(a, parents.numpy(), lengths.numpy() if length is not None else None))
    plan = prepared or backend(device).prepare_reorder([BeamState(*s) for s in states], B, W)
    plan.launch(parents.to(device), lengths.to(device))
    for (t, slot, length), w in zip(states, want):
        v = host(t).movedim(slot, 0)
        v = v.unsqueeze(1) if length is None else v.movedim(length + (length < slot), 1)
        np.testing.assert_array_equal(v.numpy().reshape(w.shape), w)
    return plan


def parents_of(kind, B, W, rng):
    if kind == "same":
        p = np.tile(np.arange(W), (B, 1))
    elif kind == "cycle":  # (each slot's state moves on by one: no order of copies serves)
        p = np.tile((np.arange(W) + 1) % W, (B, 1))
    elif kind == "one":
        p = np.full((B, W), W - 1)
    elif kind == "outside":  # (places that beam_select left empty, and values past the beams)
        p = rng.integers(-2, W + 2, (B, W))
    else:
        p = rng.integers(0, W, (B, W))
    return torch.from_numpy(p.astype(np.int32))


@pytest.mark.parametrize("kind", ["same", "cycle", "one", "outside", "any"])
@pytest.mark.parametrize("size", [(1, 2, 1, 1, 4), (3, 5, 37, 3, 6), (2, 9, 64, 2, 16), (2, 20, 11, 1, 8), (1, 32, 5, 2, 3)],
                         ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_every_layout(device, size, kind):
    B, W, L, heads, dim = size
    rng = np.random.default_rng(W + L)
    lengths = torch.from_numpy(rng.integers(0, L + 1, B).astype(np.int32))
    lengths[0] = L
    check(device, make_states(B, W, L, heads, dim, torch.bfloat16, device), B, W, parents_of(kind, B, W, rng), lengths)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_lengths_are_clamped_and_a_plan_is_reused(device):
    B, W, L = 4, 3, 19
    states = make_states(B, W, L, 2, 8, torch.float32, device)
    rng = np.random.default_rng(3)
    plan = None
    for lengths in ([0, 1, L, L - 1], [L + 5, -3, 1 << 30, -(1 << 31)]):
        plan = check(device, states, B, W, parents_of("any", B, W, rng), torch.tensor(lengths, dtype=torch.int32), plan)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_nothing_to_move(device):
    empty = torch.zeros(0, 7, device=device)
    backend(device).prepare_reorder([BeamState(empty, 0, 1)], 0, 4).launch(
        torch.zeros(0, 4, dtype=torch.int32, device=device), torch.zeros(0, dtype=torch.int32, device=device))
    t = fill(torch.empty(6, 0, 3, device=device), 1)
    u = fill(torch.empty(6, 5, device=device), 2)
    old = u.cpu()
    plan = backend(device).prepare_reorder([BeamState(t, 0, 1), BeamState(u)], 2, 3)
    plan.launch(torch.full((2, 3), -1, dtype=torch.int32, device=device), torch.zeros(2, dtype=torch.int32, device=device))
    assert torch.equal(u.cpu(), old)


@pytest.mark.gpu
def test_many_columns_and_workgroups():
    # several steps a workgroup, a run that ends inside a column, rows of many runs
    B, W, L = 33, 4, 1021
    mk = lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device=GPU)  # noqa: E731
    states = [(mk(2, B * W, 5, L, 24), 1, 3), (mk(B * W, L, 5, 40)[..., :24], 0, 1), (mk(B * W, L, dt=torch.int16), 0, 1),
              (mk(B * W, 5, 64, 64, dt=torch.float32), 0, None)]
    rng = np.random.default_rng(4)
    lengths = torch.from_numpy(rng.integers(0, L + 1, B).astype(np.int32))
    check(GPU, states, B, W, parents_of("any", B, W, rng), lengths)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    # two slots more than 4 GiB apart, one of them written, at both ends of its run
    base = torch.zeros(5 << 30, dtype=torch.uint8, device=GPU)
    t = base.as_strided((2, 4, 1000), ((4 << 30) + 512, 250 << 20, 1))
    fill(t[0], 1)
    fill(t[1], 2)
    old = t.cpu()
    backend(GPU).prepare_reorder([BeamState(t)], 1, 2).launch(torch.tensor([[0, 0]], dtype=torch.int32, device=GPU))
    new = t.cpu()
    assert torch.equal(new[0], old[0]) and torch.equal(new[1], old[0])
    assert int(base.count_nonzero()) == 2 * int(old[0].count_nonzero())


@pytest.mark.gpu
def test_graph_replays_and_other_streams():
    B, W, L = 2, 4, 100
    t = torch.empty(B * W, L, 2, 64, dtype=torch.bfloat16, device=GPU)
    plan = backend(GPU).prepare_reorder([BeamState(t, 0, 1)], B, W)
    p = torch.zeros(B, W, dtype=torch.int32, device=GPU)
    n = torch.zeros(B, dtype=torch.int32, device=GPU)
    plan.launch(p, n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.launch(p, n)
    rng = np.random.default_rng(5)
    side = torch.cuda.Stream()
    for i in range(4):
        fill(t, i)
        hp, hn = parents_of("any", B, W, rng), torch.tensor([L, 3 * i], dtype=torch.int32)
        p.copy_(hp)
        n.copy_(hn)
        want = ops_oracle.reorder(t.cpu().view(torch.int16).numpy().reshape(B, W, L, 2, 64), hp.numpy(), hn.numpy())
        if i == 3:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                plan.launch(p, n)
            side.synchronize()
        else:
            graph.replay()
        np.testing.assert_array_equal(t.cpu().view(torch.int16).numpy().reshape(want.shape), want)


@pytest.mark.gpu
def test_a_plan_may_be_dropped_behind_a_launch_on_another_stream():
    # its descriptions stay allocated until that launch has read them
    B, W, L = 2, 4, 50
    t = fill(torch.empty(B * W, L, 64, dtype=torch.bfloat16, device=GPU), 1)
    p = parents_of("cycle", B, W, np.random.default_rng(6))
    n = torch.tensor([L, 7], dtype=torch.int32)
    want = ops_oracle.reorder(t.cpu().view(torch.int16).numpy().reshape(B, W, L, 64), p.numpy(), n.numpy())
    pd, nd = p.to(GPU), n.to(GPU)
    plan = backend(GPU).prepare_reorder([BeamState(t, 0, 1)], B, W)
    at, size = plan._descs.data_ptr(), plan._descs.numel()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        plan.launch(pd, nd)
    del plan
    others = [torch.empty(size, dtype=torch.uint8, device=GPU) for _ in range(8)]
    assert all(o.data_ptr() != at for o in others)
    side.synchronize()
    np.testing.assert_array_equal(t.cpu().view(torch.int16).numpy().reshape(want.shape), want)


# ---- what the kernel is told, checked on the CPU ----------------------------------------------------------
def addresses(d, W, slot, length):
    """The bytes of one slot that the kernel moves, by its own arithmetic."""
    n, run = [d.size[i] for i in range(3)], d.run
    if d.length_dim == 3:
        run = length * d.unit
    elif d.length_dim >= 0:
        n[d.length_dim] = length
    for i0 in range(n[0]):
        for i1 in range(n[1]):
            for i2 in range(n[2]):
                a = d.data + slot * d.slot_stride + i0 * d.stride[0] + i1 * d.stride[1] + i2 * d.stride[2]
                yield from range(a, a + run)


@pytest.mark.parametrize("L", [1, 4])
def test_descriptions_cover_each_element_once_and_nothing_else(L):
    B, W = 1, 3
    lib = _vops.load()
    for t, slot_dim, length_dim in make_states(B, W, L, 2, 3, torch.bfloat16, torch.device("cpu")):
        d = describe(BeamState(t, slot_dim, length_dim))
        assert lib.vops_state_columns(ctypes.byref(d)) > 0
        size = t.element_size()
        for slot in range(B * W):
            for length in (0, 1, L):
                v = t.select(slot_dim, slot)
                if length_dim is not None:
                    v = v.narrow(length_dim - (length_dim > slot_dim), 0, length)
                idx = [np.arange(s) * st * size for s, st in zip(v.shape, v.stride())]
                at = np.array(0) if v.dim() == 0 else sum(np.ix_(*idx)) if len(idx) > 1 else idx[0]
                want = {v.data_ptr() + int(o) + k for o in np.ravel(at) for k in range(size)} if v.numel() else set()
                got = list(addresses(d, W, slot, length))
                assert len(got) == len(set(got)) and set(got) == want


BAD = [
    ([], 2, 3, "at least one"),
    ([(torch.zeros(6, 2), 0, None)], 2, 33, "beams in"),
    ([(torch.zeros(5, 2), 0, None)], 2, 3, "must hold the 6 slots"),
    ([(torch.zeros(6, 2), 2, None)], 2, 3, "must hold the 6 slots"),
    ([(torch.zeros(6, 2), 0, 0)], 2, 3, "not another dimension"),
    ([(torch.zeros(6, 2), 0, 2)], 2, 3, "not another dimension"),
    ([(torch.zeros(6, 1).expand(6, 4), 0, None)], 2, 3, "may overlap"),
    ([(torch.zeros(16).as_strided((6, 4), (2, 1)), 0, None)], 2, 3, "may overlap"),
    ([(torch.zeros(6, 2, requires_grad=True), 0, None)], 2, 3, "requires a gradient"),
]


@pytest.mark.parametrize("states,B,W,msg", BAD, ids=[str(i) for i in range(len(BAD))])
def test_states_that_cannot_be_reordered_are_refused(states, B, W, msg):
    with pytest.raises(ValueError, match=msg):
        backend(torch.device("cpu")).prepare_reorder([BeamState(*s) for s in states], B, W)


def test_one_memory_twice_is_refused():
    t = torch.zeros(6, 4)
    with pytest.raises(ValueError, match="same memory"):
        backend(torch.device("cpu")).prepare_reorder([BeamState(t), BeamState(t.view(6, 2, 2))], 2, 3)


def test_states_that_share_some_memory_are_refused():
    c = torch.zeros(6, 8, 10)
    pool = torch.zeros(6, 2, 8, 10)
    shared = [
        (c, c[:, 1:]), (c[:, :5], c[:, 4:]), (c[..., :6], c[..., 5:]), (c, c[:, :, 3]), (c[:, ::2], c[:, ::3]),
        (pool, pool[:, 1]), (pool[:, 0, 2:], pool[:, 0, :3]), (c[:, ::2, :4], c[:, 2:, 3:]),
        (c.view(-1)[1:337].view(6, 56), c), (c.view(torch.uint8)[..., 3:], c.view(torch.uint8)[..., :4]),
    ]
    for a, b in shared:
        for s in ((a, b), (b, a), (torch.zeros(6, 3), a, torch.zeros(6, 3), b)):
            with pytest.raises(ValueError, match="same memory"):
                backend(torch.device("cpu")).prepare_reorder([BeamState(t) for t in s], 2, 3)


def test_states_side_by_side_in_one_buffer_are_taken():
    c = torch.zeros(6, 8, 10)
    pool = torch.zeros(4, 6, 2, 8, 5, 12)  # layers, slots, keys and values, positions, heads, numbers
    record = torch.zeros(6, 100)  # of a slot: a matrix, a window, a few numbers; a gap behind them
    wide = torch.zeros(6, 8, 3, 10)[:, :7]
    apart = [
        (c[:, :5], c[:, 5:]), (c[..., :6], c[..., 6:]), (c[..., 0], c[..., 7]), (c[:, ::2], c[:, 1::2]), (c[:3].repeat(2, 1, 1), c),
        tuple(pool[i, :, j] for i in range(4) for j in range(2)),
        tuple(pool.transpose(0, 3)[i, :, j] for i in range(8) for j in range(2)),
        tuple(pool[0, :, :, :, :, 3 * i : 3 * i + 3] for i in range(4)),
        (record[:, :64].view(6, 8, 8), record[:, 64:80].view(6, 4, 4), record[:, 80:83]),
        (wide[:, :, 0], wide[:, :, 2, :4], wide[:, :, 2, 4:], wide[:, :, 1]),
        (c[:, :0], c),
    ]
    for s in apart:
        for t in (s, s[::-1]):
            backend(torch.device("cpu")).prepare_reorder([BeamState(x) for x in t], 2, 3)
    rng = np.random.default_rng(8)
    for _ in range(300):  # what is taken shares nothing, in layouts of any kind
        base = torch.zeros(2000, dtype=torch.uint8)
        s, held = [], []
        for _ in range(2):
            dims = [(1, int(rng.integers(1, 5)))]
            for _ in range(int(rng.integers(1, 4))):
                st, n = dims[-1]
                dims.append((st * n + int(rng.integers(0, 4)) * int(rng.integers(0, 9)), int(rng.integers(1, 4))))
            dims[-1] = (dims[-1][0], 6)
            off = int(rng.integers(0, 40))
            t = base.as_strided([n for _, n in dims[::-1]], [st for st, _ in dims[::-1]], off)
            s.append(t)
            held.append(set(np.ravel(off + sum(np.ix_(*[np.arange(n) * st for st, n in dims]))).tolist()))
        try:
            backend(torch.device("cpu")).prepare_reorder([BeamState(t) for t in s], 2, 3)
        except ValueError:
            continue
        assert not held[0] & held[1]


def test_too_many_strided_dimensions_are_refused():
    t = torch.zeros(4, 4, 4, 4, 4)[:, ::2, ::2, ::2, ::2]
    with pytest.raises(ValueError, match="strided dimensions"):
        describe(BeamState(t))


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_launch_arguments_are_checked(device):
    t = torch.zeros(6, 5, device=device)
    plan = backend(device).prepare_reorder([BeamState(t, 0, 1)], 2, 3)
    ok = torch.zeros(2, 3, dtype=torch.int32, device=device)
    n = torch.zeros(2, dtype=torch.int32, device=device)
    for p, lengths, msg in [(ok.long(), n, "parents must be"), (ok[:1], n, "parents must be"), (ok, None, "lengths must be given"),
                            (ok, n.long(), "lengths must be"), (ok, n[:1], "lengths must be")]:
        with pytest.raises(ValueError, match=msg):
            plan.launch(p, lengths)


@pytest.mark.parametrize("args,msg", [((0x1000, -1, 5, 1, 2), b"n_states"), ((0x1000, 1, 5, 70000, 2), b"requests"),
                                      ((0x1000, 1, 5, 1, 33), b"beams"), ((0x1000, 1, 1 << 31, 1, 2), b"max_columns"),
                                      ((None, 1, 5, 1, 2), b"must be set")])
def test_the_library_refuses_before_it_looks_for_a_device(args, msg):
    lib = _vops.load()
    assert lib.vops_reorder(*args, 0x2000, None, None) == 1
    assert msg in lib.vops_last_error()

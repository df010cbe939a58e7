"""The distillation loss and its gradient: the reference backend, the hip kernels and ``distill_loss`` against
the plain statement in 64 bits (``oracle/ops_oracle.py``), which is checked against differences of itself.

Tolerances. A term's exponent (x - m) c carries four roundings (the difference, 1 / T's product, the product,
the sum's reference) of 2^-24 and v_exp_f32 one ulp; under the softmax the mean distance from the maximum is at
most ln V <= 13.2, and a thread adds at most 64 terms in fp32: a sum S is off by at most
SUM = (4 * 13.2 + 2 + 64) 2^-24 of itself. The loss takes log S twice (lse and the rest), each against a mass of
at most 1, and rounds once. An unlisted gradient is exp((x - m) c) A: the exponent's roundings, A's (through S,
on either of its two terms), three products, and the rounding to the dtype. A listed one is q mass - p, rounded
to fp32, scaled, and rounded to the dtype. exp2's results below 2^-126 may be 0."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import ops_oracle
from vinfer_amd import _vops
from vinfer_amd.distill import DISTILL, distill_loss
from vinfer_amd.registry import BackendContext

SUM = (4 * 13.2 + 2 + 64) * 2.0**-24
DEVICES = [torch.device("cpu"), pytest.param(torch.device("cuda", 0), marks=pytest.mark.gpu)]
GPU = torch.device("cuda", 0)


def backend(device, dtype):
    return DISTILL.resolve("hip" if device.type == "cuda" else "reference", BackendContext(device, dtype))


def make(seed, T, V, K, dtype=torch.float32, tail=False, ragged=False, zeros=False):
    g = torch.Generator().manual_seed(seed)
    x = (2.0 * torch.randn(T, V, generator=g)).to(dtype)
    K = min(K, V)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)]) if T else torch.zeros(0, K)
    teacher = 6.0 + 3.0 * torch.randn(T, K, generator=g)
    if tail:
        teacher = teacher - torch.logsumexp(torch.cat([teacher, torch.full((T, 1), 9.0)], 1), 1, keepdim=True)
    if ragged:
        ids = torch.where(torch.rand(T, K, generator=g) < 0.6, ids, torch.where(torch.rand(T, K, generator=g) < 0.5, -1, V + 3))
    w = torch.rand(T, generator=g) * 2.0 - 0.5
    if zeros:
        w[::3] = 0.0
    return x, ids.to(torch.int32), teacher, w


def tolerance(x, ids, teacher, w, want_loss, want_grad, T, tail, dtype):
    """(loss, gradient) tolerances of each value."""
    n, V = x.shape
    wa = np.ones(n) if w is None else np.abs(w.double().numpy())
    tol_loss = wa * (2 * SUM + 2.0**-40) + 2.0**-23 * np.abs(want_loss)
    z = x.double().numpy() / T
    there = (ids.numpy() >= 0) & (ids.numpy() < V)
    member = np.zeros((n, V), bool)
    for t in range(n):
        member[t, ids.numpy()[t][there[t]]] = True
    others = np.where(member, -np.inf, z)
    with np.errstate(invalid="ignore", divide="ignore"):
        m = np.max(others, 1, keepdims=True)
        m = np.where(np.isfinite(m), m, 0.0)
        zm = np.max(z, 1, keepdims=True)
        q = np.exp(z - zm)
        q = q / q.sum(1, keepdims=True)
        e = np.where(member, 0.0, np.exp(np.minimum(z - m, 0.0)))
        share = np.where(member, 0.0, e / np.maximum(e.sum(1, keepdims=True), 1e-300)) if tail else 0.0
        size = q + share  # (the two terms of an unlisted gradient; a listed one's q mass)
        p = np.zeros((n, V))
        a = np.where(there, teacher.double().numpy() / (1.0 if tail else T), -np.inf)
        if not tail:
            a = a - np.logaddexp.reduce(a, 1, keepdims=True)
        for t in range(n):
            p[t, ids.numpy()[t][there[t]]] = np.exp(a[t][there[t]])
        d = np.where(np.isfinite(z), np.abs(z - m), 0.0)
    step = torch.finfo(dtype).eps / 2
    g = np.nan_to_num(np.abs(want_grad))
    tol = (wa / T)[:, None] * (size * (SUM + (4 * d + 8) * 2.0**-24) + 2.0**-23 * p + 2.0**-120)
    tol = np.where(np.isnan(tol), 0.0, tol)  # (rows of weight 0 that hold NaN)
    return tol_loss, tol + g * step * (1 + 2.0**-7) + 2.0**-23 * g


def compare(device, x, ids, teacher, w, T=1.0, tail=False):
    want_loss, want_grad = ops_oracle.distill(x.float().numpy(), ids.numpy(), teacher.numpy(),
                                              None if w is None else w.numpy(), T, tail)
    tol_loss, tol_grad = tolerance(x, ids, teacher, w, want_loss, want_grad, T, tail, x.dtype)
    s = backend(device, x.dtype)
    if x.stride() != (x.shape[1], 1):  # (its strides too)
        flat = torch.empty(0, dtype=x.dtype).set_(x.untyped_storage())
        xd = flat.to(device).as_strided(x.shape, x.stride(), x.storage_offset())
    else:
        xd = x.to(device)
    rest = (ids.to(device), teacher.to(device), None if w is None else w.to(device))
    loss = s.loss(xd, *rest, temperature=T, tail=tail)
    both, grad = s.loss_and_grad(xd, *rest, temperature=T, tail=tail)
    assert loss.dtype == torch.float32 and grad.dtype == x.dtype and grad.shape == x.shape
    leaf = xd.detach().requires_grad_()
    last = distill_loss(leaf, *rest, temperature=T, tail=tail, backend=s)
    (auto,) = torch.autograd.grad(last.sum(), leaf)
    for got in (loss, both, last.detach()):
        got = got.cpu().double().numpy()
        same = (got == want_loss) | (np.isnan(got) & np.isnan(want_loss))  # (infinities among them)
        with np.errstate(invalid="ignore"):
            assert np.all(same | (np.abs(got - want_loss) <= tol_loss)), (got, want_loss)
    for got in (grad, auto):
        got = got.cpu().double().numpy()
        bad = ~(np.abs(got - want_grad) <= tol_grad)
        assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want_grad[bad][:5], tol_grad[bad][:5])
    return grad


def test_the_statement_agrees_with_differences_of_itself():
    for tail in (False, True):
        for T in (1.0, 2.5):
            x, ids, teacher, w = make(3, 3, 11, 4, tail=tail, ragged=True)
            ids[:, 0] = torch.tensor([1, 2, 3]) if not (ids[:, 1:] == torch.tensor([[1], [2], [3]])).any() else ids[:, 0]
            a = x.double().numpy()
            f = lambda v: ops_oracle.distill(v, ids.numpy(), teacher.numpy(), w.numpy(), T, tail)[0]  # noqa: E731
            grad = ops_oracle.distill(a, ids.numpy(), teacher.numpy(), w.numpy(), T, tail)[1]
            h = 1e-5
            for j in range(11):
                d = np.zeros_like(a)
                d[:, j] = h
                # central differences: off by h^2 / 6 of a third derivative of at most about 1, and by rounding
                np.testing.assert_allclose((f(a + d) - f(a - d)) / (2 * h), grad[:, j], atol=1e-9)


SIZES = [(1, 1, 1), (1, 2, 1), (3, 7, 7), (5, 33, 4), (2, 2047, 20), (9, 2049, 33), (1, 50257, 100), (3, 5000, 1024)]


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T", [1.0, 0.7, 3.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_random_rows(device, size, dtype, T, tail):
    x, ids, teacher, w = make(sum(size), *size, dtype, tail=tail, ragged=size[0] > 1, zeros=size[0] > 2)
    if tail and size[2] >= size[1]:
        teacher = torch.log_softmax(teacher, 1)  # (every id is listed: no rest to hold the student to)
        ids = ids.clamp(max=size[1] - 1) if size[0] == 1 else ids
        if size[0] > 1:
            pytest.skip("a ragged list leaves ids out")
    compare(device, x, ids, teacher, w, T, tail)


@pytest.mark.parametrize("T", [1.0, 0.7, 3.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("size", [(3, 7), (5, 40), (4, 1000)], ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_lists_that_leave_one_or_two_ids_out(device, size, dtype, T):
    n, V = size
    x, ids, teacher, w = make(25, n, V, V, dtype)
    for t in range(n):
        ids[t, t % V] = -1
        ids[t, (3 * t + 1) % V] = V
    compare(device, x, ids, teacher, w, T, False)
    compare(device, x, ids, torch.log_softmax(teacher, 1) - 0.05, w, T, True)


@pytest.mark.gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("size", [(2, 524288, 64, torch.float32), (700, 3001, 16, torch.bfloat16), (300, 9000, 40, torch.float32),
                                  (270, 151936, 64, torch.bfloat16), (260, 40009, 50, torch.float32),
                                  (1600, 4101, 512, torch.bfloat16), (900, 60001, 7, torch.bfloat16), (210, 90001, 600, torch.bfloat16),
                                  (200, 75003, 70, torch.float32)], ids=str)
def test_large_rows_and_batches(size, tail):
    x, ids, teacher, w = make(9, *size[:3], size[3], tail=tail, zeros=True)
    compare(GPU, x, ids, teacher, w, 1.0, tail)


@pytest.mark.gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_large_batches_of_uneven_and_odd_rows(dtype, tail):
    # rows whose beginning says nothing of the rest, and every kind of row that is not read, in turn
    x, ids, teacher, w = make(61, 620, 9003, 20, dtype, tail=tail, ragged=True)
    x[0::7, :8500] = -torch.inf  # nothing but the end is left
    x[1::7, :9000] -= 300.0
    x[2::7, 4000:] += 250.0
    x[3::7, 1::2] = -torch.inf
    x[4::7, :] = torch.finfo(dtype).min
    w[5::7], x[5::7, :] = 0.0, float("nan")
    ids[6::14] = -1
    w[300:420] = 0.0
    w[-1] = w[0] = 0.0
    compare(GPU, x, ids, teacher, w, 1.0, tail)
    x, ids, teacher, w = make(62, 200, 9003, 300, dtype, tail=tail)
    teacher[::2, 60:250] = -torch.inf  # whole waves of entries of probability 0, and of ids that are masked
    for t in range(0, 200, 3):
        x[t, ids[t, 100:260].long()] = -torch.inf
        teacher[t, 100:260] = -torch.inf
    compare(GPU, x, ids, teacher, w, 1.0, tail)
    x, ids, teacher, w = make(63, 620, 9003, 20, dtype, tail=tail, ragged=True)
    compare(GPU, x[:, 1:], torch.where(ids < 9002, ids, -1), teacher, w, 1.7, tail)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_masks_and_empty_rows(device, dtype):
    x, ids, teacher, w = make(21, 8, 4001, 12, dtype)
    x[0, 7::2] = -torch.inf  # a masked vocabulary, the listed ids finite
    x[0, ids[0].long()] = 1.0
    x[1, :] = torch.finfo(dtype).min
    x[1, ids[1].long()] = 2.0
    x[2, 4000] = 30.0  # a certain student
    ids[3, :] = -1  # no entry at all
    ids[4, 1:] = 5000
    teacher[5, 1:] = -torch.inf  # entries of probability 0
    w[6], x[6, :] = 0.0, float("nan")  # padding: not read
    x[7, :] = -torch.inf
    x[7, ids[7].long()] = 0.5  # nothing but the listed ids is left
    grad = compare(device, x, ids, teacher, w)
    assert not grad[6].any() and not grad[3].any()


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_tail_of_rows_with_little_or_nothing_beside_the_list(device):
    x, ids, teacher, w = make(22, 5, 3000, 10, tail=True)
    x[0, ids[0].long()] += 90.0  # the rest of the student's mass is far below 2^-24
    x[1, ids[1].long()] = -torch.inf
    teacher[1] = -torch.inf  # the teacher's whole mass is outside
    teacher[2] = torch.log_softmax(teacher[2], 0)  # nearly none of it
    ids[3] = -1
    teacher[4, 3:] = -torch.inf
    compare(device, x, ids, teacher, w, 1.0, True)
    compare(device, x, ids, teacher, w, 2.0, True)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("size", [(9, 700, 8), (9, 5003, 70), (81, 5003, 8), (81, 5003, 70)], ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_rows_without_entries_have_loss_and_gradient_0(device, size, dtype, tail):
    x, ids, teacher, w = make(24, *size, dtype, tail=tail)
    w[:] = torch.linspace(-1.0, 2.0, size[0])
    kinds = [lambda r: None, lambda r: r.fill_(float("nan")), lambda r: r.fill_(-torch.inf), lambda r: r[5:6].fill_(float("nan")),
             lambda r: r[-1:].fill_(torch.inf), lambda r: r.fill_(torch.finfo(dtype).max)]
    for t in range(size[0]):
        if t % 4 != 1:
            ids[t] = -1 if t % 2 else size[1]
            kinds[t % len(kinds)](x[t])
    bare = (ids < 0).all(1) | (ids >= size[1]).all(1)
    s = backend(device, dtype)
    xd, *rest = (t.to(device) for t in (x, ids, teacher, w))
    loss = s.loss(xd, *rest, tail=tail)
    both, grad = s.loss_and_grad(xd, *rest, tail=tail)
    leaf = xd.clone().requires_grad_()
    last = distill_loss(leaf, *rest, tail=tail, backend=s)
    last.sum().backward()
    for v in (loss, both, last.detach(), grad, leaf.grad):
        assert not v[bare].any()
    live = ~bare
    compare(device, x[live], ids[live], teacher[live], w[live], 1.0, tail)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_infinite_losses_and_nan_rows(device, tail):
    x, ids, teacher, w = make(23, 3, 600, 8, tail=tail)
    w[:] = 1.0
    x[0, int(ids[0, 2])] = -torch.inf  # an entry that the student excludes
    x[1, 5] = float("nan")
    x[2, int(ids[2, 0])] = float("nan")
    loss, grad = backend(device, torch.float32).loss_and_grad(*(t.to(device) for t in (x, ids, teacher, w)), tail=tail)
    assert float(loss[0]) == np.inf and bool(torch.isnan(loss[1:]).all())
    assert bool(torch.isfinite(grad[0]).all()) and bool(torch.isnan(grad[1]).any()) and bool(torch.isnan(grad[2]).any())
    want = ops_oracle.distill(x[:1].numpy(), ids[:1].numpy(), teacher[:1].numpy(), None, 1.0, tail)[1]
    np.testing.assert_allclose(grad[0].cpu().numpy(), want[0], rtol=1e-4, atol=1e-7)


@pytest.mark.gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_large_batches_of_large_logits(dtype, tail):
    for size in (100.0, 1e4, 1e20):
        x, ids, teacher, w = make(72, 70, 5003, 9, dtype, tail=tail)
        x[::2] += size
        x[1::2] -= size
        compare(GPU, x, ids, teacher, w, 1.0, tail)


@pytest.mark.parametrize("T", [1e-6, 1e-3, 1e6])
@pytest.mark.parametrize("size", [(3, 700, 8), (70, 5001, 8)], ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_extreme_temperatures_stay_finite(device, size, T):
    # (cold: one entry and one logit hold everything; hot: all are equal. The values go by the scale of 1 / T, so only what
    # does not depend on roundings of z is asked for)
    x, ids, teacher, w = make(71, *size)
    w[:] = 1.0
    loss, grad = backend(device, torch.float32).loss_and_grad(*(t.to(device) for t in (x, ids, teacher, w)), temperature=T)
    assert bool(torch.isfinite(loss).all()) and bool(torch.isfinite(grad).all())
    total = grad.double().sum(1).cpu().abs() * T  # q and p sum to 1 each
    assert float(total.max()) <= 1e-4


@pytest.mark.parametrize("T", [0.1, 1.0 / 3.0])
@pytest.mark.parametrize("size", [(5, 33, 4), (3, 5003, 70), (80, 5003, 9)], ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_temperatures_that_fp32_does_not_hold(device, size, T):
    # (0.1 in fp32 is off by 2^-26 of itself, and the teacher's logits lie 100 apart when divided by it)
    x, ids, teacher, w = make(73, *size)
    for tail in (False, True):
        compare(device, x, ids, teacher if not tail else torch.log_softmax(teacher, 1) - 0.1, w, T, tail)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_no_rows(device):
    x, ids, teacher, w = (t.to(device) for t in make(1, 0, 50, 3))
    loss, grad = backend(device, torch.float32).loss_and_grad(x, ids, teacher, w)
    assert loss.shape == (0,) and grad.shape == (0, 50)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_rows_at_any_offset_and_stride(dtype):
    x, ids, teacher, w = make(31, 6, 4211, 9, dtype)
    ids = ids % 4001
    ids = torch.where((ids[:, :, None] == ids[:, None, :]).tril(-1).any(2), -1, ids)  # (distinct again)
    for off in (0, 1, 5):
        compare(GPU, x[:, off : off + 4003], ids, teacher, w)
    compare(GPU, x[::2, :4003], ids[::2], teacher[::2], w[::2])


@pytest.mark.parametrize("T", [5, 80])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_one_row_for_all(device, T):
    # a broadcast student: its gradient is the rows' sum
    x, ids, teacher, w = make(43, T, 5003, 9)
    want = ops_oracle.distill(x[:1].expand(T, 5003).numpy(), ids.numpy(), teacher.numpy(), w.numpy(), 1.0, False)
    s = backend(device, torch.float32)
    leaf = x[:1].clone().to(device).requires_grad_()
    loss = distill_loss(leaf.expand(T, 5003), ids.to(device), teacher.to(device), w.to(device), backend=s)
    loss.sum().backward()
    tol_loss, tol_grad = tolerance(x[:1].expand(T, 5003), ids, teacher, w, *want, 1.0, False, torch.float32)
    assert np.all(np.abs(loss.detach().cpu().double().numpy() - want[0]) <= tol_loss)
    # (summed by torch in fp32: half a step of the running sum a row)
    size = np.abs(want[1]).sum(0)
    assert np.all(np.abs(leaf.grad[0].cpu().double().numpy() - want[1].sum(0)) <= tol_grad.sum(0) + T * 2.0**-24 * size)
    both = s.loss_and_grad(leaf.detach().expand(T, 5003), ids.to(device), teacher.to(device), w.to(device))[1]
    assert np.all(np.abs(both.cpu().double().numpy() - want[1]) <= tol_grad)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_incoming_gradients_weigh_the_rows(device):
    x, ids, teacher, w = make(41, 6, 700, 9)
    w[2] = 0.0
    g = torch.tensor([1.0, 0.0, 3.0, -2.0, 0.5, 1.0])
    s = backend(device, torch.float32)
    leaf = x.clone().to(device).requires_grad_()
    rest = [t.to(device) for t in (ids, teacher, w)]
    (distill_loss(leaf, *rest, temperature=1.5, tail=False, backend=s) * g.to(device)).sum().backward()
    want = ops_oracle.distill(x.numpy(), ids.numpy(), teacher.numpy(), (w * g).numpy(), 1.5, False)[1]
    np.testing.assert_allclose(leaf.grad.cpu().numpy(), want, rtol=2e-5, atol=1e-7)
    with torch.no_grad():
        assert not distill_loss(leaf, *rest, backend=s).requires_grad


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_rows_of_weight_0_take_no_incoming_gradient(device):
    x, ids, teacher, w = make(46, 6, 700, 9)
    w[:] = 0.5
    w[[0, 2, 3]] = 0.0
    g = torch.tensor([torch.inf, 2.0, float("nan"), -torch.inf, 1.0, -3.0])
    x[0] = float("nan")
    leaf = x.clone().to(device).requires_grad_()
    loss = distill_loss(leaf, *(t.to(device) for t in (ids, teacher, w)), backend=backend(device, torch.float32))
    loss.backward(g.to(device))
    assert not leaf.grad[w == 0].any()
    eff = torch.where(w == 0, 0.0, w * g)
    want = ops_oracle.distill(x.numpy(), ids.numpy(), teacher.numpy(), eff.numpy(), 1.0, False)
    _, tol = tolerance(x, ids, teacher, eff, *want, 1.0, False, torch.float32)
    assert np.all(np.abs(leaf.grad.cpu().double().numpy() - want[1]) <= tol)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T", [1.0, 0.1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_rows_of_weight_0_have_gradient_0_under_any_later_weights(device, dtype, T, tail):
    x, ids, teacher, w = make(45, 12, 5003, 9, dtype, tail=tail)
    w[:] = 1.0
    w[[1, 3, 4, 8, 11]] = 0.0
    x[1] = 120.0  # (exp(x) and exp(x / 0.1) are infinite in fp32)
    x[3] = float("nan")
    x[4] = torch.inf
    x[8] = torch.finfo(dtype).max
    x[11, ::2] = -torch.inf
    s = backend(device, dtype)
    xd, *rest = (t.to(device) for t in (x, ids, teacher, w))
    loss, states = s.loss_and_states(xd, *rest, temperature=T, tail=tail)
    other = torch.linspace(-1.5, 2.5, 12)
    for later in (None, other):
        grad = s.grad(xd, rest[0], states, None if later is None else later.to(device), temperature=T)
        eff = (torch.ones(12) if later is None else later) * (w != 0)
        want = ops_oracle.distill(x.float().numpy(), ids.numpy(), teacher.numpy(), eff.numpy(), T, tail)
        _, tol = tolerance(x, ids, teacher, eff, *want, T, tail, dtype)
        assert not loss[w == 0].any() and not grad[w == 0].any()
        assert np.all(np.abs(grad.cpu().double().numpy() - want[1]) <= tol)


@pytest.mark.gpu
def test_calls_are_deterministic_on_any_stream_and_in_graphs():
    x, ids, teacher, w = (t.to(GPU) for t in make(51, 300, 20011, 30, torch.bfloat16, zeros=True))
    s = backend(GPU, torch.bfloat16)
    want = s.loss_and_grad(x, ids, teacher, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = s.loss_and_grad(x, ids, teacher, w)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.loss_and_grad(x, ids, teacher, w)
    for i in range(3):
        x.copy_(torch.roll(x, 1, 1))
        graph.replay()
        eager = s.loss_and_grad(x, ids, teacher, w)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.gpu
def test_forward_and_backward_in_one_graph():
    x, ids, teacher, w = (t.to(GPU) for t in make(52, 40, 5003, 12))
    x.requires_grad_()
    x.grad = torch.zeros_like(x)

    def step():
        x.grad.zero_()
        loss = distill_loss(x, ids, teacher, w, tail=False)
        loss.sum().backward()
        return loss.detach()

    side = torch.cuda.Stream()  # (a warm-up that leaves no graph of the leaf behind, as capture wants it)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    s = backend(GPU, torch.float32)
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.roll(x, 1, 1))
        graph.replay()
        # (the same calls, eagerly: loss_and_grad may take the row in one pass, whose sums round elsewhere)
        want, states = s.loss_and_states(x.detach(), ids, teacher, w)
        grad = s.grad(x.detach(), ids, states, w)
        torch.cuda.synchronize()
        assert torch.equal(loss, want) and torch.equal(x.grad, grad)


@pytest.mark.parametrize("rows,vocab,dtype,ok", [
    ((1 << 24) - 1, 200, 0, True), (1 << 24, 200, 0, False), ((1 << 31) - 1, 1, 1, False), (1 << 23, 16385, 0, False),
    ((1 << 23) - 1, 16384, 1, True), (1 << 23, 8193, 1, False), (1 << 18, 524288, 1, False)], ids=str)
def test_more_segments_than_a_launch_takes_are_refused(rows, vocab, dtype, ok):
    # a launch has fewer than 2^32 threads in a dimension (refused before any device is looked for)
    lib = _vops.load()
    a = _vops.VopsDistillArgs()
    a.student, a.dtype, a.rows, a.vocab, a.entries, a.row_stride = 0x1000, dtype, rows, vocab, 8, vocab
    a.ids, a.teacher, a.temperature, a.out_loss, a.states = 0x2000, 0x3000, 1.0, 0x4000, 0x7000
    a.workspace, a.workspace_bytes = 0x5000, 1 << 60
    if torch.cuda.is_available() and ok:
        pytest.skip("would run")
    for entry in (lib.vops_distill, lib.vops_distill_grad):
        a.out_grad, a.grad_stride = (0x6000, vocab) if entry is lib.vops_distill_grad else (None, 0)
        code = entry(ctypes.byref(a), None)
        assert (code == 1 and b"too many rows" in lib.vops_last_error()) == (not ok)


def test_the_family_has_both_backends():
    assert DISTILL.names() == ["hip", "reference"]
    with pytest.raises(ValueError, match="distill backend 'hip' does not run on cpu"):
        DISTILL.resolve("hip", BackendContext(torch.device("cpu"), torch.bfloat16))
    with pytest.raises(ValueError, match="does not support torch.float16"):
        DISTILL.resolve("hip", BackendContext(GPU, torch.float16))


BAD = [
    (dict(student=torch.zeros(4, 9, dtype=torch.float16)), "bf16 and fp32"),
    (dict(student=torch.zeros(4)), "student must be"),
    (dict(student=torch.zeros(9, 4).T), "student must be"),
    (dict(student=torch.zeros(4, 0)), "vocab must be"),
    (dict(ids=torch.zeros(4, 3, dtype=torch.int64)), "ids must be"),
    (dict(ids=torch.zeros(3, 3, dtype=torch.int32)), "ids must be"),
    (dict(ids=torch.zeros(4, 0, dtype=torch.int32)), "entries"),
    (dict(ids=torch.zeros(4, 1025, dtype=torch.int32)), "entries"),
    (dict(teacher=torch.zeros(4, 2)), "teacher must be"),
    (dict(teacher=torch.zeros(4, 3, dtype=torch.bfloat16)), "teacher must be"),
    (dict(weights=torch.zeros(3)), "weights must be"),
    (dict(temperature=0.0), "temperature"),
    (dict(temperature=1e-7), "temperature"),
    (dict(temperature=2e6), "temperature"),
    (dict(temperature=float("inf")), "temperature"),
    (dict(temperature=float("nan")), "temperature"),
]


@pytest.mark.parametrize("kw,msg", BAD, ids=[m + str(i) for i, (_, m) in enumerate(BAD)])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_arguments_that_do_not_fit_are_refused(device, kw, msg):
    a = dict(student=torch.zeros(4, 9), ids=torch.zeros(4, 3, dtype=torch.int32), teacher=torch.zeros(4, 3)) | kw
    a = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    s = backend(device, torch.float32)
    args = a.pop("student"), a.pop("ids"), a.pop("teacher")
    for f in (s.loss, s.loss_and_grad, s.loss_and_states):
        with pytest.raises(ValueError, match=msg):
            f(*args, **a)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_states_of_another_shape_and_gradients_of_constants_are_refused(device):
    x, ids, teacher, w = (t.to(device) for t in make(1, 4, 9, 3))
    s = backend(device, torch.float32)
    for states in (torch.zeros(4, 4), torch.zeros(4, 5, dtype=torch.float64), torch.zeros(5, 4).T):
        with pytest.raises(ValueError, match="states must be"):
            s.grad(x, ids, states.to(device))
    with pytest.raises(ValueError, match="student's logits only"):
        distill_loss(x, ids, teacher.requires_grad_(), w, backend=s)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_tangents_of_forward_mode_are_refused(device):
    x, ids, teacher, w = (t.to(device) for t in make(2, 4, 9, 3))
    s = backend(device, torch.float32)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(x), ids, teacher, w), (dual(x.clone().requires_grad_()), ids, teacher, w), (x, ids, dual(teacher), w),
                     (x, ids, teacher, dual(w))):
            with pytest.raises(ValueError, match="forward-mode"):
                distill_loss(*args, backend=s)
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            distill_loss(dual(x), ids, teacher, backend=s)
        assert distill_loss(x, ids, teacher, w, backend=s).shape == (4,)


@pytest.mark.parametrize(
    "kw,code,msg",
    [
        ({"dtype": 5}, 2, b"dtype"),
        ({"rows": -1}, 1, b"rows"),
        ({"vocab": 0}, 1, b"vocab"),
        ({"entries": 1025}, 1, b"entries"),
        ({"flags": 2}, 1, b"flags"),
        ({"row_stride": -1}, 1, b"row_stride"),
        ({"grad_stride": 99}, 1, b"grad_stride"),
        ({"temperature": -1.0}, 1, b"temperature"),
        ({"student": None}, 1, b"must be set"),
        ({"student": 0x1001}, 1, b"aligned"),
        ({"teacher": None}, 1, b"must be set"),
        ({"out_loss": None}, 1, b"must be set"),
        ({"workspace_bytes": 16}, 4, b"needed"),
        ({"workspace": 0x5004}, 4, b"256-byte"),
    ],
)
def test_the_library_refuses_before_it_looks_for_a_device(kw, code, msg):
    lib = _vops.load()
    a = _vops.VopsDistillArgs()
    a.student, a.dtype, a.rows, a.vocab, a.entries, a.row_stride = 0x1000, 0, 4, 100, 8, 100
    a.ids, a.teacher, a.temperature, a.out_loss, a.out_grad, a.grad_stride = 0x2000, 0x3000, 1.0, 0x4000, 0x6000, 100
    a.workspace, a.workspace_bytes = 0x5000, 1 << 20
    for k, v in kw.items():
        setattr(a, k, v)
    assert lib.vops_distill(ctypes.byref(a), None) == code
    assert msg in lib.vops_last_error()
    if "states" not in kw and kw.keys() <= {"dtype", "rows", "vocab", "entries", "flags", "temperature"}:
        assert lib.vops_distill_grad(ctypes.byref(a), None) == code

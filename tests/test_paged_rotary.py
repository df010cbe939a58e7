"""Rotation and storing of the paged cache (``rotate_store``): the reference backend and the hip kernel against
products of complex numbers in 64 bits."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import paged_oracle
from vinfer_amd.paged import PAGED, Rotary, rotary_frequencies
from vinfer_amd.registry import BackendContext

GPU = torch.device("cuda", 0)
DEVICES = [torch.device("cpu"), pytest.param(GPU, marks=pytest.mark.gpu)]
BF16, F16 = torch.bfloat16, torch.float16


def backend(device, dtype=BF16):
    return PAGED.resolve("hip" if device.type == "cuda" else "reference", BackendContext(device, dtype))


def tensors(device, dtype, N, heads, kv_heads, D, layout, seed):
    """q, k and v: apart, of one product, heads before tokens, or at odd addresses."""
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    if layout == "fused":
        x = mk(N, (heads + 2 * kv_heads) * D)
        return [t.unflatten(1, (-1, D)) for t in x.split([heads * D, kv_heads * D, kv_heads * D], 1)]
    if layout == "heads":
        return [mk(h, N, D).transpose(0, 1) for h in (heads, kv_heads, kv_heads)]
    if layout == "odd":
        return [mk(N, h, D + 3)[..., 1 : D + 1] for h in (heads, kv_heads, kv_heads)]
    return [mk(N, h, D) for h in (heads, kv_heads, kv_heads)]


def caches(device, dtype, P, page, kv_heads, D, order):
    shape = {"places": (P, page, kv_heads, D), "heads": (P, kv_heads, page, D), "odd": (P, page, kv_heads, D + 1)}[order]
    made = [torch.full(shape, 7.0, dtype=dtype, device=device) for _ in range(2)]
    return [t.transpose(1, 2) if order == "heads" else t[..., :D] if order == "odd" else t for t in made]


def check(device, dtype, N, heads, kv_heads, D, rotary, positions, slots, page=16, layout="apart", order="places", seed=0):
    q, k, v = tensors(device, dtype, N, heads, kv_heads, D, layout, seed)
    P = 3 + N // page
    k_pages, v_pages = caches(device, dtype, P, page, kv_heads, D, order)
    f = rotary.frequencies.cpu().numpy()
    pos, at = np.asarray(positions, np.int64), np.asarray(slots, np.int64)
    words = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    got = backend(device, dtype).rotate_store(q, k, v, words(pos), words(at), k_pages, v_pages, rotary)
    host = lambda t: t.double().cpu().numpy()  # noqa: E731
    step = torch.finfo(dtype).eps / 2
    # one rounding to the type (fp16: half a subnormal's step at least), and in fp32: an angle in turns rounded to 25
    # bits, its sine and cosine, the magnitude's factor, two products and a sum, all below 8 steps of 2^-24 of |x1| + |x2|
    far = np.abs(pos).max(initial=0) * 2.0**-51
    size = rotary.magnitude * 2 * 8.0

    def near(a, b):
        assert np.all(np.abs(a - b) <= step * np.abs(b) + size * (2.0**-21 + far) + 2.0**-25), np.abs(a - b).max()

    want = paged_oracle.rotate(host(q), pos, f, rotary.interleaved, rotary.magnitude)
    want[pos < 0] = 0.0
    h = 2 * len(f)
    near(host(got), want)
    np.testing.assert_array_equal(host(got)[..., h:], want[..., h:])
    turned = paged_oracle.rotate(host(k), pos, f, rotary.interleaved, rotary.magnitude)
    cache = np.full((2, P * page, kv_heads, D), 7.0)
    for i in range(N):
        if pos[i] >= 0 and 0 <= at[i] < P * page:
            cache[0, at[i]], cache[1, at[i]] = turned[i], host(v)[i]
    near(host(k_pages).reshape(P * page, kv_heads, D), cache[0])
    np.testing.assert_array_equal(host(v_pages).reshape(P * page, kv_heads, D), cache[1])


SHAPES = [  # heads, kv_heads, D, turned elements
    (4, 2, 64, 64), (3, 1, 128, 128), (8, 8, 128, 32), (6, 2, 72, 36), (5, 5, 80, 80), (2, 1, 256, 256), (7, 1, 96, 18),
    (1, 1, 2, 2), (3, 3, 7, 4), (2, 2, 192, 0),
]


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_layouts(device, dtype, shape, interleaved):
    heads, kv_heads, D, dim = shape
    for i, (N, layout, order) in enumerate(((1, "apart", "places"), (37, "fused", "heads"), (5, "heads", "places"),
                                            (9, "odd", "odd"))):
        rng = np.random.default_rng(i)
        r = Rotary(rotary_frequencies(dim, base=500000.0, device=device), interleaved=interleaved)
        check(device, dtype, N, heads, kv_heads, D, r, rng.integers(0, 5000, N), rng.permutation((3 + N // 16) * 16)[:N],
              layout=layout, order=order, seed=i)


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_far_positions_of_a_stretched_context(device, interleaved):
    f = rotary_frequencies(128, base=10000.0, stretch=32.0, trained=4096, device=device)
    r = Rotary(f, interleaved=interleaved, magnitude=0.1 * math.log(32.0) + 1.0)
    check(device, F16, 40, 2, 1, 128, r, np.linspace(1, 1 << 20, 40).astype(int), np.arange(40))
    check(device, BF16, 3, 2, 1, 128, r, [0, 1, (1 << 31) - 1], [5, 3, 4], page=4096)


@pytest.mark.parametrize("vectors", [True, False], ids=["vectors", "elements"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_tokens_that_are_none_and_slots_outside(device, interleaved, vectors):
    D = 64 if vectors else 66
    r = Rotary(rotary_frequencies(D - 2 * 16, device=device), interleaved=interleaved)
    check(device, BF16, 8, 3, 2, D, r, [4, -1, 9, -7, 0, 3, 2, 1], [0, 1, -1, -1, 4, 48 + 8 // 16 * 16, 1 << 30, -(1 << 31)])


@pytest.mark.gpu
@pytest.mark.parametrize("N", [255, 4095, 4097])
def test_many_tokens(N):
    # one token a workgroup with its heads over several, and four tokens a workgroup
    rng = np.random.default_rng(N)
    r = Rotary(rotary_frequencies(64, device=GPU))
    check(GPU, BF16, N, 4, 2, 64, r, rng.integers(-1, 100000, N), rng.permutation((3 + N // 16) * 16)[:N], layout="fused")


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_nothing(device):
    r = Rotary(rotary_frequencies(64, device=device))
    check(device, BF16, 0, 4, 2, 64, r, [], [])
    check(device, BF16, 3, 0, 1, 64, r, [1, 2, 3], [0, 1, 2])
    check(device, BF16, 3, 2, 0, 64, r, [1, 2, 3], [0, 1, 2])


def test_frequencies():
    f = rotary_frequencies(8, base=100.0)
    np.testing.assert_allclose(f.numpy(), [1.0, 100**-0.25, 0.1, 100**-0.75], rtol=1e-15)
    np.testing.assert_allclose(rotary_frequencies(8, base=100.0, stretch=4.0).numpy(), f.numpy() / 4, rtol=1e-15)
    # over 2 pi 10 positions they turn 10, 3.16, 1 and 0.316 times
    g = rotary_frequencies(8, base=100.0, stretch=4.0, trained=63, turns=(1.0, 10.0)).numpy() / f.numpy()
    turns = 63 / (2 * math.pi) * f.numpy()
    np.testing.assert_allclose(g, [1.0, 0.25 + 0.75 * (turns[1] - 1) / 9, 0.25 + 0.75 * (turns[2] - 1) / 9, 0.25], rtol=1e-13)
    for bad in (dict(dim=7), dict(dim=8, base=0.0), dict(dim=8, stretch=-1.0), dict(dim=8, trained=0),
                dict(dim=8, trained=9, turns=(2.0, 2.0))):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_refusals():
    b = backend(torch.device("cpu"))
    r = Rotary(rotary_frequencies(8))
    mk = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt)  # noqa: E731
    i32 = torch.int32
    good = dict(q=mk(3, 4, 8), k=mk(3, 2, 8), v=mk(3, 2, 8), positions=mk(3, dt=i32), slots=mk(3, dt=i32), k_pages=mk(2, 16, 2, 8),
                v_pages=mk(2, 16, 2, 8), rotary=r)
    b.rotate_store(**good)
    for bad, match in (({"q": mk(2, 4, 8)}, "q must be"), ({"v": mk(3, 1, 8)}, "k and v"), ({"k": mk(3, 2, 8, dt=F16)}, "one type"),
                       ({"q": mk(3, 8, 4).transpose(1, 2)}, "unit stride"), ({"positions": mk(3, dt=torch.int64)}, "positions"),
                       ({"slots": mk(4, dt=i32)}, "slots"), ({"k_pages": mk(2, 16, 1, 8)}, "k_pages"),
                       ({"v_pages": mk(3, 16, 2, 8)}, "one shape"), ({"v_pages": mk(2, 2, 16, 8).transpose(1, 2)}, "one layout"),
                       ({"k_pages": mk(2, 12, 2, 8), "v_pages": mk(2, 12, 2, 8)}, "power of two"),
                       ({"rotary": Rotary(rotary_frequencies(10))}, "at most 8"), ({"q": mk(3, 4, 8).requires_grad_()}, "gradient"),
                       ({"q": mk(3, 4, 264), "k": mk(3, 2, 264), "v": mk(3, 2, 264)}, "256")):
        with pytest.raises(ValueError, match=match):
            b.rotate_store(**{**good, **bad})
    for bad in (torch.zeros(4), torch.zeros(2, 2, dtype=torch.float64), torch.zeros(129, dtype=torch.float64)):
        with pytest.raises(ValueError):
            Rotary(bad)
    with pytest.raises(ValueError, match="magnitude"):
        Rotary(rotary_frequencies(8), magnitude=math.inf)


@pytest.mark.gpu
def test_more_tokens_than_a_grid_s_dimension_has_threads():
    # 2^24 tokens and some, against the same tokens in two calls
    N, cut, D = (1 << 24) + 5, 9_000_001, 8
    r = Rotary(rotary_frequencies(D, device=GPU))
    b = backend(GPU)
    q = torch.randn(N, 1, D, device=GPU).to(BF16)
    k, v = q.flip(0), -q
    positions = torch.arange(N, dtype=torch.int32, device=GPU)
    slots = positions.flip(0).contiguous()
    shape = (N + 15) // 16, 16, 1, D
    both = []
    for parts in (((0, N),), ((0, cut), (cut, N))):
        k_pages, v_pages = (torch.zeros(shape, dtype=BF16, device=GPU) for _ in range(2))
        out = [b.rotate_store(q[i:j], k[i:j], v[i:j], positions[i:j], slots[i:j], k_pages, v_pages, r) for i, j in parts]
        both.append((torch.cat(out), k_pages, v_pages))
    for x, y in zip(*both):
        assert torch.equal(x, y)
    assert int(torch.count_nonzero(both[0][0][-1])) > 0


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_derivatives_are_refused(device):
    b = backend(device)
    mk = lambda *s: torch.randn(*s).to(BF16).to(device)  # noqa: E731
    tensors = {"q": mk(3, 4, 8), "k": mk(3, 2, 8), "v": mk(3, 2, 8), "k_pages": mk(2, 16, 2, 8), "v_pages": mk(2, 16, 2, 8),
               "frequencies": rotary_frequencies(8, device=device)}
    words = torch.arange(3, dtype=torch.int32, device=device)

    def call(t):
        return b.rotate_store(t["q"], t["k"], t["v"], words, words, t["k_pages"], t["v_pages"], Rotary(t["frequencies"]))

    want = call(tensors)  # (what was checked once is checked again where a tensor asks for more)
    for name, t in tensors.items():
        with pytest.raises(ValueError, match=f"{name} requires a gradient"):
            call({**tensors, name: t.clone().requires_grad_()})
        with torch.autograd.forward_ad.dual_level():
            assert torch.equal(call(tensors), want)
            with pytest.raises(ValueError, match=f"{name} has a tangent"):
                call({**tensors, name: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))})


def test_magnitudes_that_fp32_does_not_hold_are_refused():
    for magnitude in (1e39, -1e300, math.nan):
        with pytest.raises(ValueError, match="magnitude"):
            Rotary(rotary_frequencies(8), magnitude=magnitude)

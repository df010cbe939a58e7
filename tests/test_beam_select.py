"""Beam search's selection (``beam_select``): the reference backend and the hip kernels against the plain
statement in 64 bits (``oracle/ops_oracle.py``).

Beams and tokens have to be equal. Scores are fp32: half a step of the result (2^-24 of it), and what the
hip kernels' sum of exponentials may be off. A term's exponent carries two roundings (the difference and the
product) and v_exp_f32 one ulp: relative errors of 2 |d| 2^-24 and 2^-23 for a logit d below the maximum. The
mean |d| under the softmax is at most ln V <= 13.2, and a thread adds at most 64 terms in fp32: in all
(13.2 + 1 + 32) 2^-23 relative to the sum, an absolute error of the lse."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import ops_oracle
from vinfer_amd import _vops
from vinfer_amd.registry import BackendContext
from vinfer_amd.sampler import SAMPLER

LSE_TOL = 46.2 * 2.0**-23
DEVICES = [torch.device("cpu"), pytest.param(torch.device("cuda", 0), marks=pytest.mark.gpu)]
GPU = torch.device("cuda", 0)


def backend(device, dtype):
    return SAMPLER.resolve("hip" if device.type == "cuda" else "reference", BackendContext(device, dtype))


def compare(device, logits, scores, n, finished=None, pad_id=0, keep_slots=False):
    """``logits`` on the CPU, possibly a view: moved with its strides."""
    want = ops_oracle.beam_select(logits.float().numpy(), scores.numpy(), n,
                                  None if finished is None else finished.numpy(), pad_id, keep_slots)
    if device.type == "cuda":
        flat = torch.empty(0, dtype=logits.dtype).set_(logits.untyped_storage())
        logits = flat.to(device).as_strided(logits.shape, logits.stride(), logits.storage_offset())
    got = backend(device, logits.dtype).beam_select(
        logits, scores.to(device), n, finished=None if finished is None else finished.to(device), pad_id=pad_id,
        keep_slots=keep_slots)
    s, b, t = (v.cpu().numpy() for v in got)
    assert s.dtype == np.float32 and b.dtype == np.int32 and t.dtype == np.int32
    np.testing.assert_array_equal(b, want[1])
    np.testing.assert_array_equal(t, want[2])
    live = want[1] >= 0
    assert np.all(np.isneginf(s[~live]))
    assert np.all(np.abs(s[live] - want[0][live]) <= 2.0**-24 * np.abs(want[0][live]) + LSE_TOL)
    return got


def rows(seed, B, W, V, dtype=torch.bfloat16, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, W, V, generator=g) * scale).to(dtype)
    return x, -3.0 - 2.0 * torch.rand(B, W, generator=g)


SIZES = [  # B, W, V, n
    (1, 1, 1, 1),
    (2, 3, 1, 5),
    (3, 2, 7, 16),
    (2, 1, 255, 1),
    (1, 4, 2048, 4),
    (2, 5, 2049, 10),
    (1, 16, 4099, 32),
    (3, 4, 32000, 8),
    (1, 64, 1000, 64),
    (2, 7, 50257, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_random_rows(device, size, dtype):
    B, W, V, n = size
    x, scores = rows(V + n, B, W, V, dtype)
    compare(device, x, scores, n, pad_id=3)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(1, 2, 524288, 4, torch.float32), (1, 3, 262144, 64, torch.bfloat16),
                                  (70, 4, 20011, 8, torch.bfloat16), (40, 16, 9001, 16, torch.float32)], ids=str)
def test_large_rows_and_batches(size):
    B, W, V, n, dtype = size
    x, scores = rows(V, B, W, V, dtype, scale=1.0)
    compare(GPU, x, scores, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("n", [1, 8, 9, 33])
def test_a_waves_bound_and_a_workgroups(n, dtype):
    """Requests enough for the longest segments; rows whose best logits lie in one lane's, one wave's or all places."""
    x, scores = rows(n, 72, 5, 20011, dtype)
    x[:, 0] = x[:, 0].sort(-1).values
    x[:, 1, :600] += 20.0
    x[:, 2, 64:] = -torch.inf
    x[:, 3] = -torch.inf
    x[:, 3, 1024:1032] = torch.arange(8).to(dtype)  # a single vector's or two
    x[:, 4] = x[:, 4].round()
    compare(GPU, x, scores, n)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_finished_dead_and_kept_places(device):
    x, scores = rows(5, 4, 6, 3001)
    finished = torch.zeros(4, 6, dtype=torch.bool)
    finished[0, 2] = finished[1, :] = finished[2, 0] = True
    scores[0, 4] = -torch.inf
    scores[1, 3] = -torch.inf  # (a finished beam that is dead)
    scores[3, 1:] = -torch.inf
    scores[2, 1] = float("nan")
    scores[2, 3] = torch.inf
    for keep in (False, True):
        compare(device, x, scores, 6, finished, pad_id=7, keep_slots=keep)
    compare(device, x, scores, 12, finished, pad_id=-5)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_first_step_has_one_row_for_all_beams(device):
    x, scores = rows(6, 3, 1, 5003, torch.float32)
    scores = scores.expand(3, 8).clone()
    scores[:, 1:] = -torch.inf
    for keep in (False, True):
        compare(device, x.expand(3, 8, 5003), scores, 8, keep_slots=keep)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_masks_infinities_and_nan(device, dtype):
    x, scores = rows(7, 2, 12, 9001, dtype)
    low = torch.finfo(dtype).min
    x[:, 0] = -torch.inf  # nothing is left
    x[:, 1, 5:] = -torch.inf  # fewer than are asked for
    x[:, 2, :] = low
    x[:, 2, 4000:4100] = 1.0  # a run of equal logits, the rest the type's lowest
    x[:, 3, 17] = float("nan")
    x[:, 4, 18] = torch.inf
    x[:, 5, :] = -torch.inf
    x[:, 5, 8990:] = torch.arange(11).to(dtype)  # allowed at the row's end alone
    x[:, 6, 1::2] = -torch.inf
    x[:, 7, :] = 0.0
    x[:, 7, ::3] = -0.0  # zeros of either sign are one value
    x[:, 8, 100:1500] = 12.0
    x[:, 9, :] = low
    x[:, 10, 3:700] = -torch.inf
    for n in (3, 12, 64):
        compare(device, x, scores, n)
    for w in range(12):  # each kind of row by itself
        compare(device, x[:, w : w + 1], scores[:, w : w + 1], 40)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("n", [8, 64])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_nans_among_equal_logits(device, n, dtype):
    # Equal logits crowd a segment's list. In the first beams some of each wave's lanes (8 or 4 elements every 2048 or
    # 1024) hold a NaN, and logits above the others', so that no maximum of a lane tells what the segment holds: such rows
    # have no candidates, whatever else is in them.
    g = torch.Generator().manual_seed(n)
    B, V = (72, 33001) if device.type == "cuda" else (2, 5000)
    e = 8 if dtype == torch.bfloat16 else 4
    x = torch.ones(B, 6, V, dtype=dtype)
    lane = torch.arange(V) // e % 64
    for w, (lanes, top) in enumerate([(7, 2.0), (40, 2.0), (63, 70000.0), (64, 2.0)]):
        x[:, w, lane < lanes] = top
        x[:, w, (torch.arange(V) % (256 * e) < lanes * e) & (torch.arange(V) % e == 1)] = float("nan")
    x[:, 3, 3] = torch.inf
    x[:, 4] = 70000.0
    x[:, 4, V // 3] = -float("nan")
    compare(device, x, -3.0 - 2.0 * torch.rand(B, 6, generator=g), n)
    compare(device, x[:, :4], torch.zeros(B, 4), n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_rows_of_the_lowest_value(device, dtype):
    # masked by the type's lowest value throughout, or but for a few ids: whole segments hold nothing else, and few of them
    low = torch.finfo(dtype).min
    for V in (300, 4196, 8492):
        x, scores = rows(8, 2, 3, V, dtype)
        x[:, 0] = low
        x[:, 1, 7:] = low
        x[:, 2, : V - 5] = low
        compare(device, x, scores, 6)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_logits_of_any_size(device):
    for size in (1e3, 1e5, 1e8, 1e20, 1e37):
        x, scores = rows(9, 2, 3, 5003, torch.float32, scale=1.0)
        compare(device, x + size, scores, 6)
        compare(device, x - size, scores, 6)
        compare(device, x * (size / 8), scores, 6)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_equal_rows_and_scores_go_by_beam(device):
    # every beam has the same row and score: whole lists of equal scores, in the order beam, logit, id
    x = torch.zeros(2, 9, 6000, dtype=torch.bfloat16)
    x[1, :, ::7] = 1.0
    scores = torch.full((2, 9), -1.5)
    compare(device, x, scores, 64)
    compare(device, x[:, :, :40], scores, 64)


@pytest.mark.gpu
def test_more_equal_scores_than_the_merge_holds():
    x = torch.zeros(1, 64, 70000, dtype=torch.bfloat16)
    compare(GPU, x, torch.full((1, 64), -1.0), 64)
    compare(GPU, x, torch.full((1, 64), -1.0), 64, keep_slots=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_rows_at_any_offset_and_stride(dtype):
    base, scores = rows(11, 3, 4, 4211, dtype)
    for off in (0, 1, 3):
        compare(GPU, base[:, :, off : off + 4097], scores, 6)
    compare(GPU, base[:, ::2, 2:4001], scores[:, ::2], 6)
    compare(GPU, base.transpose(0, 1)[:, :, 5:3000], scores.T, 6)


@pytest.mark.gpu
def test_large_terms_keep_their_precision():
    # a certain beam beside flat ones: their order hangs on the lse
    x = torch.zeros(1, 3, 30000, dtype=torch.float32)
    x[0, 0, 11], x[0, 1, 12] = 40.0, 10.3
    lse = [float(np.log(np.sum(np.exp(r.astype(np.float64))))) for r in x[0].numpy()]
    scores = torch.tensor([[-2.0, -2.0 + (lse[1] - 10.3), -2.0 + lse[2]]])  # the best of each: about -2
    for d in (2e-6, -2e-6):
        s = scores.clone()
        s[0, 1] += d
        compare(GPU, x, s, 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("V", [4096, 32768, 151936, 262144])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_segments_whose_listed_terms_are_all_one(device, V, dtype):
    # one logit of each 8 just above 0, the others 0: up to 512 listed vectors of 8 elements, each element's exponential 1
    x = torch.zeros(1, 4, V, dtype=dtype)
    x[..., ::8] = 1e-30
    x[:, 2, ::16] = -torch.inf
    x[:, 3] = -x[:, 3]
    scores = torch.tensor([[-1.0, -1.5, -2.0, -1.25]])
    for n in (4, 9):
        compare(device, x, scores, n)


@pytest.mark.gpu
def test_repeats_graphs_and_other_streams_agree():
    x, scores = rows(13, 5, 4, 151936)
    s = backend(GPU, torch.bfloat16)
    xd, sd = x.to(GPU), scores.to(GPU)
    want = [v.cpu() for v in s.beam_select(xd, sd, 8)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = s.beam_select(xd, sd, 8)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.beam_select(xd, sd, 8)
    for i in range(3):
        other = torch.roll(x, i, 2)
        xd.copy_(other)
        graph.replay()
        eager = s.beam_select(xd, sd, 8)
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a.view(torch.int32), b.view(torch.int32))


BAD = [
    (dict(logits=torch.zeros(2, 3)), "logits must be"),
    (dict(logits=torch.zeros(2, 3, 8).transpose(1, 2)), "logits must be"),
    (dict(logits=torch.zeros(2, 3, 8, dtype=torch.float16)), "bf16 and fp32"),
    (dict(logits=torch.zeros(2, 65, 8)), "beams must be"),
    (dict(logits=torch.zeros(1, 3, 8).expand(65536, 3, 8)), "65535 requests"),
    (dict(logits=torch.zeros(2, 3, 0)), "vocab must be"),
    (dict(n=0), "n must be"),
    (dict(n=65), "n must be"),
    (dict(n=2, keep_slots=True), "keep_slots"),
    (dict(pad_id=1 << 31), "pad_id"),
    (dict(scores=torch.zeros(2, 3, dtype=torch.float64)), "scores must be"),
    (dict(scores=torch.zeros(3, 2)), "scores must be"),
    (dict(finished=torch.zeros(2, 3, dtype=torch.uint8)), "finished must be"),
    (dict(finished=torch.zeros(2, 4, dtype=torch.bool)), "finished must be"),
]


@pytest.mark.parametrize("kw,msg", BAD, ids=[m + str(i) for i, (_, m) in enumerate(BAD)])
@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_arguments_that_do_not_fit_are_refused(device, kw, msg):
    a = dict(logits=torch.zeros(2, 3, 8), scores=torch.zeros(2, 3), n=3) | kw
    a = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    with pytest.raises(ValueError, match=msg):
        backend(device, torch.float32).beam_select(a.pop("logits"), a.pop("scores"), a.pop("n"), **a)


@pytest.mark.parametrize("device", DEVICES, ids=str)
def test_no_requests(device):
    s, b, t = backend(device, torch.float32).beam_select(torch.zeros(0, 3, 8, device=device), torch.zeros(0, 3, device=device), 3)
    assert s.shape == b.shape == t.shape == (0, 3)


@pytest.mark.parametrize(
    "kw,code,msg",
    [
        ({"dtype": 5}, 2, b"dtype"),
        ({"requests": -1}, 1, b"requests"),
        ({"requests": 65536}, 1, b"requests"),
        ({"beams": 65}, 1, b"beams"),
        ({"vocab": 600000}, 1, b"vocab"),
        ({"n": 0}, 1, b"n in"),
        ({"flags": 2}, 1, b"flags"),
        ({"flags": 1, "n": 3}, 1, b"KEEP_SLOTS"),
        ({"beam_stride": -8}, 1, b"strides"),
        ({"logits": None}, 1, b"must be set"),
        ({"logits": 0x1001}, 1, b"aligned"),
        ({"out_tokens": None}, 1, b"must be set"),
        ({"workspace_bytes": 64}, 4, b"needed"),
        ({"workspace": 0x5010}, 4, b"256-byte"),
    ],
)
def test_the_library_refuses_before_it_looks_for_a_device(kw, code, msg):
    lib = _vops.load()
    a = _vops.VopsBeamArgs()
    a.logits, a.dtype, a.requests, a.beams, a.vocab, a.request_stride, a.beam_stride = 0x1000, 0, 2, 4, 100, 400, 100
    a.scores, a.n, a.out_scores, a.out_beams, a.out_tokens = 0x2000, 4, 0x3000, 0x4000, 0x6000
    a.workspace, a.workspace_bytes = 0x5000, 1 << 20
    for k, v in kw.items():
        setattr(a, k, v)
    assert lib.vops_beam_select(ctypes.byref(a), None) == code
    assert msg in lib.vops_last_error()

"""Attention over 8-bit pages where one token draws nearly all the weight: what
the many others carry together is kept.

The scores are exact in FP32 steps (two columns of the query, whole numbers in
K, powers of two as K scales), so the bounds speak of the weights alone."""
from __future__ import annotations

import numpy as np
import pytest

import inference_c_b200 as P
from inference_c_b200 import workloads as W
from tests.gpu_cases import to_device_bits
from tests.q8_cases import Q8Case, widen

pytestmark = pytest.mark.gpu


def _case(L, at, gap, q_heads, kv_heads, hd, bs, dtype, cuda, rows=1):
    """One sequence whose position `at` scores about gap + h nats above the rest
    (h: the query head within its group) and has V of zero; the others' V is
    positive, their scores spread over a nat."""
    case = Q8Case([L], q_heads, kv_heads, hd, bs, dtype, seed=3, device=cuda, garbage=False)
    r = np.random.RandomState(L + at)
    n = case.k.q.shape[0]
    scale = 2.0 ** -3
    for pool in (case.k, case.v):
        pool.q[...] = 0
    t = np.arange(L)
    page = case.tables[0][t // bs].astype(np.int64)
    case.k.s[...] = 2.0 ** -7
    case.v.s[...] = (r.uniform(0.5, 1.0, (n, kv_heads)) * 2.0 ** -7).astype(np.float32)
    for g in range(kv_heads):
        lane, cols = case.k._cols(g)
        c0 = cols.start
        case.k.q[page, lane, t % bs, c0 + 1] = r.randint(-127, 128, L)
        case.k.q[page[at], lane, at % bs, c0] = 127
        case.k.q[page[at], lane, at % bs, c0 + 1] = 0
        case.v.q[page, lane, t % bs, cols] = r.randint(1, 128, (L, hd))
        case.v.q[page[at], lane, at % bs, cols] = 0
    q = np.zeros((rows, q_heads, hd), np.float32)
    group = q_heads // kv_heads
    # 16-bit numbers with few bits: q[0] * 127 / 128 * scale is the gap
    q[:, :, 0] = np.round((gap + np.arange(q_heads) % group) / scale)
    q[:, :, 1] = 4.0
    case.qbits = W.storage_bits(q, dtype)
    assert np.array_equal(widen(case.qbits, dtype), q)
    case.upload()
    return case, q.astype(np.float64), scale


def _want(case, q, scale, limits):
    """64-bit outputs [R, Hq, d], the sums of w |v| beside them, the largest
    |score| and the largest |v|."""
    L = int(case.lengths[0])
    k, v = case.k.read64(case.tables[0], L), case.v.read64(case.tables[0], L)
    group = case.q_heads // case.kv_heads
    out, mag, worst = np.zeros(q.shape), np.zeros(q.shape), 0.0
    for h in range(case.q_heads):
        g = h // group
        s = q[:, h] @ k[:, g].T * scale
        worst = max(worst, float(np.abs(s).max()))
        s[np.arange(L)[None] >= np.asarray(limits)[:, None]] = -np.inf
        e = np.exp(s - s.max(axis=1, keepdims=True))
        w = e / e.sum(axis=1, keepdims=True)
        out[:, h], mag[:, h] = w @ v[:, g], w @ np.abs(v[:, g])
    return out, mag, worst, float(np.abs(v).max())


def _relative(worst):
    """How far a weight may be off, relatively.  A score takes eight roundings
    (three in the sum, five in its factors and the difference to a maximum) of
    numbers up to 2 worst, exp and the steps between maxima 2^-22 each, the
    normaliser as much again; 64 roundings of the sum over the keys."""
    return 2 * (8 * 2.0 ** -24 * 2 * worst + 4 * 2.0 ** -22) + 64 * 2.0 ** -24


@pytest.mark.parametrize("q_heads,kv_heads,hd,bs,dtype", [
    (4, 1, 128, 16, "f16"), (8, 1, 128, 32, "bf16"), (16, 1, 128, 16, "f16"),
    (4, 2, 64, 16, "f16"), (8, 2, 64, 64, "bf16"), (10, 1, 64, 16, "f16"),
])
@pytest.mark.parametrize("L,at", [(40, 0), (256, 200), (700, 300), (20000, 0), (20000, 19999)])
@pytest.mark.parametrize("gap", [14, 17])
def test_decode_beside_a_dominant_token(lib, cuda, q_heads, kv_heads, hd, bs, dtype, L, at, gap):
    """A weight is kept to 2^-32 (half a step of 1 / (127 * 2^24)) of the largest
    of its 256 tokens, times the largest V scale there and a whole number up to
    127; so the keys of a pair are off by 256 * 2^-32 vmax times its largest
    weight at most, all of them by 2^-24 vmax times the pairs' largest weights
    (1 for the sink's pair, and nothing beside it for the others)."""
    import torch
    case, q, scale = _case(L, at, gap, q_heads, kv_heads, hd, bs, dtype, cuda)
    got = torch.full((1, q_heads, hd), float("nan"), device=cuda)
    P.q8_decode(case.layer(), case.batch(), case.d_q, got, scale, L,
                P.q8_decode_workspace(1, q_heads, kv_heads, hd, L))
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    want, mag, worst, vmax = _want(case, q, scale, [L])
    tol = _relative(worst) * mag + 1.01 * 2.0 ** -24 * vmax
    diff = np.abs(got.double().cpu().numpy() - want)
    assert np.all(diff <= tol), (float((diff / want).max()), float((tol / want).min()))


@pytest.mark.parametrize("gap", [14, 17])
def test_decode_beside_a_dominant_token_of_a_long_sequence(lib, cuda, gap):
    """131,072 tokens over many units, the sink first; with the mass."""
    import torch
    L, q_heads, hd = 131072, 8, 128
    case, q, scale = _case(L, 0, gap, q_heads, 1, hd, 16, "f16", cuda)
    got = torch.full((1, q_heads, hd), float("nan"), device=cuda)
    mass = torch.zeros(case.k.q.shape[0], 1, 16, device=cuda)
    P.q8_decode_mass(case.layer(), case.batch(), case.d_q, got, scale, L, mass,
                     P.decode_mass_workspace(1, q_heads, 1, hd, L))
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    want, mag, worst, vmax = _want(case, q, scale, [L])
    tol = _relative(worst) * mag + 1.01 * 2.0 ** -24 * vmax
    diff = np.abs(got.double().cpu().numpy() - want)
    assert np.all(diff <= tol), (float((diff / want).max()), float((tol / want).min()))
    # every head's weights sum to one
    assert abs(float(mass.double().sum()) - q_heads) <= q_heads * _relative(worst)


def test_decode_of_scores_that_overflow(lib, cuda):
    """A tile whose scores are all -inf has no weight; the others keep theirs."""
    import torch
    L = 512
    case = Q8Case([L], 1, 1, 128, 16, "bf16", seed=5, device=cuda, garbage=False)
    case.k.q[...], case.v.q[...] = 0, 1
    case.k.s[...], case.v.s[...] = 1.0, 0.5
    t = np.arange(L)
    page = case.tables[0][t // 16].astype(np.int64)
    case.k.q[page[:256], 0, t[:256] % 16, 0] = -127
    case.k.s[page[:256], 0] = 2.0 ** 100
    case.v.q[page[:256], 0, t[:256] % 16] = 100
    q = np.zeros((1, 1, 128), np.float32)
    q[..., 0] = 2.0 ** 60
    case.qbits = W.storage_bits(q, "bf16")
    case.upload()
    got = torch.full((1, 1, 128), float("nan"), device=cuda)
    P.q8_decode(case.layer(), case.batch(), case.d_q, got, 1.0, L,
                P.q8_decode_workspace(1, 1, 1, 128, L))
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    # 256 equal weights of one value: 64 roundings of the sum, the digits' half step
    assert np.all(np.abs(got.double().cpu().numpy() - 0.5) <= 0.5 * (64 + 1) * 2.0 ** -24 + 2.0 ** -22)


@pytest.mark.parametrize("q_heads,kv_heads,hd,bs,dtype", [
    (4, 1, 128, 16, "f16"), (3, 1, 128, 32, "bf16"), (4, 2, 64, 16, "f16"), (2, 2, 64, 64, "bf16"),
])
@pytest.mark.parametrize("L,at", [(300, 0), (700, 300), (20000, 0), (20000, 19000)])
@pytest.mark.parametrize("gap", [14, 17])
def test_prefill_beside_a_dominant_token(lib, cuda, q_heads, kv_heads, hd, bs, dtype, L, at, gap):
    """A weight is kept as two 16-bit halves: fp16 2^-22 of it and down to 2^-36
    of the row's largest weight times V scale (half of fp16's least step,
    weights up to 2^15 above the running maximum), bf16 2^-16.  The first
    multiplies a whole number up to 127 and is divided by a sum of 1 / max(vs)
    at least, so L keys are off by L 2^-36 vmax.  The sum over the keys in 32
    bits takes an addition a half and 16 keys, each off by 2^-23 at most."""
    import torch
    n = 5
    case, q, scale = _case(L, at, gap, q_heads, kv_heads, hd, bs, dtype, cuda, rows=n)
    got = torch.full((n, q_heads, hd), float("nan"), device=cuda)
    P.q8_prefill(case.layer(), case.batch(), case.d_q, torch.tensor([0, n], dtype=torch.int32,
                                                                    device=cuda), got, scale, n, L,
                 P.q8_prefill_workspace(case.layer(), 1, L))
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    want, mag, worst, vmax = _want(case, q, scale, L - n + 1 + np.arange(n))
    halves = 2.0 ** -16 if dtype == "bf16" else 2.0 ** -22
    tol = (_relative(worst + 16) + halves + L / 8 * 2.0 ** -23) * mag
    tol += (L * 2.0 ** -36 if dtype == "f16" else 0) * vmax
    diff = np.abs(got.double().cpu().numpy() - want)
    assert np.all(diff <= tol), (float((diff / want).max()), float((tol / want).min()))

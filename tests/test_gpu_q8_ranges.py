"""8-bit pages whose V scales are far apart (bf16 rows span 2^-126 .. 2^121 of
scale): the pages of small values keep their share of the softmax."""
from __future__ import annotations

import numpy as np
import pytest

import inference_c_b200 as P
from inference_c_b200 import workloads as W
from tests.gpu_cases import to_device_bits
from tests.q8_cases import Q8Case, attend64, attend_tol, widen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,kv", [(128, 1), (64, 2)])
@pytest.mark.parametrize("amps", [
    (1.0, 1e-36), (1e-36, 1.0), (1e-30, 1e-34), (1e-36, 1e-36), (1e30, 1.0), (1e30, 1e-30),
])
@pytest.mark.parametrize("prefill", [True, False])
def test_scales_far_apart(lib, cuda, hd, kv, amps, prefill):
    """The errors stay in proportion to the largest value (bounds of the prefill
    and decode tests, vmax the case's own)."""
    import torch
    L, n, qh = 400, 40, 2 * kv
    case = Q8Case([L], qh, kv, hd, 16, "bf16", seed=57, device=cuda)
    x = W.normal(58, L * kv * hd).reshape(L, kv, hd).astype(np.float64)
    block = (np.arange(L) // 16) % 2
    x *= np.where(block == 0, amps[0], amps[1])[:, None, None]
    x = widen(W.storage_bits(x.astype(np.float32).reshape(-1), "bf16"), "bf16").reshape(L, kv, hd)
    case.v.write(case.tables[0], 0, x)
    case.upload()
    qbits = W.normal_bits(59, (n, qh, hd), "bf16", stream=9)
    q = widen(qbits, "bf16").astype(np.float64)
    if prefill:
        got = torch.full((n, qh, hd), float("nan"), device=cuda)
        offs = torch.tensor([0, n], dtype=torch.int32, device=cuda)
        ws = P.q8_prefill_workspace(case.layer(), 1, L)
        ws.fill_(255)
        P.q8_prefill(case.layer(), case.batch(), to_device_bits(qbits, "bf16", cuda), offs, got,
                     case.scale, n, L, ws)
    else:
        q = q[-1:]
        got = torch.full((1, qh, hd), float("nan"), device=cuda)
        P.q8_decode(case.layer(), case.batch(), to_device_bits(qbits[-1:], "bf16", cuda), got,
                    case.scale, L, P.q8_decode_workspace(1, qh, kv, hd, L))
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    k, v = case.k.read64(case.tables[0], L), case.v.read64(case.tables[0], L)
    rows = len(q)
    want, _, worst = attend64(q, k, v, case.scale, L - rows + 1 + np.arange(rows))
    vmax = float(np.abs(v).max())
    # beside the relative errors: 64 roundings of FP32's least numbers
    tol = attend_tol(worst, hd, vmax, want, 0) + 64 * 2.0 ** -149
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= tol + prefill * 2.0 ** -16 * vmax)

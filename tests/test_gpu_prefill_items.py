"""Prefills with several work items a CTA where a KV head's query heads do not
pair up: the tensor cores run ahead of the softmax from one item into the next."""
from __future__ import annotations

import numpy as np
import pytest

import inference_c_b200 as P
from tests.q8_cases import attend_tol

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("q_heads,kv_heads,hd,past,rows", [
    (28, 4, 128, 1400, 60), (15, 3, 64, 5, 400), (24, 8, 128, 200, 150), (8, 8, 128, 900, 520),
    (40, 8, 64, 350, 300), (5, 1, 128, 60, 2000),
])
def test_unpaired_heads_over_many_items(lib, cuda, q8, q_heads, kv_heads, hd, past, rows):
    """Against 64 bits, then the same bits in twenty more calls."""
    import torch
    B, bs, half = 8, 16, torch.float16
    g = torch.Generator(device="cuda").manual_seed(17)
    n = [rows - 7 * b % rows for b in range(B)]
    lens = [past + 13 * b + n[b] for b in range(B)]
    per = [-(-x // bs) for x in lens]
    pages = sum(per) + 1
    tables = torch.zeros(B, max(per), dtype=torch.int32, device=cuda)
    perm = torch.randperm(pages, generator=g, device=cuda).int()
    for b in range(B):
        tables[b, :per[b]] = perm[sum(per[:b]):sum(per[:b + 1])]
    if q8:
        lanes = P.q8_lanes(kv_heads, hd)
        pools = [torch.randint(-127, 128, (pages, lanes, bs, 128), generator=g, device=cuda,
                               dtype=torch.int8) for _ in range(2)]
        scales = [torch.rand(pages, kv_heads, generator=g, device=cuda) * 0.02 + 0.005
                  for _ in range(2)]
        layer = P.make_q8_layer(*pools, *scales, kv_heads, hd, half)

        def values(i, idx):
            x = pools[i][idx].transpose(1, 2).reshape(len(idx), bs, -1)[..., :kv_heads * hd]
            return x.reshape(len(idx), bs, kv_heads, hd).double() * \
                scales[i][idx].double()[:, None, :, None]
    else:
        pools = [torch.randn(pages * bs, kv_heads * hd, generator=g, device=cuda, dtype=half)
                 for _ in range(2)]
        layer = P.make_layer(*pools, bs, kv_heads, hd)

        def values(i, idx):
            return pools[i].view(pages, bs, kv_heads, hd)[idx].double()
    offs = torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device=cuda)
    d_lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
    batch = P.make_batch(tables, d_lens)
    q = torch.randn(sum(n), q_heads, hd, generator=g, device=cuda, dtype=half)
    ws = P.q8_prefill_workspace(layer, B, max(lens)) if q8 else None

    def call():
        out = torch.full((sum(n), q_heads, hd), float("nan"), device=cuda)
        if q8:
            P.q8_prefill(layer, batch, q, offs, out, hd ** -0.5, max(n), max(lens), ws)
        else:
            P.paged_prefill(layer, batch, q, offs, out, hd ** -0.5, max(n))
        return out
    out = call()
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    at = 0
    for b in range(B):
        idx = tables[b, :per[b]].long()
        k, v = (values(i, idx).reshape(-1, kv_heads, hd)[:lens[b]] for i in range(2))
        qd = q[at:at + n[b]].double().view(n[b], kv_heads, -1, hd)
        s = torch.einsum("rghd,tgd->rght", qd, k) * hd ** -0.5
        worst = float(torch.einsum("rghd,tgd->rght", qd.abs(), k.abs()).max()) * hd ** -0.5
        limit = lens[b] - n[b] + 1 + torch.arange(n[b], device=cuda)
        s.masked_fill_(torch.arange(lens[b], device=cuda) >= limit[:, None, None, None],
                       float("-inf"))
        want = torch.einsum("rght,tgd->rghd", torch.softmax(s, -1), v).reshape(n[b], q_heads, hd)
        vmax = float(v.abs().max())
        # weights as two fp16 halves
        tol = attend_tol(worst, hd, vmax, want.cpu().numpy(), 0) + 2.0 ** -21 * vmax
        assert np.all(np.abs((out[at:at + n[b]].double() - want).cpu().numpy()) <= tol), b
        at += n[b]
    for _ in range(20):
        again = call()
        off = (again - out).abs()
        assert torch.equal(again, out), (int((off != 0).sum()), float(off.max()), P.device_fault(0))
    assert P.device_fault(0) == 0

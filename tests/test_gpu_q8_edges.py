"""8-bit calls at the ends of what their arguments allow: no tokens at all, many
KV heads, scales of zero and below, captured and concurrent prefills."""
from __future__ import annotations

import numpy as np
import pytest

import inference_c_b200 as P
from inference_c_b200 import workloads as W
from tests.gpu_cases import to_device_bits
from tests.q8_cases import Q8Case, attend64, attend_tol, widen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [1, 3, 600])
def test_batches_without_a_token(lib, cuda, batch):
    """Zeros from the decodes, nothing added, nothing kept, nothing written."""
    import torch
    case = Q8Case([0] * batch, 8, 2, 64, 16, "f16", seed=3, device=cuda)
    before = [t.clone() for t in (case.d_kq, case.d_vq, case.d_ks, case.d_vs)]
    pages = case.k.q.shape[0]
    for bound in (0, 1, 500):
        out = torch.full((batch, 8, 64), float("nan"), device=cuda)
        mass = torch.rand(pages, 2, 16, device=cuda)
        held = mass.clone()
        ws = P.decode_mass_workspace(batch, 8, 2, 64, bound)
        P.q8_decode(case.layer(), case.batch(), case.d_q, out, case.scale, bound, ws)
        assert not out.any()
        out.fill_(float("nan"))
        P.q8_decode_mass(case.layer(), case.batch(), case.d_q, out, case.scale, bound, mass, ws)
        assert not out.any() and torch.equal(mass, held)
        kept = torch.full((batch, 2, 5), 9, dtype=torch.int32, device=cuda)
        P.kv_evict(case.layer(), case.batch(), mass, 5, 2, kept, bound)
        assert (kept == -1).all() and torch.equal(mass, held)
    offs = torch.zeros(batch + 1, dtype=torch.int32, device=cuda)
    rows = torch.ones(4, 128, dtype=torch.float16, device=cuda)  # none of them anyone's
    P.q8_append(case.layer(), case.batch(), rows, rows, offs)
    P.q8_import(case.layer(), case.batch(), rows, rows, offs)
    P.q8_gather(case.layer(), case.batch(), rows, rows, offs)
    P.mass_clear(case.layer(), case.batch(), mass, offs)
    query = torch.ones(4, 8, 64, dtype=torch.float16, device=cuda)
    out = torch.full((4, 8, 64), 7.0, device=cuda)
    P.q8_prefill(case.layer(), case.batch(), query, offs, out, 0.125, 1, 64,
                 P.q8_prefill_workspace(case.layer(), batch, 64))
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    assert (out == 7.0).all() and (rows == 1.0).all() and torch.equal(mass, held)
    for t, b in zip((case.d_kq, case.d_vq, case.d_ks, case.d_vs), before):
        assert torch.equal(t.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("kv_heads,hd", [(1024, 64), (1023, 64), (1024, 128)])
def test_as_many_kv_heads_as_a_layer_holds(lib, cuda, kv_heads, hd):
    import torch
    lens = [3, 0, 130]
    bs, pages = 16, 12
    g = torch.Generator(device="cuda").manual_seed(7)
    lanes = P.q8_lanes(kv_heads, hd)
    pools = [torch.zeros(pages, lanes, bs, 128, dtype=torch.int8, device=cuda) for _ in range(2)]
    scales = [torch.zeros(pages, kv_heads, device=cuda) for _ in range(2)]
    layer = P.make_q8_layer(*pools, *scales, kv_heads, hd, torch.float16)
    tables = torch.zeros(3, 9, dtype=torch.int32, device=cuda)
    perm = torch.randperm(pages, generator=g, device=cuda).int()
    tables[0, 0], tables[2] = perm[9], perm[:9]
    d_lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
    batch = P.make_batch(tables, d_lens)
    rows = [torch.randn(133, kv_heads * hd, generator=g, device=cuda).half() for _ in range(2)]
    offs = torch.tensor([0, 3, 3, 133], dtype=torch.int32, device=cuda)
    P.q8_import(layer, batch, *rows, offs)
    back = [torch.empty_like(r) for r in rows]
    P.q8_gather(layer, batch, *back, offs)
    q = torch.randn(3, kv_heads, hd, generator=g, device=cuda).half()
    out = torch.full((3, kv_heads, hd), float("nan"), device=cuda)
    mass = torch.zeros(pages, kv_heads, bs, device=cuda)
    ws = P.decode_mass_workspace(3, kv_heads, kv_heads, hd, 130)
    P.q8_decode_mass(layer, batch, q, out, hd ** -0.5, 130, mass, ws)
    pre = torch.full((3, kv_heads, hd), float("nan"), device=cuda)
    one = torch.tensor([0, 1, 1, 2], dtype=torch.int32, device=cuda)
    P.q8_prefill(layer, batch, q[[0, 2]], one, pre[:2], hd ** -0.5, 1, 130,
                 P.q8_prefill_workspace(layer, 3, 130))
    kept = torch.empty(3, kv_heads, 20, dtype=torch.int32, device=cuda)
    P.kv_evict(layer, batch, mass, 20, 4, kept, 130)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    assert not out[1].any()
    for b, (a, z) in ((0, (0, 3)), (2, (3, 133))):
        x, k = rows[0][a:z].float(), back[0][a:z].double().view(z - a, kv_heads, hd)
        v = back[1][a:z].double().view(z - a, kv_heads, hd)
        # stored within half a step of the page's scale, gathered with fp16's rounding
        top = x.view(z - a, kv_heads, hd).abs().amax(dim=(0, 2))
        assert bool(((k.float() - x.view_as(k)).abs() <=
                     (top / 127 * 0.501 + top * 2.0 ** -11)[None, :, None]).all())
        s = torch.einsum("hd,thd->ht", q[b].double(), k) * hd ** -0.5
        want = torch.einsum("ht,thd->hd", torch.softmax(s, -1), v)
        # the rows read back are rounded to fp16: values by 2^-11, scores by
        # 2^-11 of their terms
        worst = float(torch.einsum("hd,thd->ht", q[b].double().abs(), k.abs()).max()) * hd ** -0.5
        tol = (2 * 2.0 ** -11 * worst + 2.0 ** -10) * float(v.abs().max())
        assert float((out[b].double() - want).abs().max()) <= tol
        assert float((pre[0 if b == 0 else 1].double() - want).abs().max()) <= tol
    got = kept.cpu().numpy()
    assert (got[0, :, :3] == [0, 1, 2]).all() and (got[0, :, 3:] == -1).all()
    assert (got[1] == -1).all() and (got[2, :, -4:] == [126, 127, 128, 129]).all()
    assert (np.diff(got[2], axis=1) > 0).all()


@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30])
def test_decode_scales_of_zero_and_below(lib, cuda, scale):
    import torch
    case = Q8Case([300, 17], 12, 2, 128, 32, "bf16", seed=5, device=cuda)
    out = torch.full((2, 12, 128), float("nan"), device=cuda)
    ws = P.q8_decode_workspace(2, 12, 2, 128, 300)
    P.q8_decode(case.layer(), case.batch(), case.d_q, out, scale, 300, ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    q, got = widen(case.qbits, "bf16").astype(np.float64), out.double().cpu().numpy()
    for b, L in enumerate((300, 17)):
        k, v = case.k.read64(case.tables[b], L), case.v.read64(case.tables[b], L)
        want, _, worst = attend64(q[b:b + 1], k, v, scale)
        tol = attend_tol(worst, 128, float(np.abs(v).max()), want, 0)
        assert np.all(np.abs(got[b] - want[0]) <= tol[0])


def test_captured_and_concurrent_prefills(lib, cuda):
    """A captured append and prefill replayed on changed rows, and two prefills
    at once on streams and workspaces of their own, give the eager bits."""
    import torch
    cases = [Q8Case([700, 33, 260], 10, 2, 64, 16, "f16", seed=s, device=cuda) for s in (91, 92)]
    rows = [40, 33, 7]
    offs = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device=cuda)
    new = [[to_device_bits(W.normal_bits(s, (80, 128), "f16", stream=i), "f16", cuda) for i in (1, 2)]
           for s in (93, 94)]
    qs = [to_device_bits(W.normal_bits(s, (80, 10, 64), "f16", stream=3), "f16", cuda)
          for s in (93, 94)]
    ws = [P.q8_prefill_workspace(c.layer(), 3, 700) for c in cases]
    outs = [torch.empty(80, 10, 64, device=cuda) for _ in cases]

    def calls(i, stream=None):
        c = cases[i]
        P.q8_append(c.layer(), c.batch(), *new[i], offs, stream=stream)
        P.q8_prefill(c.layer(), c.batch(), qs[i], offs, outs[i], c.scale, 40, 700, ws[i],
                     stream=stream)
    for i in range(2):
        calls(i)
    torch.cuda.synchronize()
    eager = [o.clone() for o in outs]
    streams = [torch.cuda.Stream() for _ in cases]
    for o in outs:
        o.fill_(float("nan"))
    torch.cuda.synchronize()
    for _ in range(10):
        for i in range(2):
            calls(i, streams[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, eager))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        calls(0)
    for seed in (95, 96):
        for i in range(2):
            new[0][i].copy_(to_device_bits(W.normal_bits(seed, (80, 128), "f16", stream=i + 4),
                                           "f16", cuda))
        pages = [t.clone() for t in (cases[0].d_kq, cases[0].d_vq, cases[0].d_ks, cases[0].d_vs)]
        calls(0)
        torch.cuda.synchronize()
        want = outs[0].clone()
        for t, p in zip((cases[0].d_kq, cases[0].d_vq, cases[0].d_ks, cases[0].d_vs), pages):
            t.copy_(p)
        outs[0].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want)
    assert P.device_fault(0) == 0

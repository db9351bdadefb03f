"""The 8-bit cache as a program runs it: a pool with its transaction, captured
graphs, side streams, batches above one launch, pages past 4 GiB, bad input."""
from __future__ import annotations

import numpy as np
import pytest

import inference_c_b200 as P
from inference_c_b200 import workloads as W
from tests.gpu_cases import to_device_bits, torch_dtype
from tests.q8_cases import Q8Case, Q8Pool, attend64, attend_tol, lanes_of, widen
from tests.test_gpu_mass_evict import keep_list
from tests.test_gpu_q8 import check_decode

pytestmark = pytest.mark.gpu


def test_pool_steps_evict_and_set_length(lib, cuda):
    """Two sequences in an 8-bit pool: a prompt and a few tokens by steps, an
    eviction inside a step without new tokens, the pages behind it returned to
    the allocator, and more steps."""
    import torch
    kv, hd, bs, qh = 2, 128, 16, 8
    cache = P.PagedKVCache(bs, 40, 2)
    pool = P.PagedPool.q8(cache, 0, P.PKV_DTYPE_F16, 2, kv, hd, 2, 20, mass=True)
    with pytest.raises(P.PkvError):
        pool.layer(0)
    layer = pool.q8_layer(1)
    assert pool.mass(1) and layer.block_count == 40
    seqs = [cache.sequence_create(), cache.sequence_create()]
    host = [Q8Pool(40, kv, hd, bs) for _ in range(2)]  # K, V
    mass = np.zeros((2, kv, 512))
    lens = [0, 0]
    ws = P.decode_mass_workspace(2, qh, kv, hd, 320)
    out = torch.empty(2, qh, hd, dtype=torch.float32, device=cuda)
    kept = torch.empty(2, kv, 64, dtype=torch.int32, device=cuda)

    def step(new, seed, evict=False):
        bits = [W.normal_bits(seed, (sum(new), kv * hd), "f16", stream=s) for s in (1, 2)]
        qb = W.normal_bits(seed, (2, qh, hd), "f16", stream=3)
        pool.step_begin(seqs, new)
        batch = pool.step_batch()
        tables = [cache.block_table(s) for s in seqs]
        if evict:
            P.kv_evict(layer, batch, pool.mass(1), 64, 16, kept, 320)
        else:
            P.q8_append(layer, batch, to_device_bits(bits[0], "f16", cuda),
                        to_device_bits(bits[1], "f16", cuda), pool.step_row_offsets())
            P.mass_clear(layer, batch, pool.mass(1), pool.step_row_offsets())
            P.q8_decode_mass(layer, batch, to_device_bits(qb, "f16", cuda), out, hd ** -0.5, 320,
                             pool.mass(1), ws)
        torch.cuda.synchronize()
        pool.step_end(True)
        assert P.device_fault(0) == 0
        if evict:
            return tables
        at = 0
        for b in range(2):
            for p, x in zip(host, bits):
                rows = widen(x, "f16").reshape(-1, kv, hd)[at:at + new[b]]
                p.write(tables[b], lens[b], rows)
            at += new[b]
            lens[b] += new[b]
            k, v = (p.read64(tables[b], lens[b]) for p in host)
            want, w, worst = attend64(widen(qb[b:b + 1], "f16").astype(np.float64), k, v,
                                      hd ** -0.5)
            tol = attend_tol(worst, hd, float(np.abs(v).max()), want, 0)
            assert np.all(np.abs(out[b].double().cpu().numpy() - want[0]) <= tol[0])
            mass[b, :, :lens[b]] += w[0].reshape(kv, -1, lens[b]).sum(axis=1)
        return tables

    step([200, 33], 101)
    for i in range(3):
        step([1, 1], 110 + i)
    tables = step([0, 0], 0, evict=True)
    got = kept.cpu().numpy()
    for b in range(2):
        m = min(64, lens[b])
        assert (got[b, :, m:] == -1).all()
        for g in range(kv):
            pick = got[b, g, :m]
            old = lens[b] - 16
            if lens[b] > 64:  # the device's mass is within its tolerance of this one
                assert np.array_equal(np.sort(pick), pick) and (pick[-16:] == old + np.arange(16)).all()
                rest = np.setdiff1d(np.arange(old), pick)
                assert mass[b, g, rest].max() <= mass[b, g, pick[:-16]].min() * (1 + 1e-3)
            mass[b, g, :m] = mass[b, g, pick]
            mass[b, g, m:] = 0
            for p in host:
                lane, cols = p._cols(g)
                src = np.asarray(tables[b])[pick // bs]
                q, s = p.q[src, lane, pick % bs, cols].astype(np.float32), p.s[src, g].copy()
                for j in range(-(-m // bs)):
                    sl = slice(j * bs, min(m, (j + 1) * bs))
                    top = s[sl].max()
                    p.q[tables[b][j], lane, :sl.stop - sl.start, cols] = np.rint(
                        q[sl] * (s[sl] / top)[:, None])
                    p.s[tables[b][j], g] = top
        free = cache.free_blocks()
        assert cache.set_length(seqs[b], m)
        assert cache.free_blocks() == free + len(tables[b]) - (-(-m // bs))
        lens[b] = m
    for i in range(3):
        step([1, 1], 120 + i)
    step([40, 5], 130)
    cache.free()


def test_captured_graph_replays(lib, cuda):
    """Append, clear, decode with mass and an eviction into other pages as one
    captured graph, replayed on changed inputs, equals the eager calls."""
    import torch
    case = Q8Case([130, 40], 8, 2, 128, 16, "f16", seed=91, device=cuda, extra_pages=20)
    used = set(case.tables[:, :9].reshape(-1).tolist())
    free = [p for p in range(case.k.q.shape[0]) if p not in used][:8]
    dst = torch.tensor(free, dtype=torch.int32, device=cuda).view(2, 4)
    rows = to_device_bits(W.normal_bits(92, (2, 256), "f16", stream=1), "f16", cuda)
    ws = P.decode_mass_workspace(2, 8, 2, 128, 200)
    pages = case.k.q.shape[0]
    bufs = [case.d_kq, case.d_vq, case.d_ks, case.d_vs]
    mass = torch.rand(pages, 2, 16, device=cuda)
    out = torch.empty(2, 8, 128, dtype=torch.float32, device=cuda)
    kept = torch.empty(2, 2, 60, dtype=torch.int32, device=cuda)
    start = [t.clone() for t in bufs + [mass]]

    def calls():
        P.q8_append(case.layer(), case.batch(), rows, rows)
        P.mass_clear(case.layer(), case.batch(), mass)
        P.q8_decode_mass(case.layer(), case.batch(), case.d_q, out, case.scale, 200, mass, ws)
        P.kv_evict(case.layer(), case.batch(), mass, 60, 8, kept, 200, dst_tables=dst)

    def reset():
        for t, s in zip(bufs + [mass], start):
            t.copy_(s)
    calls()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        calls()
    for seed in (1, 2):
        case.d_q.copy_(to_device_bits(W.normal_bits(seed, (2, 8, 128), "f16", stream=7), "f16", cuda))
        rows.copy_(to_device_bits(W.normal_bits(seed, (2, 256), "f16", stream=8), "f16", cuda))
        reset()
        calls()
        torch.cuda.synchronize()
        want = [t.clone() for t in bufs + [mass, out, kept]]
        reset()
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(bufs + [mass, out, kept], want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert P.device_fault(0) == 0


def test_side_streams_with_workspaces_of_their_own(lib, cuda):
    import torch
    cases = [Q8Case([700, 33], 8, 2, 128, 16, "f16", seed=s, device=cuda) for s in (93, 94)]
    streams = [torch.cuda.Stream() for _ in cases]
    ws = [P.q8_decode_workspace(2, 8, 2, 128, 700) for _ in cases]
    outs = [torch.full((2, 8, 128), float("nan"), device=cuda) for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s, w, o in zip(cases, streams, ws, outs):
            P.q8_decode(c.layer(), c.batch(), c.d_q, o, c.scale, 700, w, stream=s)
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        check_decode(c, o.double().cpu().numpy(), 0)
    assert P.device_fault(0) == 0


def test_batch_above_one_launch_and_one_workspace_for_all(lib, cuda):
    """More sequences than one launch holds, many segments in a work unit, then
    a small batch with the same scratch."""
    import torch
    lengths = (W.uniform(5, 700) * 200).astype(np.int64)
    case = Q8Case(lengths, 2, 1, 64, 16, "f16", seed=95, device=cuda)
    ws = P.decode_mass_workspace(700, 2, 1, 64, 200)
    out = torch.full((700, 2, 64), float("nan"), device=cuda)
    mass = torch.zeros(case.k.q.shape[0], 1, 16, device=cuda)
    P.q8_decode_mass(case.layer(), case.batch(), case.d_q, out, case.scale, 200, mass, ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    check_decode(case, out.double().cpu().numpy(), 0)
    # every sequence's weights sum to its two query heads
    t = mass.cpu().numpy().reshape(case.k.q.shape[0], 16)
    for b, L in enumerate(lengths):
        total = t[case.tables[b][:-(-int(L) // 16)].astype(np.int64)].sum(dtype=np.float64)
        assert abs(total - (2 if L else 0)) < 1e-4
    one = Q8Case([150], 2, 1, 64, 16, "f16", seed=96, device=cuda)
    got = torch.full((1, 2, 64), float("nan"), device=cuda)
    P.q8_decode(one.layer(), one.batch(), one.d_q, got, one.scale, 200, ws)
    torch.cuda.synchronize()
    check_decode(one, got.double().cpu().numpy(), 0)


def test_long_launch_with_dynamic_units(lib, cuda):
    """Shares of more than 64 tiles a CTA: units of the dynamic tail, segments
    in several pieces, one far longer than the others; checked against the
    gathered rows in 64 bits on the GPU."""
    import torch
    lens = [60000, 3, 20011, 128, 9000, 31000]
    kv, hd, bs, qh = 8, 128, 64, 16
    pages = sum(-(-n // bs) for n in lens)
    g = torch.Generator(device="cuda").manual_seed(97)
    pools = [torch.randint(-127, 128, (pages, kv, bs, 128), generator=g, device=cuda,
                           dtype=torch.int8) for _ in range(2)]
    scales = [torch.rand(pages, kv, generator=g, device=cuda) * 0.02 + 0.005 for _ in range(2)]
    layer = P.make_q8_layer(*pools, *scales, kv, hd, torch.float16)
    tables = torch.zeros(len(lens), 1000, dtype=torch.int32, device=cuda)
    perm = torch.randperm(pages, generator=g, device=cuda).int()
    at = 0
    for b, n in enumerate(lens):
        tables[b, :-(-n // bs)] = perm[at:at + -(-n // bs)]
        at += -(-n // bs)
    d_lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
    q = torch.randn(len(lens), qh, hd, generator=g, device=cuda).half()
    out = torch.full((len(lens), qh, hd), float("nan"), device=cuda)
    ws = P.q8_decode_workspace(len(lens), qh, kv, hd, max(lens))
    P.q8_decode(layer, P.make_batch(tables, d_lens), q, out, hd ** -0.5, max(lens), ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    for b, n in enumerate(lens):
        idx = tables[b, :-(-n // bs)].long()
        k, v = (p[idx].double().mul(s[idx].double()[:, :, None, None]).transpose(1, 2)
                .reshape(-1, kv, hd)[:n] for p, s in zip(pools, scales))
        qd = q[b].double().view(kv, -1, hd)
        s = torch.einsum("ghd,tgd->ght", qd, k) * hd ** -0.5
        worst = float(torch.einsum("ghd,tgd->ght", qd.abs(), k.abs()).max()) * hd ** -0.5
        want = torch.einsum("ght,tgd->ghd", torch.softmax(s, -1), v).reshape(qh, hd).cpu().numpy()
        tol = attend_tol(worst, hd, float(v.abs().max()), want, 0)
        assert np.all(np.abs(out[b].double().cpu().numpy() - want) <= tol), b


@pytest.mark.parametrize("hd,kv", [(128, 1), (64, 2)])
def test_pages_past_four_gib(lib, cuda, hd, kv):
    """Page offsets above 2^32 bytes: write, decode, gather, prefill, evict."""
    import torch
    bs, pages = 128, (5 << 30) // (128 * 128)
    pools = [torch.empty(pages, 1, bs, 128, dtype=torch.int8, device=cuda) for _ in range(2)]
    scales = [torch.zeros(pages, kv, device=cuda) for _ in range(2)]
    layer = P.make_q8_layer(*pools, *scales, kv, hd, torch.float16)
    ids = [pages - 1, pages - 3, pages - 2]
    tables = torch.tensor([ids], dtype=torch.int32, device=cuda)
    L = 300
    lens = torch.tensor([L], dtype=torch.int32, device=cuda)
    batch = P.make_batch(tables, lens)
    offs = torch.tensor([0, L], dtype=torch.int32, device=cuda)
    bits = [W.normal_bits(98, (L, kv * hd), "f16", stream=s) for s in (1, 2)]
    P.q8_import(layer, batch, *(to_device_bits(b, "f16", cuda) for b in bits), offs)
    host = [Q8Pool(3, kv, hd, bs) for _ in range(2)]
    for p, b in zip(host, bits):
        p.write([0, 1, 2], 0, widen(b, "f16").reshape(L, kv, hd))
    qb = W.normal_bits(99, (1, 2 * kv, hd), "f16", stream=3)
    q = to_device_bits(qb, "f16", cuda)
    out = torch.empty(1, 2 * kv, hd, device=cuda)
    ws = P.q8_decode_workspace(1, 2 * kv, kv, hd, L)
    P.q8_decode(layer, batch, q, out, hd ** -0.5, L, ws)
    pre = torch.empty(1, 2 * kv, hd, device=cuda)
    P.q8_prefill(layer, batch, q, torch.tensor([0, 1], dtype=torch.int32, device=cuda), pre,
                 hd ** -0.5, 1, L, P.q8_prefill_workspace(layer, 1, L))
    got = [torch.empty(L, kv * hd, dtype=torch.float16, device=cuda) for _ in range(2)]
    P.q8_gather(layer, batch, *got, offs)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    k, v = (p.read64([0, 1, 2], L) for p in host)
    want, _, worst = attend64(widen(qb, "f16").astype(np.float64), k, v, hd ** -0.5)
    tol = attend_tol(worst, hd, float(np.abs(v).max()), want, 0)
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= tol)
    assert np.all(np.abs(pre.double().cpu().numpy() - want) <= tol + 2.0 ** -21 * np.abs(v).max())
    for p, o in zip(host, got):
        w = p.read([0, 1, 2], L).reshape(L, -1).astype(np.float16)
        assert np.array_equal(o.cpu().numpy().view(np.uint16), w.view(np.uint16))
    mass = torch.zeros(pages, kv, bs, device=cuda)
    mass[ids[2], :, 5] = 1.0  # position 261
    kept = torch.empty(1, kv, 4, dtype=torch.int32, device=cuda)
    P.kv_evict(layer, batch, mass, 4, 2, kept, L, dst_tables=torch.tensor(
        [[pages - 9]], dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    assert kept.cpu().numpy().tolist() == [[[0, 261, 298, 299]] * kv]


def test_bad_page_and_nan_query_stay_where_they_are(lib, cuda):
    import torch
    case = Q8Case([300, 300, 300], 8, 2, 128, 16, "bf16", seed=99, device=cuda)
    q = case.d_q.clone()
    q[2, 3, 17] = float("nan")
    bad = case.d_tables.clone()
    bad[0, 4] = 1 << 30
    out = torch.full((3, 8, 128), 7.0, device=cuda)
    ws = P.q8_decode_workspace(3, 8, 2, 128, 300)
    P.q8_decode(case.layer(), P.make_batch(bad, case.d_lens), q, out, case.scale, 300, ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 1
    got = out.double().cpu().numpy()
    assert np.isnan(got[2, 3]).all() and not np.isnan(got[2, [0, 1, 2, 4, 5, 6, 7]]).any()
    case.lengths, case.tables, case.qbits = case.lengths[1:2], case.tables[1:2], case.qbits[1:2]
    check_decode(case, got[1:2], 0)
    # a length past the bound is cut there and reported
    P.q8_decode(case.layer(), P.make_batch(case.d_tables, case.d_lens), case.d_q, out, case.scale,
                128, ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 2
    case.lengths = np.array([128])
    check_decode(case, out.double().cpu().numpy()[1:2], 0)


def test_rows_outside_their_buffer_are_reported(lib, cuda):
    import torch
    case = Q8Case([40, 40], 2, 2, 128, 16, "f16", seed=100, device=cuda)
    before = case.d_kq.clone()
    rows = torch.zeros(3, 256, dtype=torch.float16, device=cuda)
    for offs in ([0, 2, 9], [-1, 1, 3]):  # past the end; before the start
        P.q8_append(case.layer(), case.batch(), rows, rows,
                    torch.tensor(offs, dtype=torch.int32, device=cuda))
        torch.cuda.synchronize()
        assert P.device_fault(0) == 3
    keep = case.d_kq.clone()
    assert not torch.equal(before, torch.zeros_like(before)) and keep.shape == before.shape


def test_refused_rows_leave_their_sequence_and_not_the_other(lib, cuda):
    """Of a call whose offsets leave the rows' buffer for one sequence, that
    sequence's pages stay bit for bit and the other's rows are written."""
    import torch
    for offs, good in (([0, 2, 9], 0), ([-1, 1, 3], 1)):
        case = Q8Case([40, 40], 2, 2, 128, 16, "f16", seed=100, device=cuda)
        bits = [W.normal_bits(101, (3, 256), "f16", stream=s) for s in (1, 2)]
        P.q8_append(case.layer(), case.batch(), *(to_device_bits(b, "f16", cuda) for b in bits),
                    torch.tensor(offs, dtype=torch.int32, device=cuda))
        torch.cuda.synchronize()
        assert P.device_fault(0) == 3 and P.device_fault(0) == 0
        a, z = offs[good], offs[good + 1]
        for pool, b in zip((case.k, case.v), bits):
            x = widen(b, "f16").reshape(3, 2, 128)
            pool.write(case.tables[good], 40 - (z - a), x[a:z])
        case.same_pages()  # every page, the refused sequence's among them


@pytest.mark.parametrize("qh,kv,hd", [(32, 8, 128), (16, 16, 64)])
def test_the_same_call_gives_the_same_bits(lib, cuda, qh, kv, hd):
    """Work units are claimed by whichever CTA is free: no sum depends on it."""
    import torch
    lens = [3000 + 311 * i for i in range(24)]  # more than 64 tiles a CTA
    bs, per = 16, [-(-n // 16) for n in lens]
    g = torch.Generator(device="cuda").manual_seed(13)
    pages, lanes = sum(per), lanes_of(kv, hd)
    pools = [torch.randint(-127, 128, (pages, lanes, bs, 128), generator=g, device=cuda,
                           dtype=torch.int8) for _ in range(2)]
    scales = [torch.rand(pages, kv, generator=g, device=cuda) * 0.02 + 0.005 for _ in range(2)]
    layer = P.make_q8_layer(*pools, *scales, kv, hd, torch.bfloat16)
    tables = torch.zeros(24, max(per), dtype=torch.int32, device=cuda)
    perm = torch.randperm(pages, generator=g, device=cuda).int()
    for b, n in enumerate(per):
        tables[b, :n] = perm[sum(per[:b]):sum(per[:b]) + n]
    d_lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
    batch = P.make_batch(tables, d_lens)
    q = torch.randn(24, qh, hd, generator=g, device=cuda).bfloat16()
    ws = P.q8_decode_workspace(24, qh, kv, hd, max(lens))
    outs = [torch.empty(24, qh, hd, device=cuda) for _ in range(12)]
    for o in outs:
        P.q8_decode(layer, batch, q, o, hd ** -0.5, max(lens), ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    assert all(torch.equal(o, outs[0]) for o in outs)

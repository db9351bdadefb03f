"""8-bit pages on the GPU: rows written, rescaled and read back bit for bit
against the header's rule, and decode attention against 64 bits, over head
layouts, page sizes, types and lengths from none to several pages."""
from __future__ import annotations

import numpy as np
import pytest

import inference_c_b200 as P
from inference_c_b200 import workloads as W
from tests.gpu_cases import to_device_bits, to_host_bits, torch_dtype
from tests.q8_cases import Q8Case, attend64, attend_tol, widen

pytestmark = pytest.mark.gpu

SHAPES = [  # kv_heads, head_dim, block_size, dtype
    (8, 128, 16, "f16"), (8, 128, 16, "bf16"), (2, 128, 32, "bf16"), (1, 128, 64, "f16"),
    (3, 128, 128, "f16"), (8, 64, 16, "f16"), (3, 64, 16, "bf16"), (1, 64, 128, "f16"),
    (4, 64, 32, "bf16"), (5, 64, 64, "f16"),
]


def _rows(seed, n, kv_heads, hd, dtype, stream, amp=None):
    x = W.normal(seed, n * kv_heads * hd, stream=stream).reshape(n, kv_heads * hd)
    if amp is not None:
        x = x * amp[:, None].astype(np.float32)
    return W.storage_bits(x, dtype)


def _append(case, new, seed, device, dtype, one_row=False, amp=None):
    """Appends new[b] rows behind every sequence's current length minus
    new[b] (the lengths already count them), on both sides."""
    import torch
    offs = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    kb, vb = (_rows(seed, int(offs[-1]), case.kv_heads, case.hd, dtype, s, amp) for s in (61, 62))
    P.q8_append(case.layer(), case.batch(), to_device_bits(kb, dtype, device),
                to_device_bits(vb, dtype, device),
                None if one_row else torch.from_numpy(offs).to(device))
    for pool, bits in ((case.k, kb), (case.v, vb)):
        x = widen(bits, dtype).reshape(-1, case.kv_heads, case.hd)
        for b, L in enumerate(case.lengths):
            pool.write(case.tables[b], int(L) - int(new[b]), x[offs[b]:offs[b + 1]])


@pytest.mark.parametrize("kv_heads,hd,bs,dtype", SHAPES)
def test_append_rescale_import_gather(lib, cuda, kv_heads, hd, bs, dtype):
    import torch
    lengths = np.array([0, 1, 2, bs - 1, bs, bs + 1, 3 * bs + 5, 150])
    case = Q8Case(lengths, kv_heads, kv_heads, hd, bs, dtype, seed=7, device=cuda)
    # the last rows again: none, one, some of a page, over a page's end, all
    new = np.minimum(lengths, np.array([0, 1, 1, 3, bs, bs + 1, bs + 2, 99]))
    amp = 1.0 + 3.0 * W.uniform(9, int(new.sum()))
    _append(case, new, 11, cuda, dtype, amp=amp)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    case.same_pages()
    # one row for every sequence that has room for it
    some = lengths > 0
    case.lengths, case.tables = lengths[some], case.tables[some]
    case.d_tables = torch.from_numpy(np.ascontiguousarray(case.tables).view(np.int32)).to(cuda)
    case.d_lens = torch.from_numpy(case.lengths.astype(np.int32)).to(cuda)
    n = len(case.lengths)
    _append(case, np.ones(n, np.int64), 13, cuda, dtype, one_row=True, amp=np.full(n, 9.0))
    torch.cuda.synchronize()
    case.same_pages()
    # gather: q * s rounded to the row type
    offs = np.concatenate([[0], np.cumsum(case.lengths)]).astype(np.int32)
    kvw = kv_heads * hd
    outs = [torch.full((int(offs[-1]), kvw), float("nan"), dtype=torch_dtype(dtype), device=cuda)
            for _ in range(2)]
    P.q8_gather(case.layer(), case.batch(), *outs, torch.from_numpy(offs).to(cuda))
    torch.cuda.synchronize()
    for pool, out in ((case.k, outs[0]), (case.v, outs[1])):
        want = np.concatenate([pool.read(case.tables[b], int(L)).reshape(-1, kvw)
                               for b, L in enumerate(case.lengths)])
        assert np.array_equal(to_host_bits(out), W.storage_bits(want, dtype))
    case.same_pages()
    assert P.device_fault(0) == 0


@pytest.mark.parametrize("batch", [1, 5, 70])
def test_offsets_that_start_behind_the_first_row(lib, cuda, batch):
    """The rows of a call may be any run of a longer buffer: append, import and
    gather with row_offsets[0] > 0 do as with the run by itself."""
    import torch
    skip, kv_heads, hd, bs, dtype = 75, 3, 64, 16, "f16"
    lengths = 20 + (np.arange(batch) * 7) % 31
    case = Q8Case(lengths, kv_heads, kv_heads, hd, bs, dtype, seed=15, device=cuda)
    offs = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    n = int(offs[-1])
    bits = [_rows(17, skip + n, kv_heads, hd, dtype, s) for s in (4, 5)]
    dev = [to_device_bits(x, dtype, cuda) for x in bits]
    d_offs = torch.from_numpy(offs + skip).to(cuda)
    x = [widen(b, dtype).reshape(-1, kv_heads, hd)[skip:] for b in bits]
    for call, tail in ((P.q8_import, 0), (P.q8_append, 1)):
        take = np.minimum(lengths, 9) if tail else lengths
        at = np.concatenate([[0], np.cumsum(take)]).astype(np.int32)
        rows = [torch.cat([d[:skip], d[skip:skip + int(at[-1])]]) for d in dev]
        call(case.layer(), case.batch(), *rows, torch.from_numpy(at + skip).to(cuda))
        for pool, r in zip((case.k, case.v), x):
            for b, L in enumerate(lengths):
                pool.write(case.tables[b], int(L - take[b]), r[at[b]:at[b + 1]])
        torch.cuda.synchronize()
        assert P.device_fault(0) == 0
        case.same_pages()
    outs = [torch.full((skip + n, kv_heads * hd), 7.0, dtype=torch.float16, device=cuda)
            for _ in range(2)]
    P.q8_gather(case.layer(), case.batch(), *outs, d_offs)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    for pool, out in zip((case.k, case.v), outs):
        want = np.concatenate([pool.read(case.tables[b], int(L)).reshape(int(L), -1)
                               for b, L in enumerate(lengths)])
        assert (out[:skip] == 7.0).all()
        assert np.array_equal(to_host_bits(out[skip:]), W.storage_bits(want, dtype))


@pytest.mark.parametrize("kv_heads,hd,bs,dtype", SHAPES[::3])
def test_import_equals_write_at_zero(lib, cuda, kv_heads, hd, bs, dtype):
    import torch
    lengths = np.array([bs, 0, 1, 5 * bs + 3, 40])
    case = Q8Case(lengths, kv_heads, kv_heads, hd, bs, dtype, seed=21, device=cuda)
    offs = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    kb, vb = (_rows(23, int(offs[-1]), kv_heads, hd, dtype, s) for s in (4, 5))
    P.q8_import(case.layer(), case.batch(), to_device_bits(kb, dtype, cuda),
                to_device_bits(vb, dtype, cuda), torch.from_numpy(offs).to(cuda))
    torch.cuda.synchronize()
    for pool, bits in ((case.k, kb), (case.v, vb)):
        x = widen(bits, dtype).reshape(-1, kv_heads, hd)
        for b in range(len(lengths)):
            pool.write(case.tables[b], 0, x[offs[b]:offs[b + 1]])
    case.same_pages()
    assert P.device_fault(0) == 0


def test_extreme_values(lib, cuda):
    """Zeros, the smallest and largest numbers, infinities and NaN."""
    import torch
    for dtype, tiny, huge in (("bf16", 1e-39, 3e38), ("f16", 6e-8, 65504.0)):
        case = Q8Case([16, 16, 16, 16, 16], 1, 1, 128, 16, dtype, seed=5, device=cuda)
        x = np.zeros((80, 128), np.float32)
        x[16:32] = tiny                       # bf16: a subnormal, its scale underflows
        x[32:48] = huge
        x[48:64] = W.normal(3, 16 * 128).reshape(16, 128)
        x[50, 3], x[51, 4], x[52, 5] = np.inf, -np.inf, np.nan
        x[64, :2] = np.inf, np.nan            # nothing finite but zeros
        bits = W.storage_bits(x, dtype)
        d = to_device_bits(bits, dtype, cuda)
        offs = torch.arange(0, 81, 16, dtype=torch.int32, device=cuda)
        P.q8_import(case.layer(), case.batch(), d, d, offs)
        torch.cuda.synchronize()
        assert P.device_fault(0) == 5 and P.device_fault(0) == 0
        y = widen(bits, dtype).reshape(80, 1, 128)
        for pool in (case.k, case.v):
            for b in range(5):
                pool.write(case.tables[b], 0, y[16 * b:16 * b + 16])
        case.same_pages()


def test_bad_pages_and_lengths_are_reported(lib, cuda):
    import torch
    case = Q8Case([20, 20], 2, 2, 64, 16, "f16", seed=3, device=cuda)
    before = case.d_kq.clone()
    bad = case.d_tables.clone()
    bad[:, 1] = case.d_kq.shape[0] + 5
    rows = torch.zeros(2, 128, dtype=torch.float16, device=cuda)
    P.q8_append(case.layer(), P.make_batch(bad, case.d_lens), rows, rows)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 1
    lens = torch.zeros(2, dtype=torch.int32, device=cuda)  # no room for a row
    P.q8_append(case.layer(), P.make_batch(case.d_tables, lens), rows, rows)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 3
    lens += 40  # past the table
    P.q8_append(case.layer(), P.make_batch(case.d_tables, lens), rows, rows)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 2
    assert torch.equal(case.d_kq, before)


def check_decode(case, got, out_eps, what=""):
    q = widen(case.qbits, case.dtype).astype(np.float64)
    for b, L in enumerate(case.lengths):
        L = int(L)
        k, v = case.k.read64(case.tables[b], L), case.v.read64(case.tables[b], L)
        want, _, worst = attend64(q[b:b + 1], k, v, case.scale)
        vmax = float(np.abs(v).max()) if L else 0.0
        tol = attend_tol(worst, case.hd, vmax, want, out_eps)
        diff = np.abs(got[b] - want[0])
        assert np.all(diff <= tol[0]), (what, b, L, float(diff.max()), float(tol.min()))


DECODE = [  # q_heads, kv_heads, head_dim, block_size, dtype, out
    (32, 8, 128, 16, "f16", "f32"), (32, 8, 128, 16, "bf16", "bf16"),
    (8, 8, 64, 16, "f16", "f32"), (8, 8, 64, 16, "f16", "f16"),
    (16, 1, 128, 64, "bf16", "f32"), (7, 1, 128, 32, "f16", "f32"),
    (15, 3, 64, 16, "bf16", "f32"), (14, 2, 64, 128, "f16", "f32"),
    (48, 3, 64, 32, "f16", "f32"), (6, 2, 128, 128, "bf16", "f32"), (1, 1, 64, 16, "bf16", "f32"),
    (24, 8, 128, 16, "f16", "f32"), (16, 2, 128, 16, "bf16", "f32"), (33, 3, 128, 16, "f16", "f32"),
]
LENGTHS = [0, 1, 2, 15, 16, 17, 127, 128, 129, 255, 257, 700, 1031]


@pytest.mark.parametrize("q_heads,kv_heads,hd,bs,dtype,out", DECODE)
def test_decode(lib, cuda, q_heads, kv_heads, hd, bs, dtype, out):
    import torch
    case = Q8Case(LENGTHS, q_heads, kv_heads, hd, bs, dtype, seed=31, device=cuda)
    od = torch.float32 if out == "f32" else torch_dtype(out)
    ws = P.q8_decode_workspace(len(LENGTHS), q_heads, kv_heads, hd, max(LENGTHS))
    for _ in range(2):  # the scratch serves the next call as it was left
        got = torch.full((len(LENGTHS), q_heads, hd), float("nan"), dtype=od, device=cuda)
        P.q8_decode(case.layer(), case.batch(), case.d_q, got, case.scale, max(LENGTHS), ws)
        torch.cuda.synchronize()
        assert P.device_fault(0) == 0
        check_decode(case, got.double().cpu().numpy(), 0 if out == "f32" else torch.finfo(od).eps)
    case.same_pages()


@pytest.mark.parametrize("q_heads,kv_heads,hd,bs,dtype,out,causal", [
    (8, 2, 128, 16, "bf16", "bf16", True), (14, 2, 64, 32, "f16", "f16", True),
    (5, 1, 128, 128, "f16", "f32", False), (9, 3, 64, 16, "bf16", "f32", True),
    (4, 4, 128, 64, "f16", "f32", True),
])
@pytest.mark.parametrize("parts", [False, True])
def test_prefill(lib, cuda, q_heads, kv_heads, hd, bs, dtype, out, causal, parts):
    """Chunks of none, one and many rows, over the exact values q * s."""
    import torch
    lengths = np.array([1, 129, 0, 300, 131, 17])
    rows = np.array([1, 129, 0, 40, 0, 5])
    case = Q8Case(lengths, q_heads, kv_heads, hd, bs, dtype, seed=51, device=cuda)
    offs = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    qbits = W.normal_bits(53, (int(offs[-1]), q_heads, hd), dtype, stream=9)
    od = torch.float32 if out == "f32" else torch_dtype(out)
    got = torch.full((int(offs[-1]), q_heads, hd), float("nan"), dtype=od, device=cuda)
    full = P.q8_prefill_workspace(case.layer(), 1 if parts else len(lengths), 300)
    full.fill_(255)  # NaN wherever nothing is written
    P.q8_prefill(case.layer(), case.batch(), to_device_bits(qbits, dtype, cuda),
                 torch.from_numpy(offs).to(cuda), got, case.scale, int(rows.max()), 300, full,
                 causal=causal)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    q = widen(qbits, dtype).astype(np.float64)
    got = got.double().cpu().numpy()
    for b, L in enumerate(lengths):
        L, n = int(L), int(rows[b])
        if n == 0:
            continue
        k, v = case.k.read64(case.tables[b], L), case.v.read64(case.tables[b], L)
        limits = L - n + 1 + np.arange(n) if causal else np.full(n, L)
        want, _, worst = attend64(q[offs[b]:offs[b + 1]], k, v, case.scale, limits)
        # the 16-bit prefill keeps weights as two 16-bit halves: bf16 2^-16,
        # fp16 2^-22 of a weight, down to fp16's smallest step 2^-25
        halves = 2.0 ** -16 if dtype == "bf16" else 2.0 ** -21
        vmax = float(np.abs(v).max())
        tol = attend_tol(worst, hd, vmax, want, 0 if out == "f32" else torch.finfo(od).eps)
        diff = np.abs(got[offs[b]:offs[b + 1]] - want)
        assert np.all(diff <= tol + halves * vmax), (b, float(diff.max()))


@pytest.mark.parametrize("dtype,amp", [("f16", 1e-3), ("f16", 2e-5), ("bf16", 1e-12)])
def test_small_values_beside_pages_of_zeros(lib, cuda, dtype, amp):
    """A page of zeros in V does not cost the other pages' weights their bits:
    the error stays in proportion to the values (bounds of test_prefill and
    test_decode with vmax the case's own)."""
    import torch
    L, n = 700, 40
    case = Q8Case([L], 4, 2, 128, 16, dtype, seed=57, device=cuda)
    for pool, a in ((case.k, 1.0), (case.v, amp)):
        x = widen(W.storage_bits(W.normal(58, L * 256) * np.float32(a), dtype), dtype)
        x = x.reshape(L, 2, 128)
        x[:32] = 0
        x[320:336, 1] = 0
        pool.write(case.tables[0], 0, x)
    case.upload()
    qbits = W.normal_bits(59, (n, 4, 128), dtype, stream=9)
    q = widen(qbits, dtype).astype(np.float64)
    got = torch.full((n, 4, 128), float("nan"), device=cuda)
    offs = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    P.q8_prefill(case.layer(), case.batch(), to_device_bits(qbits, dtype, cuda), offs, got,
                 case.scale, n, L, P.q8_prefill_workspace(case.layer(), 1, L))
    one = torch.full((1, 4, 128), float("nan"), device=cuda)
    P.q8_decode(case.layer(), case.batch(), to_device_bits(qbits[-1:], dtype, cuda), one,
                case.scale, L, P.q8_decode_workspace(1, 4, 2, 128, L))
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    k, v = case.k.read64(case.tables[0], L), case.v.read64(case.tables[0], L)
    want, _, worst = attend64(q, k, v, case.scale, L - n + 1 + np.arange(n))
    vmax = float(np.abs(v).max())
    tol = attend_tol(worst, 128, vmax, want, 0)
    assert np.all(np.abs(one.double().cpu().numpy()[0] - want[-1]) <= tol[-1])
    # A weight is kept relative to the row's largest p vs, in fp16 halves with an
    # error of 2^-25 at most, and multiplies a whole number up to 127; the sum
    # it is divided by is sum(p) / max(p vs) >= 1 / max(vs).  So L keys are off
    # by at most L 2^-25 127 max(vs) = L 2^-25 vmax.
    halves = 2.0 ** -16 if dtype == "bf16" else 2.0 ** -21 + L * 2.0 ** -25
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= tol + halves * vmax)


@pytest.mark.parametrize("hd,kv", [(128, 2), (64, 2)])
def test_decode_of_the_smallest_scales(lib, cuda, hd, kv):
    """bf16 V near 2^-100, with scales that a weight's digits divided by them
    would leave FP32: digits are cut against 2^-103 there, half a step of which
    (2^-103 / (127 2^16) / 2) times 127 for each of the keys bounds the error."""
    import torch
    L = 300
    case = Q8Case([L], 4, kv, hd, 16, "bf16", seed=57, device=cuda)
    x = W.normal(58, L * kv * hd).astype(np.float64) * 2.0 ** -100
    x = widen(W.storage_bits(x.astype(np.float32), "bf16"), "bf16").reshape(L, kv, hd)
    case.v.write(case.tables[0], 0, x)
    assert 0 < case.v.s[case.tables[0][:19]].max() < 2.0 ** -104
    case.upload()
    got = torch.full((1, 4, hd), float("nan"), device=cuda)
    P.q8_decode(case.layer(), case.batch(), case.d_q, got, case.scale, L,
                P.q8_decode_workspace(1, 4, kv, hd, L))
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    k, v = case.k.read64(case.tables[0], L), case.v.read64(case.tables[0], L)
    want, _, worst = attend64(widen(case.qbits, "bf16").astype(np.float64), k, v, case.scale)
    tol = attend_tol(worst, hd, float(np.abs(v).max()), want, 0) + L * 2.0 ** -120
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= tol)


def test_prefill_longer_than_bound_is_reported(lib, cuda):
    """Such a sequence gets no output, whatever its length says; the others do."""
    import torch
    case = Q8Case([200, 20], 4, 2, 128, 16, "f16", seed=3, device=cuda)
    offs = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)
    ws = P.q8_prefill_workspace(case.layer(), 2, 100)
    for long in (200, 101, 1 << 28):
        lens = torch.tensor([long, 20], dtype=torch.int32, device=cuda)
        out = torch.full((2, 4, 128), 7.0, device=cuda)
        P.q8_prefill(case.layer(), P.make_batch(case.d_tables, lens), case.d_q, offs, out,
                     case.scale, 1, 100, ws)
        torch.cuda.synchronize()
        assert P.device_fault(0) in (2, 3)
        assert P.device_fault(0) == 0
        assert (out[0] == 7.0).all()
        q = widen(case.qbits, "f16").astype(np.float64)
        want, _, _ = attend64(q[1:2], case.k.read64(case.tables[1], 20),
                              case.v.read64(case.tables[1], 20), case.scale)
        assert np.abs(out[1].double().cpu().numpy() - want[0]).max() < 1e-4


def test_prefill_of_more_sequences_than_a_launch(lib, cuda):
    """1,100 sequences, some of no rows: each reads its own pages' scales."""
    import torch
    r = np.random.RandomState(5)
    lengths = r.randint(0, 70, 1100)
    rows = np.minimum(lengths, r.randint(0, 4, 1100))
    case = Q8Case(lengths, 2, 1, 64, 16, "bf16", seed=61, device=cuda)
    offs = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    n = int(offs[-1])
    qbits = W.normal_bits(63, (n, 2, 64), "bf16", stream=9)
    got = torch.full((n, 2, 64), float("nan"), device=cuda)
    ws = P.q8_prefill_workspace(case.layer(), 1100, 70)
    P.q8_prefill(case.layer(), case.batch(), to_device_bits(qbits, "bf16", cuda),
                 torch.from_numpy(offs).to(cuda), got, case.scale, 3, 70, ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    q, got = widen(qbits, "bf16").astype(np.float64), got.double().cpu().numpy()
    for b in range(1100):
        L, m = int(lengths[b]), int(rows[b])
        if m == 0:
            continue
        k, v = case.k.read64(case.tables[b], L), case.v.read64(case.tables[b], L)
        want, _, worst = attend64(q[offs[b]:offs[b + 1]], k, v, case.scale, L - m + 1 + np.arange(m))
        vmax = float(np.abs(v).max())
        tol = attend_tol(worst, 64, vmax, want, 0) + 2.0 ** -16 * vmax  # as test_prefill
        assert np.all(np.abs(got[offs[b]:offs[b + 1]] - want) <= tol), b

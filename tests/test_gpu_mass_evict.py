"""Attention mass of decode steps and eviction by it, on 16-bit and 8-bit
pages: weights against 64 bits, kept positions and moved rows exactly."""
from __future__ import annotations

import numpy as np
import pytest

import inference_c_b200 as P
from inference_c_b200 import workloads as W
from tests.gpu_cases import PagedCase, to_host_bits, torch_dtype
from tests.q8_cases import Q8Case, attend64, attend_tol, widen

pytestmark = pytest.mark.gpu

LENGTHS = [0, 1, 17, 128, 129, 400, 1031]


def _mass(rng, pages, heads, bs):
    return rng.random((pages, heads, bs)).astype(np.float32) * 0.05


def _rows16(case, which, b, L):
    pool = getattr(case, which + "pool").reshape(-1, case.block_size, case.kv_heads, case.head_dim)
    t = np.arange(L)
    bits = pool[case.tables[b][t // case.block_size].astype(np.int64), t % case.block_size]
    return widen(bits, case.dtype).astype(np.float64)


def _check_mass(tables, lengths, bs, hd, rows, q, scale, before, after, out, out_eps):
    want_mass, slack = before.astype(np.float64), np.zeros(before.shape)
    for b, L in enumerate(lengths):
        L = int(L)
        if L == 0:
            assert not out[b].any()
            continue
        k, v = rows("k", b, L), rows("v", b, L)
        want, w, worst = attend64(q[b:b + 1], k, v, scale)
        vmax = float(np.abs(v).max())
        assert np.all(np.abs(out[b] - want[0]) <= attend_tol(worst, hd, vmax, want, out_eps)[0])
        Hkv = k.shape[1]
        G = q.shape[1] // Hkv
        # a weight is off by the factor of its score's error (attend_tol), the
        # sum over the group and the addition by a rounding each
        delta = (hd + 4) * 2.0 ** -24 * worst * 1.5 + 2.0 ** -21
        t = np.arange(L)
        page = tables[b][t // bs].astype(np.int64)
        for g in range(Hkv):
            add = w[0, g * G:(g + 1) * G].sum(axis=0)
            want_mass[page, g, t % bs] += add
            slack[page, g, t % bs] += add * (2 * delta + (G + 4) * 2.0 ** -24) + 2.0 ** -100
    slack += np.abs(want_mass) * 2.0 ** -23
    assert np.all(np.abs(after - want_mass) <= slack)
    same = slack <= np.abs(want_mass) * 2.0 ** -23  # cells of no position: untouched
    assert np.array_equal(after[same].view(np.uint32), before[same].view(np.uint32))


@pytest.mark.parametrize("q_heads,kv_heads,hd,bs,dtype,out", [
    (32, 8, 128, 16, "f16", "f32"), (8, 8, 64, 16, "f16", "f16"), (16, 1, 128, 64, "bf16", "f32"),
    (16, 4, 64, 32, "bf16", "bf16"), (2, 2, 128, 128, "f16", "f32"),
])
def test_paged_decode_mass(lib, cuda, q_heads, kv_heads, hd, bs, dtype, out):
    import torch
    case = PagedCase(LENGTHS, q_heads, kv_heads, hd, bs, dtype, seed=61, device=cuda)
    od = torch.float32 if out == "f32" else torch_dtype(out)
    before = _mass(np.random.default_rng(5), case.pool_pages, kv_heads, bs)
    mass = torch.from_numpy(before).to(cuda)
    got = torch.full((len(LENGTHS), q_heads, hd), float("nan"), dtype=od, device=cuda)
    ws = P.decode_mass_workspace(len(LENGTHS), q_heads, kv_heads, hd, max(LENGTHS))
    P.paged_decode_mass(case.layer(), case.batch(), case.d_q, got, case.scale, max(LENGTHS), mass,
                        ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    # the output is the plain decode's, bit for bit
    plain = torch.empty_like(got)
    ws2 = P.decode_workspace(len(LENGTHS), q_heads, hd, max(LENGTHS))
    P.paged_decode(case.layer(), case.batch(), case.d_q, plain, case.scale, max(LENGTHS), ws2)
    assert torch.equal(plain, got)
    q = widen(case.q, dtype).astype(np.float64)
    # the 16-bit kernel keeps a weight as two 16-bit halves for the output
    halves = 2.0 ** -16 if dtype == "bf16" else 2.0 ** -21
    eps = (0 if out == "f32" else torch.finfo(od).eps) + 2 * halves * 4
    _check_mass(case.tables, case.lengths, bs, hd, lambda w, b, L: _rows16(case, w, b, L), q,
                case.scale, before, mass.cpu().numpy(), got.double().cpu().numpy(), eps + 2e-5)


@pytest.mark.parametrize("q_heads,kv_heads,hd,bs,dtype,out", [
    (32, 8, 128, 16, "f16", "f32"), (7, 1, 128, 32, "bf16", "bf16"), (15, 3, 64, 16, "f16", "f32"),
    (48, 3, 64, 64, "bf16", "f32"), (16, 1, 128, 128, "f16", "f32"), (8, 8, 64, 16, "f16", "f16"),
])
def test_q8_decode_mass(lib, cuda, q_heads, kv_heads, hd, bs, dtype, out):
    import torch
    case = Q8Case(LENGTHS, q_heads, kv_heads, hd, bs, dtype, seed=63, device=cuda)
    od = torch.float32 if out == "f32" else torch_dtype(out)
    before = _mass(np.random.default_rng(6), case.k.q.shape[0], kv_heads, bs)
    mass = torch.from_numpy(before).to(cuda)
    got = torch.full((len(LENGTHS), q_heads, hd), float("nan"), dtype=od, device=cuda)
    ws = P.decode_mass_workspace(len(LENGTHS), q_heads, kv_heads, hd, max(LENGTHS))
    P.q8_decode_mass(case.layer(), case.batch(), case.d_q, got, case.scale, max(LENGTHS), mass, ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    q = widen(case.qbits, dtype).astype(np.float64)
    _check_mass(case.tables, case.lengths, bs, hd,
                lambda w, b, L: getattr(case, w).read64(case.tables[b], L), q, case.scale, before,
                mass.cpu().numpy(), got.double().cpu().numpy(),
                0 if out == "f32" else torch.finfo(od).eps)


@pytest.mark.parametrize("q_heads,kv_heads,hd", [(32, 8, 128), (4, 2, 64)])
def test_one_workspace_serves_both_decodes_in_turn(lib, cuda, q_heads, kv_heads, hd):
    """A model with 16-bit and 8-bit layers: whatever ran before in the
    workspace, each call gives the bits it gives in a fresh one."""
    import torch
    lens = [1031, 5, 700]  # segments in several pieces
    a = PagedCase(lens, q_heads, kv_heads, hd, 16, "f16", seed=64, device=cuda)
    b = Q8Case(lens, q_heads, kv_heads, hd, 16, "f16", seed=65, device=cuda)

    def run(half, ws, with_mass):
        case = a if half else b
        pages = a.pool_pages if half else b.k.q.shape[0]
        mass = torch.zeros(pages, kv_heads, 16, device=cuda)
        out = torch.full((3, q_heads, hd), float("nan"), device=cuda)
        args = (case.layer(), case.batch(), case.d_q, out, case.scale, 1031)
        if with_mass:
            (P.paged_decode_mass if half else P.q8_decode_mass)(*args, mass, ws)
        else:
            (P.paged_decode if half else P.q8_decode)(*args, ws)
        return out, mass

    def fresh():
        return P.decode_mass_workspace(3, q_heads, kv_heads, hd, 1031)

    calls = [(h, m) for h in (True, False) for m in (True, False)]
    want = {c: run(c[0], fresh(), c[1]) for c in calls}
    ws = fresh()
    for first in calls:
        for second in calls:
            for c in (first, second):
                out, mass = run(c[0], ws, c[1])
                assert torch.equal(out, want[c][0]) and torch.equal(mass, want[c][1]), (c, first)
    assert P.device_fault(0) == 0


@pytest.mark.parametrize("q8", [False, True])
def test_mass_of_one_long_sequence_adds_up(lib, cuda, q8):
    """Many pieces and the merge kernel; over three steps every head's mass
    grows by three times its query heads (weights sum to one)."""
    import torch
    L, steps = 20011, 3
    if q8:
        case = Q8Case([L], 16, 2, 128, 16, "f16", seed=65, device=cuda)
        pages, call, lens = case.k.q.shape[0], P.q8_decode_mass, [L]
    else:
        case = PagedCase([L], 16, 2, 128, 16, "f16", seed=65, device=cuda)
        pages, call = case.pool_pages, P.paged_decode_mass
    mass = torch.zeros(pages, 2, 16, device=cuda)
    ws = P.decode_mass_workspace(1, 16, 2, 128, L)
    out = torch.empty(1, 16, 128, dtype=torch.float32, device=cuda)
    for _ in range(steps):
        call(case.layer(), case.batch(), case.d_q, out, case.scale, L, mass, ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    total = mass.double().sum(dim=(0, 2)).cpu().numpy()
    # each weight is off by at most 2 delta (attend_tol with worst <= 30)
    delta = 132 * 2.0 ** -24 * 45 + 2.0 ** -21
    assert np.all(np.abs(total - steps * 8) <= steps * 8 * (2 * delta + 2.0 ** -20))
    # a length past the declared bound adds nothing and is reported
    before = mass.clone()
    call(case.layer(), case.batch(), case.d_q, out, case.scale, 1000, mass, ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 2 and torch.equal(mass, before)


@pytest.mark.parametrize("q8", [False, True])
def test_mass_past_the_bound_beside_short_sequences(lib, cuda, q8):
    """The scratch would hold the scores, the bound is broken all the same."""
    import torch
    lens = [300, 10, 10, 10]
    if q8:
        case = Q8Case(lens, 4, 2, 128, 16, "f16", seed=67, device=cuda)
        pages, call = case.k.q.shape[0], P.q8_decode_mass
    else:
        case = PagedCase(lens, 4, 2, 128, 16, "f16", seed=67, device=cuda)
        pages, call = case.pool_pages, P.paged_decode_mass
    mass = torch.zeros(pages, 2, 16, device=cuda)
    ws = P.decode_mass_workspace(4, 4, 2, 128, 300)
    out = torch.empty(4, 4, 128, dtype=torch.float32, device=cuda)
    call(case.layer(), case.batch(), case.d_q, out, case.scale, 128, mass, ws)
    torch.cuda.synchronize()
    fault = P.device_fault(0)
    t = mass.double().cpu().numpy()
    # each sequence's weights are there whole or not at all, and it is reported;
    # the 8-bit decode cuts the long one, so the others always fit
    assert fault == 2
    for b, L in enumerate(lens):
        own = t[case.tables[b][:-(-L // 16)].astype(np.int64)].sum(axis=(0, 2))
        full = np.allclose(own, 2, atol=1e-4)
        assert full or not own.any()
        assert not q8 or full == (b > 0)


def test_paged_decode_mass_refuses_other_shapes(lib, cuda):
    import torch
    case = PagedCase([40], 3, 3, 64, 16, "f16", seed=5, device=cuda)  # odd KV heads of 64
    ws = P.decode_mass_workspace(1, 3, 3, 64, 40)
    out = torch.empty(1, 3, 64, dtype=torch.float32, device=cuda)
    mass = torch.zeros(case.pool_pages, 3, 16, device=cuda)
    with pytest.raises(P.PkvError, match="even number"):
        P.paged_decode_mass(case.layer(), case.batch(), case.d_q, out, case.scale, 40, mass, ws)
    with pytest.raises(ValueError, match="mass"):
        P.paged_decode_mass(case.layer(), case.batch(), case.d_q, out, case.scale, 40,
                            mass[:, :2], ws)


# ---------------------------------------------------------------------------
# Eviction
# ---------------------------------------------------------------------------

def keep_list(mass, L, keep, recent):
    """mass [L] -> ascending kept positions."""
    m = min(L, keep)
    if L <= keep:
        return np.arange(L)
    old = L - recent
    x = mass[:old].astype(np.float64) + 0.0
    x = np.where(np.isnan(x), -np.inf, x)
    nan = np.isnan(mass[:old])
    # lowest last: NaN below everything, then by value, ties by position
    order = np.lexsort((np.arange(old), -x, nan))
    return np.sort(np.concatenate([order[:m - recent], np.arange(old, L)]))


def _evict_case(q8, lengths, kv_heads, hd, bs, dtype, seed, cuda, keep, extra=3):
    need = sum(-(-min(int(L), keep) // bs) for L in lengths)
    if q8:
        case = Q8Case(lengths, kv_heads, kv_heads, hd, bs, dtype, seed, cuda,
                      extra_pages=need + extra)
        pages = case.k.q.shape[0]
    else:
        pages = int(sum(-(-int(L) // bs) for L in lengths)) + need + extra
        case = PagedCase(lengths, kv_heads, kv_heads, hd, bs, dtype, seed, cuda, pool_pages=pages)
    return case, pages


def _run_evict(case, pages, q8, kv_heads, hd, bs, keep, recent, mass, in_place, cuda, max_len):
    import torch
    lengths = case.lengths
    n = len(lengths)
    if in_place:
        dst, d_dst = case.tables, None
    else:
        used = {int(p) for b, L in enumerate(lengths) for p in case.tables[b][:-(-int(L) // bs)]}
        free = [p for p in range(pages) if p not in used]
        width = max(1, max(-(-min(int(L), keep) // bs) for L in lengths))
        dst, at = np.zeros((n, width), np.uint32), 0
        for b, L in enumerate(lengths):
            k = -(-min(int(L), keep) // bs)
            dst[b, :k] = free[at:at + k]
            at += k
        d_dst = torch.from_numpy(dst.view(np.int32)).to(cuda)
    d_mass = torch.from_numpy(mass).to(cuda)
    kept = torch.full((n, kv_heads, keep), -7, dtype=torch.int32, device=cuda)
    P.kv_evict(case.layer(), case.batch(), d_mass, keep, recent, kept, max_len, dst_tables=d_dst)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    # ---- the same on the host ----
    want_kept = np.full((n, kv_heads, keep), -1, np.int32)
    want_mass = mass.copy()
    if q8:
        pools = [(p, p.q.copy(), p.s.copy()) for p in (case.k, case.v)]
    else:
        shape = (pages, bs, kv_heads, hd)
        old = [case.kpool.reshape(shape), case.vpool.reshape(shape)]
        new = [o.copy() for o in old]
    for b, L in enumerate(lengths):
        L = int(L)
        t = np.arange(L)
        src = case.tables[b].astype(np.int64)
        to = dst[b].astype(np.int64)
        for g in range(kv_heads):
            pick = keep_list(mass[src[t // bs], g, t % bs], L, keep, recent)
            m = len(pick)
            want_kept[b, g, :m] = pick
            i = np.arange(m)
            want_mass[to[i // bs], g, i % bs] = mass[src[pick // bs], g, pick % bs]
            if not q8:
                for o, w in zip(old, new):
                    w[to[i // bs], i % bs, g] = o[src[pick // bs], pick % bs, g]
                continue
            for pool, q, s in pools:
                lane, cols = pool._cols(g)
                for j in range(-(-m // bs)):
                    idx = pick[j * bs:(j + 1) * bs]
                    ss = pool.s[src[idx // bs], g]
                    top = ss.max()
                    x = pool.q[src[idx // bs], lane, idx % bs, cols].astype(np.float32)
                    f = (ss / top)[:, None] if top > 0 else np.float32(0)
                    q[to[j], lane, :len(idx), cols] = np.rint(x * f).astype(np.int8)
                    s[to[j], g] = top
    assert np.array_equal(kept.cpu().numpy(), want_kept)
    assert np.array_equal(d_mass.cpu().numpy().view(np.uint32), want_mass.view(np.uint32))
    if q8:
        for (pool, q, s), d_q, d_s in zip(pools, (case.d_kq, case.d_vq), (case.d_ks, case.d_vs)):
            assert np.array_equal(d_q.cpu().numpy(), q)
            assert np.array_equal(d_s.cpu().numpy().view(np.uint32), s.view(np.uint32))
    else:
        for w, d in zip(new, (case.d_kpool, case.d_vpool)):
            assert np.array_equal(to_host_bits(d).reshape(w.shape), w)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kv_heads,hd,bs,dtype,keep,recent", [
    (8, 128, 16, "f16", 100, 20), (3, 64, 16, "bf16", 64, 64), (2, 128, 64, "bf16", 130, 0),
    (5, 64, 128, "f16", 1, 0), (1, 128, 32, "f16", 300, 299), (2, 64, 32, "f16", 33, 1),
])
def test_evict(lib, cuda, q8, in_place, kv_heads, hd, bs, dtype, keep, recent):
    lengths = np.array([0, 1, keep, keep + 1, 700, 131, 1500])
    case, pages = _evict_case(q8, lengths, kv_heads, hd, bs, dtype, 71, cuda, keep)
    mass = np.random.default_rng(7).random((pages, kv_heads, bs)).astype(np.float32)
    _run_evict(case, pages, q8, kv_heads, hd, bs, keep, recent, mass, in_place, cuda, 1500)


@pytest.mark.parametrize("max_len", [4096, 9000, 100000, 200000, 1 << 20])  # 4 or 16 keys a thread, one CTA or eight, in shared memory, gathered
def test_evict_ties_and_odd_masses(lib, cuda, max_len):
    """Few distinct values (ties to the lower position), signed zeros,
    infinities and NaN, over every way a list is shared."""
    lengths = np.array([3000, 4096, 65])
    case, pages = _evict_case(False, lengths, 2, 64, 16, "f16", 73, cuda, 777)
    rng = np.random.default_rng(9)
    mass = rng.choice(np.array([0.0, -0.0, 1.0, 0.5, np.inf, -np.inf, np.nan, -3.0, 1e-42],
                               np.float32), (pages, 2, 16),
                      p=[.3, .1, .1, .2, .02, .08, .1, .05, .05])
    _run_evict(case, pages, False, 2, 64, 16, 777, 50, mass, False, cuda, max_len)


def test_evict_long_sequence_shared_list(lib, cuda):
    lengths = np.array([40000])
    case, pages = _evict_case(True, lengths, 2, 128, 16, "bf16", 75, cuda, 5000)
    mass = (np.random.default_rng(11).random((pages, 2, 16)) ** 3).astype(np.float32)
    _run_evict(case, pages, True, 2, 128, 16, 5000, 128, mass, False, cuda, 40000)


def test_evict_bad_pages_are_reported(lib, cuda):
    import torch
    case, pages = _evict_case(False, np.array([100]), 2, 128, 16, "f16", 77, cuda, 20)
    mass = torch.ones(pages, 2, 16, device=cuda)
    kept = torch.empty(1, 2, 20, dtype=torch.int32, device=cuda)
    before = case.d_kpool.clone()
    dst = torch.full((1, 2), pages + 9, dtype=torch.int32, device=cuda)
    P.kv_evict(case.layer(), case.batch(), mass, 20, 4, kept, 100, dst_tables=dst)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 1 and torch.equal(case.d_kpool, before)
    P.kv_evict(case.layer(), case.batch(), mass, 20, 4, kept, 100, dst_tables=dst[:, :1] * 0)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 2  # the result's second page has no entry


def test_evict_leaves_a_sequence_past_the_bound_alone(lib, cuda):
    import torch
    case, pages = _evict_case(False, np.array([5000, 60]), 2, 128, 16, "f16", 78, cuda, 20)
    mass = torch.rand(pages, 2, 16, device=cuda)
    kept = torch.full((2, 2, 20), 7, dtype=torch.int32, device=cuda)
    before = case.d_kpool.clone()
    P.kv_evict(case.layer(), case.batch(), mass, 20, 4, kept, 4096)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 2
    assert (kept[0] == -1).all() and (kept[1] >= 0).all()
    own = case.d_tables[0].long()
    rows = (own[:, None] * 16 + torch.arange(16, device=cuda)).reshape(-1)
    assert torch.equal(case.d_kpool[rows], before[rows])


def test_evict_refusals(lib, cuda):
    import torch
    case, pages = _evict_case(False, np.array([40]), 2, 128, 16, "f16", 79, cuda, 20)
    mass = torch.ones(pages, 2, 16, device=cuda)
    kept = torch.empty(1, 2, 20, dtype=torch.int32, device=cuda)
    with pytest.raises(P.PkvError, match="recent"):
        P.kv_evict(case.layer(), case.batch(), mass, 20, 21, kept, 40)
    with pytest.raises(P.PkvError, match="keep"):
        P.kv_evict(case.layer(), case.batch(), mass, 0, 0, kept[:, :, :0].contiguous(), 40)
    with pytest.raises(ValueError, match="kept"):
        P.kv_evict(case.layer(), case.batch(), mass, 19, 2, kept, 40)


def test_steps_then_eviction_then_steps(lib, cuda):
    """A sequence as a server runs it, on 8-bit pages: prompt imported, steps
    that append, attend and add mass, an eviction in place, more steps."""
    import torch
    kv_heads, hd, bs, q_heads, dtype = 2, 128, 16, 8, "f16"
    prompt, steps, keep = 230, 5, 96
    case = Q8Case([prompt + steps], q_heads, kv_heads, hd, bs, dtype, seed=81, device=cuda)
    host_k, host_v = case.k, case.v
    table = case.tables[0]
    mass = torch.zeros(case.k.q.shape[0], kv_heads, bs, device=cuda)
    L_max = prompt + steps
    ws = P.decode_mass_workspace(1, q_heads, kv_heads, hd, L_max)
    rows = W.normal_bits(83, (L_max + steps, kv_heads * hd), dtype, stream=5)
    qs = W.normal_bits(85, (2 * steps, 1, q_heads, hd), dtype, stream=6)
    from tests.gpu_cases import to_device_bits
    d_rows, d_q = to_device_bits(rows, dtype, cuda), to_device_bits(qs, dtype, cuda)
    x = widen(rows, dtype).reshape(-1, kv_heads, hd)
    lens = torch.tensor([prompt], dtype=torch.int32, device=cuda)
    batch = P.make_batch(case.d_tables, lens)
    offs = torch.tensor([0, prompt], dtype=torch.int32, device=cuda)
    P.q8_import(case.layer(), batch, d_rows[:prompt], d_rows[:prompt], offs)
    for pool in (host_k, host_v):
        pool.write(table, 0, x[:prompt])
    out = torch.empty(1, q_heads, hd, dtype=torch.float32, device=cuda)
    want_mass = np.zeros((kv_heads, L_max))
    L = prompt

    def step(i):
        nonlocal L
        L += 1
        lens.fill_(L)
        r = prompt + i
        P.q8_append(case.layer(), batch, d_rows[r:r + 1], d_rows[r:r + 1])
        P.q8_decode_mass(case.layer(), batch, d_q[i], out, case.scale, L_max, mass, ws)
        torch.cuda.synchronize()
        for pool in (host_k, host_v):
            pool.write(table, L - 1, x[r:r + 1])
        k, v = host_k.read64(table, L), host_v.read64(table, L)
        want, w, worst = attend64(widen(qs[i], dtype).astype(np.float64), k, v, case.scale)
        tol = attend_tol(worst, hd, float(np.abs(v).max()), want, 0)
        assert np.all(np.abs(out.double().cpu().numpy() - want) <= tol)
        want_mass[:, :L] += w[0].reshape(kv_heads, -1, L).sum(axis=1)
    for i in range(steps):
        step(i)
    case.same_pages()
    t = np.arange(L)
    pages = table[t // bs].astype(np.int64)
    m = np.stack([mass.cpu().numpy()[pages, g, t % bs] for g in range(kv_heads)])
    assert np.allclose(m, want_mass, rtol=1e-4, atol=1e-7)
    kept = torch.empty(1, kv_heads, keep, dtype=torch.int32, device=cuda)
    P.kv_evict(case.layer(), batch, mass, keep, 16, kept, L_max)
    torch.cuda.synchronize()
    got = kept.cpu().numpy()[0]
    for g in range(kv_heads):  # by the device's own mass, then moved on the host
        assert np.array_equal(got[g], keep_list(m[g], L, keep, 16))
        for pool in (host_k, host_v):
            lane, cols = pool._cols(g)
            src = table[got[g] // bs].astype(np.int64)
            q, s = pool.q[src, lane, got[g] % bs, cols].astype(np.float32), pool.s[src, g].copy()
            for j in range(keep // bs):
                sl = slice(j * bs, (j + 1) * bs)
                top = s[sl].max()
                pool.q[int(table[j]), lane, :, cols] = np.rint(q[sl] * (s[sl] / top)[:, None])
                pool.s[int(table[j]), g] = top
    case.same_pages()
    L = keep
    want_mass[:] = 0
    for i in range(steps, 2 * steps):
        step(i)
    case.same_pages()
    assert P.device_fault(0) == 0


def test_tensors_of_other_types_are_refused(lib, cuda):
    import torch
    case = Q8Case([40], 4, 2, 128, 16, "f16", seed=3, device=cuda)
    pages = case.k.q.shape[0]
    mass = torch.zeros(pages, 2, 16, device=cuda)
    kept = torch.zeros(1, 2, 8, dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="float32"):
        P.mass_clear(case.layer(), case.batch(), mass.half())
    with pytest.raises(ValueError, match="float32"):
        P.kv_evict(case.layer(), case.batch(), mass.double(), 8, 2, kept, 40)
    with pytest.raises(ValueError, match="int32"):
        P.kv_evict(case.layer(), case.batch(), mass, 8, 2, kept.long(), 40)
    with pytest.raises(ValueError, match="int32"):
        P.kv_evict(case.layer(), case.batch(), mass, 8, 2, kept, 40,
                   dst_tables=torch.zeros(1, 1, dtype=torch.int64, device=cuda))


@pytest.mark.parametrize("in_place", [True, False])
def test_keep_far_above_the_lengths(lib, cuda, in_place):
    """The list is filled to its end, the rows are those there are."""
    import torch
    case, pages = _evict_case(True, [40, 0, 300], 2, 128, 16, "f16", 87, cuda, 100000)
    mass = _mass(np.random.default_rng(7), pages, 2, 16)
    _run_evict(case, pages, True, 2, 128, 16, 100000, 3, mass, in_place, cuda, 300)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("lens,bound", [
    ([2000] + [0] * 15, 128),           # the long one's scores would fit the scratch
    ([2000, 0], 1000), ([10, 300, 10, 40, 0, 128, 129], 128),
    ([1010, 999, 1000, 1001], 1000),    # the same number of tiles as the bound
    ([50, 7], 0),
])
def test_mass_and_output_of_lengths_past_the_bound(lib, cuda, q8, lens, bound):
    """A sequence past the bound adds nothing and is reported, its output that
    of its first positions; those beside it keep theirs."""
    import torch
    q_heads, kv_heads, hd = 4, 2, 128
    make = Q8Case if q8 else PagedCase
    case = make(lens, q_heads, kv_heads, hd, 16, "f16", seed=89, device=cuda)
    pages = case.k.q.shape[0] if q8 else case.pool_pages
    before = _mass(np.random.default_rng(8), pages, kv_heads, 16)
    mass = torch.from_numpy(before).to(cuda)
    out = torch.full((len(lens), q_heads, hd), float("nan"), device=cuda)
    # the scratch of a far larger bound: what is refused is not for want of room
    ws = P.decode_mass_workspace(len(lens), q_heads, kv_heads, hd, 4096)
    (P.q8_decode_mass if q8 else P.paged_decode_mass)(
        case.layer(), case.batch(), case.d_q, out, case.scale, bound, mass, ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 2 and P.device_fault(0) == 0
    rows = (lambda w, b, L: getattr(case, w).read64(case.tables[b], L)) if q8 else \
        (lambda w, b, L: _rows16(case, w, b, L))
    q = widen(case.qbits if q8 else case.q, "f16").astype(np.float64)
    want = before.astype(np.float64)
    got = out.double().cpu().numpy()
    for b, L in enumerate(lens):
        seen = min(L, bound)
        if seen == 0:
            assert not got[b].any()
            continue
        k, v = rows("k", b, seen), rows("v", b, seen)
        o, w, worst = attend64(q[b:b + 1], k, v, case.scale)
        vmax = float(np.abs(v).max())
        tol = attend_tol(worst, hd, vmax, o, 0) + (0 if q8 else 2.0 ** -21 * vmax)
        assert np.all(np.abs(got[b] - o[0]) <= tol[0]), b
        if L > bound:
            continue
        t = np.arange(L)
        for g in range(kv_heads):
            want[case.tables[b][t // 16].astype(np.int64), g, t % 16] += \
                w[0, 2 * g:2 * g + 2].sum(axis=0)
    after = mass.cpu().numpy()
    # weights as in _check_mass (worst score error below 2^-11, sums of two)
    assert np.all(np.abs(after - want) <= (want - before) * 2.0 ** -10 + np.abs(want) * 2.0 ** -22)
    same = want == before
    assert np.array_equal(after[same].view(np.uint32), before[same].view(np.uint32))


def test_evict_from_two_threads(lib, cuda):
    """Calls of different bounds, whose select kernels take different amounts of
    shared memory, from two threads on streams of their own."""
    import ctypes
    import threading

    import torch
    kv, n = 4, 40  # more lists than SMs: one CTA a list
    cases = [_evict_case(False, np.full(n, 40), kv, 64, 16, "f16", 90 + i, cuda, 20)
             for i in range(2)]
    want, errors = [], []
    for case, pages in cases:
        kept = torch.empty(n, kv, 20, dtype=torch.int32, device=cuda)
        mass = torch.rand(pages, kv, 16, device=cuda)
        dst = torch.tensor([p for p in range(pages) if p not in set(case.tables[:, :3].ravel())]
                           [:2 * n], dtype=torch.int32, device=cuda).view(n, 2)
        want.append((kept, mass, dst))
    torch.cuda.synchronize()

    def run(i, bound):
        (case, _), (kept, mass, dst) = cases[i], want[i]
        stream, err = torch.cuda.Stream(), ctypes.create_string_buffer(256)
        layer, batch = case.layer(), case.batch()
        # the arguments once, so that the threads spend their time in the calls
        args = (ctypes.byref(layer), ctypes.byref(batch), mass.data_ptr(), 20, 4, dst.data_ptr(),
                2, kept.data_ptr(), bound, stream.cuda_stream, err, 256)
        for k in range(3000):
            if not lib.pkv_kv_evict(*args):
                errors.append(err.value.decode())
            if k % 200 == 0:
                stream.synchronize()
        stream.synchronize()
    threads = [threading.Thread(target=run, args=a)
               for a in ((0, 17000), (1, 49000), (0, 20000), (1, 48000))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert P.device_fault(0) == 0
    for (case, _), (kept, mass, _) in zip(cases, want):
        m, got = mass.cpu().numpy(), kept.cpu().numpy()
        t = np.arange(40)
        for b in range(0, n, 13):
            for g in range(kv):
                w = m[case.tables[b][t // 16].astype(np.int64), g, t % 16]
                assert np.array_equal(got[b, g], keep_list(w, 40, 20, 4))


@pytest.mark.parametrize("max_len", [3000, 5000, 100000, 200000, 1 << 20])
def test_positions_of_bad_source_pages_rank_last(lib, cuda, max_len):
    """However a list is shared (as in the test of ties), positions that cannot
    be read come after all others, masses of zero and below included."""
    import torch
    L, keep = 3000, 777
    case, pages = _evict_case(False, np.array([L]), 2, 64, 16, "f16", 73, cuda, keep)
    rng = np.random.default_rng(9)
    mass = rng.choice(np.array([0.0, -2.0, 0.5], np.float32), (pages, 2, 16), p=[.6, .2, .2])
    tables = case.d_tables.clone()
    bad = np.arange(0, L // 16 - 4, 3)  # none among the newest positions
    tables[0, torch.from_numpy(bad).to(cuda)] = 1 << 30
    used = set(case.tables[0][:-(-L // 16)].tolist())
    dst = torch.tensor([[p for p in range(pages) if p not in used][:-(-keep // 16)]],
                       dtype=torch.int32, device=cuda)
    kept = torch.empty(1, 2, keep, dtype=torch.int32, device=cuda)
    P.kv_evict(case.layer(), P.make_batch(tables, case.d_lens), torch.from_numpy(mass).to(cuda),
               keep, 20, kept, max_len, dst_tables=dst)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 1 and P.device_fault(0) == 0
    t = np.arange(L)
    got = kept.cpu().numpy()[0]
    for g in range(2):
        w = mass[case.tables[0][t // 16].astype(np.int64), g, t % 16].copy()
        w[np.isin(t // 16, bad)] = np.nan
        assert np.array_equal(got[g], keep_list(w, L, keep, 20))


def test_tensors_of_other_four_byte_types_are_refused(lib, cuda):
    import torch
    case = Q8Case([40], 4, 2, 128, 16, "f16", seed=3, device=cuda)
    pages = case.k.q.shape[0]
    mass = torch.zeros(pages, 2, 16, device=cuda)
    kept = torch.zeros(1, 2, 8, dtype=torch.int32, device=cuda)
    dst = torch.zeros(1, 1, dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="mass"):
        P.kv_evict(case.layer(), case.batch(), mass.int(), 8, 2, kept, 40)
    with pytest.raises(ValueError, match="kept"):
        P.kv_evict(case.layer(), case.batch(), mass, 8, 2, kept.float(), 40)
    for bad in (dst.float(), dst.cpu(), dst.view(-1)):
        with pytest.raises(ValueError, match="dst_tables"):
            P.kv_evict(case.layer(), case.batch(), mass, 8, 2, kept, 40, dst_tables=bad)
    for d in (dst + pages - 1, (dst + pages - 1).view(torch.uint32)):
        P.kv_evict(case.layer(), case.batch(), mass, 8, 2, kept, 40, dst_tables=d)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("lens,q_heads,kv_heads,hd,bs", [
    # segments cut over CTAs, merged in the 16-bit decode kernel itself
    ([300 + 97 * i for i in range(24)], 32, 8, 128, 16),
    ([1 + 143 * i for i in range(20)], 128, 8, 128, 32),
    ([40 + 211 * i for i in range(16)], 24, 12, 64, 16),
    # above 64 tiles a CTA: units of the dynamic tail as well
    ([3000 + 311 * i for i in range(24)], 32, 8, 128, 64),
    ([2900 + 401 * i for i in range(20)], 24, 24, 64, 128),
    # more sequences than a launch holds: the scratch serves the next launch
    ([(7 * i) % 300 for i in range(1100)], 4, 2, 128, 16),
    # few segments: the merge kernel
    ([9000, 0, 17], 8, 2, 128, 16),
])
def test_mass_of_every_way_to_merge(lib, cuda, q8, lens, q_heads, kv_heads, hd, bs):
    """Weights and outputs against 64 bits on the GPU."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(11)
    per = [-(-n // bs) for n in lens]
    pages = sum(per) + 2
    tables = torch.zeros(len(lens), max(per), dtype=torch.int32, device=cuda)
    perm = torch.randperm(pages, generator=g, device=cuda).int()
    at = 0
    for b, n in enumerate(per):
        tables[b, :n] = perm[at:at + n]
        at += n
    half = torch.float16
    if q8:
        lanes = P.q8_lanes(kv_heads, hd)
        pools = [torch.randint(-127, 128, (pages, lanes, bs, 128), generator=g, device=cuda,
                               dtype=torch.int8) for _ in range(2)]
        scales = [torch.rand(pages, kv_heads, generator=g, device=cuda) * 0.02 + 0.005
                  for _ in range(2)]
        layer = P.make_q8_layer(*pools, *scales, kv_heads, hd, half)

        def rows(i, idx):  # [pages, bs, kv_heads, hd]
            x = pools[i][idx].transpose(1, 2).reshape(len(idx), bs, -1)[..., :kv_heads * hd]
            return x.reshape(len(idx), bs, kv_heads, hd).double() * scales[i][idx].double()[:, None, :, None]
    else:
        pools = [torch.randn(pages * bs, kv_heads * hd, generator=g, device=cuda, dtype=half)
                 for _ in range(2)]
        layer = P.make_layer(*pools, bs, kv_heads, hd)

        def rows(i, idx):
            return pools[i].view(pages, bs, kv_heads, hd)[idx].double()
    q = torch.randn(len(lens), q_heads, hd, generator=g, device=cuda, dtype=half)
    before = torch.rand(pages, kv_heads, bs, generator=g, device=cuda) * 0.05
    mass, out = before.clone(), torch.full((len(lens), q_heads, hd), float("nan"), device=cuda)
    d_lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
    batch = P.make_batch(tables, d_lens)
    ws = P.decode_mass_workspace(len(lens), q_heads, kv_heads, hd, max(lens))
    call = P.q8_decode_mass if q8 else P.paged_decode_mass
    call(layer, batch, q, out, hd ** -0.5, max(lens), mass, ws)
    plain = torch.empty_like(out)
    if q8:
        P.q8_decode(layer, batch, q, plain, hd ** -0.5, max(lens), ws)
    else:
        P.paged_decode(layer, batch, q, plain, hd ** -0.5, max(lens), ws)
    torch.cuda.synchronize()
    assert P.device_fault(0) == 0
    assert torch.equal(plain, out)
    want, slack = before.double(), torch.zeros_like(before).double()
    group = q_heads // kv_heads
    for b, n in enumerate(lens):
        if n == 0:
            assert not out[b].any()
            continue
        idx = tables[b, :per[b]].long()
        k, v = (rows(i, idx).reshape(-1, kv_heads, hd)[:n] for i in range(2))
        qd = q[b].double().view(kv_heads, group, hd)
        s = torch.einsum("ghd,tgd->ght", qd, k) * hd ** -0.5
        worst = float(torch.einsum("ghd,tgd->ght", qd.abs(), k.abs()).max()) * hd ** -0.5
        w = torch.softmax(s, -1)
        o = torch.einsum("ght,tgd->ghd", w, v).reshape(q_heads, hd)
        vmax = float(v.abs().max())
        # the 16-bit kernel keeps a weight as two fp16 halves
        tol = attend_tol(worst, hd, vmax, o.cpu().numpy(), 0) + (0 if q8 else 2.0 ** -21 * vmax)
        assert np.all(np.abs((out[b].double() - o).cpu().numpy()) <= tol), b
        # as in _check_mass
        delta = (hd + 4) * 2.0 ** -24 * worst * 1.5 + 2.0 ** -21
        pad = torch.zeros(kv_heads, per[b] * bs, dtype=torch.float64, device=cuda)
        pad[:, :n] = w.sum(dim=1)
        add = pad.view(kv_heads, per[b], bs).transpose(0, 1)
        want[idx] += add
        slack[idx] += add * (2 * delta + (group + 4) * 2.0 ** -24)
    slack += want.abs() * 2.0 ** -23 + 2.0 ** -100
    assert bool(((mass.double() - want).abs() <= slack).all())
    untouched = want == before.double()
    assert torch.equal(mass[untouched], before[untouched])

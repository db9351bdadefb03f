"""Steps of an 8-bit pool that are rolled back: the committed rows stay as they
were, bytes and scales."""
from __future__ import annotations

import numpy as np
import pytest

import inference_c_b200 as P
from inference_c_b200 import workloads as W
from tests.gpu_cases import to_device_bits, to_host_bits, torch_dtype
from tests.q8_cases import Q8Pool, widen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,hd,bs,dtype", [
    (2, 128, 16, "f16"), (3, 64, 32, "bf16"), (8, 128, 128, "f16"), (1, 64, 64, "bf16"),
])
def test_rolled_back_steps_leave_committed_rows(lib, cuda, kv, hd, bs, dtype):
    """Rows a hundred times larger than those before them, rolled back, then
    other rows committed: pages equal those of a pool that never saw the first,
    in every layer, for open pages, full ones, none, and a sequence that got
    nothing in the step."""
    import torch
    layers, n = 3, 5
    lens = [bs + 5, 2 * bs, 0, 3 * bs - 1, 7]
    cache = P.PagedKVCache(bs, 64, n)
    code = P.PKV_DTYPE_F16 if dtype == "f16" else P.PKV_DTYPE_BF16
    pool = P.PagedPool.q8(cache, 0, code, layers, kv, hd, n, 12)
    seqs = [cache.sequence_create() for _ in range(n)]
    host = [[Q8Pool(64, kv, hd, bs) for _ in range(2)] for _ in range(layers)]
    now = [0] * n

    def step(new, seed, amp, commit, order=None):
        order = list(range(n)) if order is None else order
        ids, new = [seqs[i] for i in order], [new[i] for i in order]
        pool.step_begin(ids, new)
        batch, offs = pool.step_batch(), np.concatenate([[0], np.cumsum(new)])
        tables = [cache.block_table(s) for s in ids]
        for l in range(layers if sum(new) else 0):
            bits = [W.storage_bits(W.normal(seed + l, sum(new) * kv * hd, stream=s) *
                                   np.float32(amp), dtype) for s in (1, 2)]
            P.q8_append(pool.q8_layer(l), batch,
                        *(to_device_bits(b, dtype, cuda).view(-1, kv * hd) for b in bits),
                        pool.step_row_offsets())
            if commit:
                for p, b in zip(host[l], bits):
                    x = widen(b, dtype).reshape(-1, kv, hd)
                    for i, s in enumerate(order):
                        p.write(tables[i], now[s], x[offs[i]:offs[i + 1]])
        pool.step_end(commit)
        if commit:
            for i, s in enumerate(order):
                now[s] += new[i]
        assert [cache.length(s) for s in seqs] == now

    def check():
        pool.step_begin(seqs, [0] * n)
        total = sum(now)
        offs = torch.tensor(np.concatenate([[0], np.cumsum(now)]), dtype=torch.int32, device=cuda)
        tables = [cache.block_table(s) for s in seqs]
        for l in range(layers):
            out = [torch.full((total, kv * hd), float("nan"), dtype=torch_dtype(dtype), device=cuda)
                   for _ in range(2)]
            P.q8_gather(pool.q8_layer(l), pool.step_batch(), *out, offs)
            torch.cuda.synchronize()
            for p, o in zip(host[l], out):
                want = np.concatenate([p.read(tables[b], now[b]).reshape(-1, kv * hd)
                                       for b in range(n)])
                assert np.array_equal(to_host_bits(o), W.storage_bits(want, dtype).reshape(o.shape))
        pool.step_end(True)
        assert P.device_fault(0) == 0

    step(lens, 100, 1.0, True)
    check()
    step([1, 1, 1, 1, 1], 200, 100.0, False)            # decode step
    check()
    step([3, 0, 2, bs + 3, 0], 300, 1000.0, False, [3, 0, 4, 1, 2])  # chunks, another order
    check()
    step([1, 2, 0, 1, bs], 400, 2.0, True)              # the scales grow from what they were
    check()
    step([0] * n, 500, 1.0, False)
    check()
    cache.free()


def test_rolled_back_step_on_a_side_stream(lib, cuda):
    """The restored page belongs to the step's stream."""
    import torch
    cache = P.PagedKVCache(16, 8, 1)
    pool = P.PagedPool.q8(cache, 0, P.PKV_DTYPE_F16, 1, 2, 128, 1, 4)
    seq = cache.sequence_create()
    side = torch.cuda.Stream()
    rows = [to_device_bits(W.normal_bits(s, (5, 256), "f16", stream=s), "f16", cuda) for s in (1, 2)]
    torch.cuda.synchronize()

    def step(r, commit):
        pool.step_begin([seq], [len(r)], stream=side)
        P.q8_append(pool.q8_layer(0), pool.step_batch(), r, r, pool.step_row_offsets(), stream=side)
        pool.step_end(commit)

    def read():
        pool.step_begin([seq], [0], stream=side)
        out = torch.empty(2, 5, 256, dtype=torch.float16, device=cuda)
        P.q8_gather(pool.q8_layer(0), pool.step_batch(), out[0], out[1],
                    torch.tensor([0, 5], dtype=torch.int32, device=cuda), stream=side)
        pool.step_end(True)
        side.synchronize()
        return out

    step(rows[0], True)
    before = read()
    big = rows[1] * 50
    torch.cuda.synchronize()
    for _ in range(10):
        step(big, False)
    assert torch.equal(read(), before)
    assert P.device_fault(0) == 0
    cache.free()

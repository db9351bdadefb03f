"""Plain forms of the 8-bit page operators for the tests: the quantisation
rule in the FP32 steps the header states (so bytes and scales compare bit for
bit), attention and weights in 64 bits."""
from __future__ import annotations

import numpy as np

from inference_c_b200 import workloads as W

F = np.float32
MIN_SCALE = F(2.0 ** -126)


def lanes_of(kv_heads: int, head_dim: int) -> int:
    return -(-kv_heads * head_dim // 128)


def widen(bits: np.ndarray, dtype: str) -> np.ndarray:
    """16-bit storage bits -> float32 (exact)."""
    return bits.view(np.float16).astype(F) if dtype == "f16" else W.bf16_bits_to_f32(bits)


class Q8Pool:
    """Host pages of one of K or V: q [pages, lanes, block, 128], s [pages, kv_heads]."""

    def __init__(self, pages, kv_heads, head_dim, block_size):
        self.kv_heads, self.hd, self.bs = kv_heads, head_dim, block_size
        self.q = np.zeros((pages, lanes_of(kv_heads, head_dim), block_size, 128), np.int8)
        self.s = np.zeros((pages, kv_heads), F)

    def _cols(self, h):
        c = h * self.hd
        return c // 128, slice(c % 128, c % 128 + self.hd)

    def write(self, table, first, rows):
        """rows [n, kv_heads, hd] float32 become positions first .. first+n-1."""
        n = rows.shape[0]
        for page in range(first // self.bs, -(-(first + n) // self.bs)) if n else []:
            p = int(table[page])
            a, z = max(first, page * self.bs), min(first + n, (page + 1) * self.bs)
            held = a - page * self.bs if page * self.bs < first else 0
            for h in range(self.kv_heads):
                lane, cols = self._cols(h)
                x = rows[a - first:z - first, h]
                fine = np.abs(x[np.isfinite(x)])
                top = fine.max() if fine.size else F(0)
                s_old = self.s[p, h] if held else F(0)
                s = max(s_old, F(top) / F(127))
                if s < MIN_SCALE:
                    s = F(0)
                inv = F(1) / s if s > 0 else F(0)
                with np.errstate(invalid="ignore"):
                    y = np.where(np.isinf(x), np.copysign(F(127), x), x * inv)
                y = np.clip(np.nan_to_num(np.rint(y.astype(F)), nan=0.0), -127, 127)
                at = a - page * self.bs
                if held and s > s_old:
                    old = self.q[p, lane, :held, cols].astype(F)
                    self.q[p, lane, :held, cols] = np.rint(old * (s_old / s)).astype(np.int8)
                self.q[p, lane, at:at + len(x), cols] = y.astype(np.int8)
                self.s[p, h] = s

    def read(self, table, L):
        """Values of positions 0 .. L-1 as float32 products: [L, kv_heads, hd]."""
        out = np.zeros((L, self.kv_heads, self.hd), F)
        t = np.arange(L)
        page = np.asarray(table, np.int64)[t // self.bs]
        for h in range(self.kv_heads):
            lane, cols = self._cols(h)
            out[:, h] = self.q[page, lane, t % self.bs, cols].astype(F) * self.s[page, h][:, None]
        return out

    def read64(self, table, L):
        out = np.zeros((L, self.kv_heads, self.hd))
        t = np.arange(L)
        page = np.asarray(table, np.int64)[t // self.bs]
        for h in range(self.kv_heads):
            lane, cols = self._cols(h)
            out[:, h] = (self.q[page, lane, t % self.bs, cols].astype(np.float64) *
                         self.s[page, h].astype(np.float64)[:, None])
        return out


class Q8Case:
    """A seeded batch over 8-bit pages, on the host and on the device."""

    def __init__(self, lengths, q_heads, kv_heads, head_dim, block_size, dtype, seed, device,
                 extra_pages=3, garbage=True):
        import torch
        self.lengths = np.asarray(lengths, np.int64)
        self.q_heads, self.kv_heads, self.hd = q_heads, kv_heads, head_dim
        self.bs, self.dtype, self.device = block_size, dtype, device
        pages = int(sum(-(-int(L) // block_size) for L in self.lengths)) + extra_pages
        self.tables, _ = W.shuffled_tables(self.lengths, block_size, pages, seed)
        self.k, self.v = (Q8Pool(pages, kv_heads, head_dim, block_size) for _ in range(2))
        for i, pool in enumerate((self.k, self.v)):
            if garbage:  # what no sequence owns may hold anything
                r = np.random.RandomState(seed + i)
                pool.q[...] = r.randint(-128, 128, pool.q.shape)
                pool.s[...] = r.choice([np.nan, np.inf, 1e30, -1.0], pool.s.shape)
            for b, L in enumerate(self.lengths):
                x = W.normal(seed, int(L) * kv_heads * head_dim, stream=40 + 2 * b + i)
                pool.write(self.tables[b], 0, x.reshape(int(L), kv_heads, head_dim))
        self.qbits = W.normal_bits(seed, (len(self.lengths), q_heads, head_dim), dtype, stream=3)
        self.upload()

    @property
    def scale(self):
        return float(1.0 / np.sqrt(self.hd))

    def upload(self):
        import torch
        from tests.gpu_cases import to_device_bits

        def up(a):
            return torch.from_numpy(np.ascontiguousarray(a)).to(self.device)
        self.d_kq, self.d_vq, self.d_ks, self.d_vs = (up(a) for a in (self.k.q, self.v.q, self.k.s,
                                                                      self.v.s))
        self.d_tables = up(self.tables.view(np.int32))
        self.d_lens = up(self.lengths.astype(np.int32))
        self.d_q = to_device_bits(self.qbits, self.dtype, self.device)

    def layer(self):
        from inference_c_b200 import make_q8_layer
        from tests.gpu_cases import torch_dtype
        return make_q8_layer(self.d_kq, self.d_vq, self.d_ks, self.d_vs, self.kv_heads, self.hd,
                             torch_dtype(self.dtype))

    def batch(self):
        from inference_c_b200 import make_batch
        return make_batch(self.d_tables, self.d_lens)

    def same_pages(self):
        """Bytes and scales on the device equal the host's, bit for bit."""
        for d, h in ((self.d_kq, self.k.q), (self.d_vq, self.v.q)):
            assert np.array_equal(d.cpu().numpy(), h)
        for d, h in ((self.d_ks, self.k.s), (self.d_vs, self.v.s)):
            assert np.array_equal(d.cpu().numpy().view(np.uint32), h.view(np.uint32))


def attend64(q, k, v, scale, limits=None):
    """q [R, Hq, d], k/v [L, Hkv, d] in 64 bits; row r sees keys below
    limits[r].  Returns (out [R, Hq, d], weights [R, Hq, L], worst) where worst
    is the largest sum of |q_i k_i| * scale of a score."""
    R, Hq, d = q.shape
    L, Hkv = k.shape[:2]
    out = np.zeros((R, Hq, d))
    w = np.zeros((R, Hq, L))
    worst = 0.0
    if L == 0:
        return out, w, worst
    limits = np.full(R, L) if limits is None else limits
    seen = np.arange(L)[None] < np.asarray(limits)[:, None]
    for h in range(Hq):
        g = h * Hkv // Hq
        s = q[:, h] @ k[:, g].T * scale
        worst = max(worst, float((np.abs(q[:, h]) @ np.abs(k[:, g]).T).max()) * abs(scale))
        s = np.where(seen, s, -np.inf)
        m = s.max(axis=1, keepdims=True)
        e = np.exp(s - np.where(np.isfinite(m), m, 0))
        l = e.sum(axis=1, keepdims=True)
        w[:, h] = e / np.where(l > 0, l, 1)
        out[:, h] = w[:, h] @ v[:, g]
    return out, w, worst


def attend_tol(worst, d, vmax, want, out_eps):
    """How far a kernel's output may be off.  A score is a sum of d products
    kept in 32 bits: off by at most d 2^-24 sum|q_i k_i| scale, plus its scaling
    and the subtraction of the maximum (two roundings of up to 2 worst) and
    exp (2^-21 relative): delta.  Weights off by a factor 1 +- delta move a
    weighted mean of values up to vmax by at most 2 delta vmax; the sum over
    the keys, kept in 32 bits and merged in pieces, is off by at most 64
    roundings of vmax.  Then one rounding to the output's type."""
    delta = (d + 4) * 2.0 ** -24 * worst * 1.5 + 2.0 ** -21
    return 2 * delta * vmax + 64 * 2.0 ** -24 * vmax + out_eps / 2 * np.abs(want)

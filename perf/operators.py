"""The cases on which the 8-bit cache and the eviction operators are measured.

Each case is one call a serving loop makes: rows written into 8-bit pages and
read back, one decode step, a prompt's chunk, a decode step that also adds up
attention weights, an eviction.  ``run`` computes it with elementary torch
operations in 32 bits, or (``own``) through this repository's entry points.

Layouts: 8-bit pages are int8 [pages][lanes][block][128] (a lane is 128
columns of a token's row) with one float32 scale per page and KV head; 16-bit
pages are [pages * block][kv_heads * head_dim]; weights are float32
[pages][kv_heads][block].
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One token of one chat appended in the middle of a page (the page's
        # earlier tokens may have to be rescaled): latency counts.
        dict(name="write one token", op="write", batch=1, q_heads=8, kv_heads=8, head_dim=64, block=16,
             dtype="f16", out="f16", lo=500, hi=500, rows_lo=1, rows_hi=1, empty=False, lens=1),
        # Chunks of a long prompt for a batch, at unaligned positions.
        dict(name="write chunks", op="write", batch=8, q_heads=32, kv_heads=8, head_dim=128, block=16,
             dtype="bf16", out="bf16", lo=700, hi=9000, rows_lo=1500, rows_hi=2048, empty=False, lens=2),
        # One short chat on a small model.
        dict(name="decode 1 x 512", op="decode", batch=1, q_heads=8, kv_heads=8, head_dim=64, block=16,
             dtype="f16", out="f32", lo=512, hi=512, empty=False, lens=3),
        # A server's ordinary batch.
        dict(name="decode 32 x 1k-4k", op="decode", batch=32, q_heads=32, kv_heads=8, head_dim=128, block=16,
             dtype="f16", out="f16", lo=1024, hi=4096, empty=False, lens=4),
        # A full server: many sequences, lengths far apart.
        dict(name="decode 64 x 512-32k", op="decode", batch=64, q_heads=32, kv_heads=8, head_dim=128, block=16,
             dtype="bf16", out="bf16", lo=512, hi=32768, empty=False, lens=5),
        # One very long document.
        dict(name="decode 1 x 131072", op="decode", batch=1, q_heads=64, kv_heads=8, head_dim=128, block=16,
             dtype="f16", out="f32", lo=131072, hi=131072, empty=False, lens=6),
        # A short follow-up question: few rows over a short past, odd sizes.
        dict(name="prefill 3 x 33", op="prefill", batch=3, q_heads=14, kv_heads=2, head_dim=64, block=32,
             dtype="f16", out="f16", lo=100, hi=300, rows_lo=17, rows_hi=33, empty=False, lens=7),
        # Chunked prefill of long prompts.
        dict(name="prefill 8 x 2048 past 8k", op="prefill", batch=8, q_heads=32, kv_heads=8, head_dim=128, block=16,
             dtype="bf16", out="bf16", lo=8192, hi=8192, rows_lo=2048, rows_hi=2048, empty=False, lens=8),
        # The ordinary batch on 16-bit pages, gathering weights for eviction.
        dict(name="weights 32 x 1k-4k", op="weights", batch=32, q_heads=32, kv_heads=8, head_dim=128, block=16,
             dtype="f16", out="f16", lo=1024, hi=4096, empty=False, lens=9, q8=False),
        # The long document on 8-bit pages, gathering weights.
        dict(name="weights 1 x 131072 8-bit", op="weights", batch=1, q_heads=64, kv_heads=8, head_dim=128, block=16,
             dtype="bf16", out="bf16", lo=131072, hi=131072, empty=False, lens=10, q8=True),
        # The ordinary batch cut down to 1024 tokens a sequence.
        dict(name="evict 32 x 1k-4k", op="evict", batch=32, q_heads=32, kv_heads=8, head_dim=128, block=16,
             dtype="f16", out="f16", lo=1024, hi=4096, keep=1024, recent=256, empty=False, lens=11, q8=False),
        # The long document cut down to an eighth, 8-bit pages.
        dict(name="evict 1 x 131072 8-bit", op="evict", batch=1, q_heads=64, kv_heads=8, head_dim=128, block=16,
             dtype="bf16", out="bf16", lo=131072, hi=131072, keep=16384, recent=1024, empty=False, lens=12, q8=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "decode", "decode", "prefill", "weights", "evict"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    head_dim = rng.choice([64, 128])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    q8 = rng.random() < 0.5
    if not q8 and op == "weights":
        # 16-bit pages: the shapes of the paged decode on the tensor cores
        group = rng.choice([1, 2, 4, 8])
        kv_heads = rng.choice([2, 4, 8])
    dtype = rng.choice(["f16", "bf16"])
    tokens = _log_int(rng, 64, 262144)  # of the whole batch
    batch = min(_log_int(rng, 1, 64), max(1, tokens // 4))
    mean = max(2, tokens // batch)
    lo = max(1, int(mean * rng.uniform(0.3, 1.0)))
    hi = max(lo, min(131072, int(mean * rng.uniform(1.0, 2.0))))
    c = dict(op=op, batch=batch, q_heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
             block=rng.choice([16, 16, 32, 64, 128]), dtype=dtype,
             out=rng.choice([dtype, "f32"]) if op in ("decode", "weights") else dtype,
             lo=lo, hi=hi, empty=rng.random() < 0.3 and batch > 1, lens=rng.randrange(1 << 30))
    if op in ("write", "prefill"):
        rows = _log_int(rng, 1, 4096 if op == "write" else 1024)
        if op == "prefill":
            c["lo"], c["hi"] = min(c["lo"], 8192), min(c["hi"], 8192)
            c["batch"] = min(c["batch"], 8)
            c["empty"] = c["empty"] and c["batch"] > 1
        rows = max(1, min(rows, 16384 // c["batch"]))
        c["rows_lo"], c["rows_hi"] = max(1, rows // 2), rows
    if op in ("weights", "evict"):
        c["q8"] = q8
    if op == "evict":
        c["keep"] = _log_int(rng, 1, max(2, int(hi * 0.75)))
        c["recent"] = int(c["keep"] * rng.choice([0.0, 0.25, 0.5, 1.0]))
    return c


# ---------------------------------------------------------------------------
# Shapes
# ---------------------------------------------------------------------------

def _lengths(c):
    """(length after the call, new rows) of each sequence, by the case alone."""
    r = np.random.RandomState(c["lens"])
    n = c["batch"]
    past = np.exp(r.uniform(math.log(c["lo"]), math.log(c["hi"] + 0.999), n)).astype(np.int64)
    past = np.clip(past, c["lo"], c["hi"])
    rows = r.randint(c["rows_lo"], c["rows_hi"] + 1, n) if "rows_lo" in c else np.zeros(n, np.int64)
    if c["empty"]:
        past[n // 2], rows[n // 2] = 0, 0
    return past + rows, rows


def _lanes(c):
    return -(-c["kv_heads"] * c["head_dim"] // 128)


def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def _is_q8(c):
    return c["op"] in ("write", "decode", "prefill") or c.get("q8", False)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _quantised(c, pages, g):
    """Pages of N(0, 1) rows in 8 bits, and their scales."""
    bs, hd = c["block"], c["head_dim"]
    heads = _lanes(c) * 128 // hd
    x = torch.randn(pages, heads, bs, hd, generator=g, device="cuda", dtype=torch.float32)
    s = x.abs().amax(dim=(2, 3)) / 127.0
    q = torch.round(x / s[:, :, None, None]).to(torch.int8)
    q = q.view(pages, _lanes(c), heads // _lanes(c), bs, hd).transpose(2, 3)
    return q.reshape(pages, _lanes(c), bs, 128), s[:, :c["kv_heads"]].contiguous()


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + c["lens"] % 7919)
    lens, rows = _lengths(c)
    bs, kvw = c["block"], c["kv_heads"] * c["head_dim"]
    dt = DTYPES[c["dtype"]]
    per = -(-lens // bs)
    width = max(1, int(per.max()))
    kept = np.minimum(lens, c["keep"]) if c["op"] == "evict" else None
    per2 = -(-kept // bs) if kept is not None else np.zeros(1, np.int64)
    width2 = max(1, int(per2.max()))
    need, need2 = int(per.sum()), int(per2.sum())
    pages = need + need2 + 8
    perm = torch.randperm(pages, generator=g, device=dev)

    def table(counts, w, at):
        t = torch.zeros(len(counts), w, dtype=torch.int64, device=dev)
        m = torch.arange(w, device=dev)[None, :] < torch.from_numpy(counts).to(dev)[:, None]
        t[m] = perm[at:at + int(counts.sum())]
        return t.to(torch.int32)

    st = {"case": c, "tables": table(per, width, 0), "scale": 1.0 / math.sqrt(c["head_dim"]),
          "lens": torch.from_numpy(lens.astype(np.int32)).to(dev), "max_len": int(lens.max()),
          "offsets": torch.from_numpy(_offsets(lens)).to(dev), "tokens": int(lens.sum())}
    if _is_q8(c):
        st["kq"], st["ks"] = _quantised(c, pages, g)
        st["vq"], st["vs"] = _quantised(c, pages, g)
    else:
        st["k"] = _normal((pages * bs, kvw), g, dt)
        st["v"] = _normal((pages * bs, kvw), g, dt)
    if "rows_lo" in c:
        st["row_offsets"] = torch.from_numpy(_offsets(rows)).to(dev)
        st["max_rows"] = int(rows.max())
    total_rows = int(rows.sum())
    if c["op"] == "write":
        # some rows larger than their page's earlier tokens, as outlier tokens are
        amp = 1.0 + torch.rand(total_rows, 1, generator=g, device=dev)
        st["k_rows"] = (_normal((total_rows, kvw), g, torch.float32) * amp).to(dt)
        st["v_rows"] = _normal((total_rows, kvw), g, dt)
        st["k_out"] = torch.empty(st["tokens"], kvw, dtype=dt, device=dev)
        st["v_out"] = torch.empty_like(st["k_out"])
    if c["op"] in ("decode", "weights", "prefill"):
        n = total_rows if c["op"] == "prefill" else c["batch"]
        st["q"] = _normal((n, c["q_heads"], c["head_dim"]), g, dt)
        st["out"] = torch.empty(n, c["q_heads"], c["head_dim"], dtype=DTYPES[c["out"]], device=dev)
    if c["op"] in ("weights", "evict"):
        # about one earlier step's weights; a few tokens draw much of the attention
        u = torch.rand(pages, c["kv_heads"], bs, generator=g, device=dev)
        st["mass"] = u.clamp_min(1e-3) ** -0.75 * (c["q_heads"] / c["kv_heads"] / float(lens.mean()))
    if c["op"] == "evict":
        st["dst_tables"] = table(per2, width2, need)
        st["dst_lens"] = torch.from_numpy(kept.astype(np.int32)).to(dev)
        st["kept"] = torch.empty(c["batch"], c["kv_heads"], c["keep"], dtype=torch.int32, device=dev)
        if _is_q8(c):
            st["dst_offsets"] = torch.from_numpy(_offsets(kept)).to(dev)
            st["dst_tokens"] = int(kept.sum())
            st["k_out"] = torch.empty(st["dst_tokens"], kvw, dtype=dt, device=dev)
            st["v_out"] = torch.empty_like(st["k_out"])
    if own:
        _handles(st)
    return st


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------

def _handles(st):
    """The views of the state's buffers and the scratch a program keeps."""
    import inference_c_b200 as P
    c = st["case"]
    st["P"] = P
    if _is_q8(c):
        st["layer"] = P.make_q8_layer(st["kq"], st["vq"], st["ks"], st["vs"], c["kv_heads"], c["head_dim"],
                                      DTYPES[c["dtype"]])
    else:
        st["layer"] = P.make_layer(st["k"], st["v"], c["block"], c["kv_heads"], c["head_dim"])
    st["batch"] = P.make_batch(st["tables"], st["lens"])
    if c["op"] == "decode":
        st["ws"] = P.q8_decode_workspace(c["batch"], c["q_heads"], c["kv_heads"], c["head_dim"], st["max_len"])
    elif c["op"] == "weights":
        st["ws"] = P.decode_mass_workspace(c["batch"], c["q_heads"], c["kv_heads"], c["head_dim"], st["max_len"])
    elif c["op"] == "prefill":
        st["ws"] = P.q8_prefill_workspace(st["layer"], c["batch"], st["max_len"])
    elif c["op"] == "evict":
        st["dst_batch"] = P.make_batch(st["dst_tables"], st["dst_lens"])


def _run_own(st):
    c, P = st["case"], st["P"]
    if c["op"] == "write":
        P.q8_append(st["layer"], st["batch"], st["k_rows"], st["v_rows"], st["row_offsets"])
        P.q8_gather(st["layer"], st["batch"], st["k_out"], st["v_out"], st["offsets"])
        return [st["k_out"], st["v_out"]]
    if c["op"] == "decode":
        P.q8_decode(st["layer"], st["batch"], st["q"], st["out"], st["scale"], st["max_len"], st["ws"])
        return [st["out"]]
    if c["op"] == "prefill":
        P.q8_prefill(st["layer"], st["batch"], st["q"], st["row_offsets"], st["out"], st["scale"], st["max_rows"],
                     st["max_len"], st["ws"])
        return [st["out"]]
    if c["op"] == "weights":
        call = P.q8_decode_mass if _is_q8(c) else P.paged_decode_mass
        call(st["layer"], st["batch"], st["q"], st["out"], st["scale"], st["max_len"], st["mass"], st["ws"])
        return [st["out"], st["mass"]]
    P.kv_evict(st["layer"], st["batch"], st["mass"], c["keep"], c["recent"], st["kept"], st["max_len"],
               dst_tables=st["dst_tables"])
    if _is_q8(c):
        P.q8_gather(st["layer"], st["dst_batch"], st["k_out"], st["v_out"], st["dst_offsets"])
        return [st["kept"], st["k_out"], st["v_out"], st["mass"]]
    return [st["kept"], st["k"], st["v"], st["mass"]]


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _unpack(c, pool, pages):
    """8-bit values of pages [B, P] as [B, P, block, kv_heads, head_dim]."""
    x = pool[pages].transpose(2, 3)
    B, n, bs = x.shape[:3]
    return x.reshape(B, n, bs, -1)[..., :c["kv_heads"] * c["head_dim"]].reshape(B, n, bs, c["kv_heads"], c["head_dim"])


def _pack(c, x):
    """[N, block, kv_heads, head_dim] -> [N, block, lanes, 128] and which columns are values."""
    n, bs = x.shape[:2]
    w = c["kv_heads"] * c["head_dim"]
    y = torch.zeros(n, bs, _lanes(c) * 128, dtype=torch.int8, device=x.device)
    y[..., :w] = x.reshape(n, bs, w)
    return y.view(n, bs, _lanes(c), 128).transpose(1, 2)


def _dense(c, st, which, tables):
    """A pool's rows through a table: [B, T, kv_heads, head_dim] in 32 bits."""
    pages = tables.long()
    B, n = pages.shape
    bs = c["block"]
    if _is_q8(c):
        x = _unpack(c, st[which + "q"], pages).float() * st[which + "s"][pages][:, :, None, :, None]
    else:
        x = st[which].view(-1, bs, c["kv_heads"], c["head_dim"])[pages].float()
    return x.reshape(B, n * bs, c["kv_heads"], c["head_dim"])


def _attend(q, k, v, seen, scale):
    """q [B, R, Hq, d], k/v [B, T, Hkv, d], seen [B, R, T] -> out [B, R, Hq, d], weights [B, Hkv, G, R, T]."""
    B, R, Hq, d = q.shape
    Hkv = k.shape[2]
    qf = q.float().view(B, R, Hkv, Hq // Hkv, d).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, d)
    s = torch.matmul(qf, k.permute(0, 2, 3, 1)).mul_(scale).view(B, Hkv, Hq // Hkv, R, -1)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    p = s.sub_(torch.where(torch.isfinite(m), m, 0.0)).exp_()
    l = p.sum(dim=-1, keepdim=True)
    p = p.div_(torch.where(l > 0, l, 1.0))
    o = torch.matmul(p.view(B, Hkv, -1, p.shape[-1]), v.permute(0, 2, 1, 3))
    return o.view(B, Hkv, Hq // Hkv, R, d).permute(0, 3, 1, 2, 4).reshape(B, R, Hq, d), p


def _gather_rows(c, st, tables, lens, tokens):
    """The first lens[b] rows of each sequence, one after another, in the rows' type."""
    kvw = c["kv_heads"] * c["head_dim"]
    k, v = _dense(c, st, "k", tables), _dense(c, st, "v", tables)
    B, T = k.shape[:2]
    at = torch.arange(T, device=k.device)[None] < lens[:, None]
    dt = DTYPES[c["dtype"]]
    return k.view(B, T, kvw)[at].to(dt), v.view(B, T, kvw)[at].to(dt)


def _write_plain(c, st, q, s, rows):
    """New rows quantised into their blocks; a block's scale only grows while it fills."""
    bs, Hkv, d = c["block"], c["kv_heads"], c["head_dim"]
    pages = st["tables"].long()
    B, n = pages.shape
    off = st["row_offsets"].long()
    count = off[1:] - off[:-1]
    L = st["lens"].long()
    pos = torch.arange(n * bs, device=q.device)[None]
    first = (L - count)[:, None]
    new = (pos >= first) & (pos < L[:, None])
    r = (pos - first + off[:-1, None]).clamp(0, max(0, rows.shape[0] - 1))
    x = torch.where(new[..., None], rows[r].float(), 0.0).view(B, n, bs, Hkv, d)
    new = new.view(B, n, bs)
    touched = new.any(dim=-1)
    held = touched & (pos.view(1, n, bs)[..., 0] < first)
    s_old = torch.where(held[..., None], s[pages], 0.0)
    s_new = torch.maximum(s_old, x.abs().amax(dim=(2, 4)) / 127.0)
    s_new = torch.where(s_new < 2.0 ** -126, 0.0, s_new)
    some = torch.where(s_new > 0, s_new, 1.0)
    fresh = torch.round(x * (1.0 / some)[:, :, None, :, None]).clamp(-127, 127)
    old = _unpack(c, q, pages).float()
    again = torch.round(old * (s_old / some)[:, :, None, :, None])
    before = (pos.view(1, n, bs) < first[:, :, None])[..., None, None]
    y = torch.where(new[..., None, None], fresh, torch.where(before, again, old)).to(torch.int8)
    q[pages[touched]] = _pack(c, y[touched])
    s[pages[touched]] = s_new[touched]


def _evict_plain(c, st):
    bs, Hkv, keep, recent = c["block"], c["kv_heads"], c["keep"], c["recent"]
    pages = st["tables"].long()
    B, n = pages.shape
    T = n * bs
    L = st["lens"].long()[:, None, None]
    w = st["mass"][pages].permute(0, 2, 1, 3).reshape(B, Hkv, T)
    t = torch.arange(T, device=w.device).view(1, 1, T)
    w = torch.where(t >= L, -math.inf, torch.where(t >= L - recent, math.inf, w))
    width = min(keep, T)
    first = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :width]
    kept = torch.sort(torch.where(first < L, first, T), dim=-1).values
    i = torch.arange(width, device=w.device).view(1, 1, width)
    ok = i < L
    st["kept"].fill_(-1)
    st["kept"][..., :width] = torch.where(ok, kept, -1).to(torch.int32)
    src = torch.where(ok, kept, 0)
    # where row i of the result goes
    to = st["dst_tables"].long()
    page = to[:, (i[0, 0] // bs).clamp_max(to.shape[1] - 1)]
    b_i, r_i = (ok[:, 0]).nonzero(as_tuple=True)
    dst_page, dst_in = page[b_i, r_i], r_i % bs
    s_page = torch.gather(pages[:, None].expand(B, Hkv, n), 2, src // bs)[b_i, :, r_i]   # [N, Hkv]
    s_in = (src % bs)[b_i, :, r_i]
    heads = torch.arange(Hkv, device=w.device)[None]
    moved = st["mass"][s_page, heads, s_in]
    if not _is_q8(c):
        k = st["k"].view(-1, bs, Hkv, c["head_dim"])
        v = st["v"].view(-1, bs, Hkv, c["head_dim"])
        k[dst_page, dst_in] = k[s_page, s_in, heads]
        v[dst_page, dst_in] = v[s_page, s_in, heads]
    else:
        _move_q8(c, st["kq"], st["ks"], s_page, s_in, heads, dst_page, dst_in)
        _move_q8(c, st["vq"], st["vs"], s_page, s_in, heads, dst_page, dst_in)
    st["mass"][dst_page[:, None], heads, dst_in[:, None]] = moved


def _move_q8(c, q, s, s_page, s_in, heads, dst_page, dst_in):
    """Rows of one head each to their new blocks, at the largest scale that meets there."""
    d, lanes = c["head_dim"], _lanes(c)
    per = 128 // d
    scales = s[s_page, heads]                                            # [N, Hkv]
    x = q.view(q.shape[0], lanes, q.shape[2], per, d)[s_page, heads // per, s_in, heads % per].float()
    top = torch.zeros_like(s)
    top.scatter_reduce_(0, dst_page[:, None].expand_as(scales), scales, "amax")
    there = top[dst_page]
    y = torch.round(x * (scales / torch.where(there > 0, there, 1.0))[..., None]).to(torch.int8)
    q.view(q.shape[0], lanes, q.shape[2], per, d)[dst_page[:, None], heads // per, dst_in[:, None], heads % per] = y
    s[dst_page] = there


def run(state):
    if own:
        return _run_own(state)
    st, c = state, state["case"]
    lens = st["lens"].long()
    if c["op"] == "write":
        _write_plain(c, st, st["kq"], st["ks"], st["k_rows"])
        _write_plain(c, st, st["vq"], st["vs"], st["v_rows"])
        return list(_gather_rows(c, st, st["tables"], lens, st["tokens"]))
    if c["op"] == "evict":
        _evict_plain(c, st)
        if _is_q8(c):
            k, v = _gather_rows(c, st, st["dst_tables"], st["dst_lens"].long(), st["dst_tokens"])
            return [st["kept"], k, v, st["mass"]]
        return [st["kept"], st["k"], st["v"], st["mass"]]
    k, v = _dense(c, st, "k", st["tables"]), _dense(c, st, "v", st["tables"])
    B, T = k.shape[:2]
    t = torch.arange(T, device=k.device)
    if c["op"] == "prefill":
        off = st["row_offsets"].long()
        count = off[1:] - off[:-1]
        j = torch.arange(st["max_rows"], device=k.device)[None]
        live = j < count[:, None]
        q = st["q"][torch.where(live, off[:-1, None] + j, 0)]
        seen = t[None, None] < (lens - count)[:, None, None] + j[..., None] + 1
        o, _ = _attend(q, k, v, seen, st["scale"])
        return [o[live].to(DTYPES[c["out"]])]
    seen = (t[None] < lens[:, None])[:, None]
    o, p = _attend(st["q"][:, None], k, v, seen, st["scale"])
    out = o[:, 0].to(DTYPES[c["out"]])
    if c["op"] == "decode":
        return [out]
    bs = c["block"]
    w = p.sum(dim=2)[:, :, 0].view(B, c["kv_heads"], T // bs, bs).transpose(1, 2)     # [B, P, Hkv, bs]
    pages = st["tables"].long()
    held = (t.view(1, -1, bs)[..., 0] < lens[:, None])
    st["mass"][pages[held]] += w[held]
    return [out, st["mass"]]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c = case
    lens, rows = _lengths(c)
    tokens, n = float(lens.sum()), float(rows.sum())
    kvw = c["kv_heads"] * c["head_dim"]
    blocks = float((-(-lens // c["block"])).sum())
    held = 2 * tokens * kvw * (1 if _is_q8(c) else 2) + (8 * blocks * c["kv_heads"] if _is_q8(c) else 0) + 4 * blocks
    size = DTYPES[c["out"]].itemsize
    if c["op"] == "write":
        # rows in, their 8-bit form out; then all 8-bit rows in, 16-bit rows out
        return {"bytes": 2 * n * kvw * 3 + held + 2 * tokens * kvw * 2, "flops": 4 * n * kvw + 2 * tokens * kvw}
    if c["op"] == "evict":
        kept = float(np.minimum(lens, c["keep"]).sum())
        moved = 2 * kept * kvw * (2 if _is_q8(c) else 4) + kept * c["kv_heads"] * 12
        back = 2 * kept * kvw * 3 if _is_q8(c) else 0
        return {"bytes": 4 * tokens * c["kv_heads"] + moved + back, "flops": tokens * c["kv_heads"]}
    if c["op"] == "prefill":
        keys = float(np.sum(rows * (lens - rows) + rows * (rows + 1) / 2))
        io = n * c["q_heads"] * c["head_dim"] * (2 + size)
        return {"bytes": held + io, "flops": 4 * c["head_dim"] * c["q_heads"] * keys}
    io = c["batch"] * c["q_heads"] * c["head_dim"] * (2 + size)
    mass = 8 * tokens * c["kv_heads"] if c["op"] == "weights" else 0
    return {"bytes": held + io + mass, "flops": 4 * c["head_dim"] * c["q_heads"] * tokens}


# ---------------------------------------------------------------------------
# The same in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------

def exact(case, seed):
    c = case
    if c["batch"] > 512:
        return None
    st = prepare(case, seed)
    bs, Hkv, d, Hq = c["block"], c["kv_heads"], c["head_dim"], c["q_heads"]
    G, q8, scale = Hq // Hkv, _is_q8(c), 1.0 / math.sqrt(d)
    lens, rows = _lengths(c)
    tables = st["tables"].cpu().numpy().astype(np.int64)
    dev = st["tables"].device

    def values(which, b, L):
        """Rows 0 .. L-1 of sequence b: [Hkv, L, d]."""
        t = torch.arange(L, device=dev)
        page = torch.from_numpy(tables[b]).to(dev)[t // bs]
        out = torch.empty(Hkv, L, d, dtype=torch.float64, device=dev)
        for h in range(Hkv):
            if q8:
                col = (h * d) % 128
                x = st[which + "q"][page, h * d // 128, t % bs, col:col + d].double()
                out[h] = x * st[which + "s"][page, h].double()[:, None]
            else:
                out[h] = st[which][page * bs + t % bs, h * d:(h + 1) * d].double()
        return out

    def softmax(qrow, k, limit):
        """qrow [R, d], k [L, d], row i sees keys below limit[i]."""
        s = (qrow @ k.T) * scale
        s[torch.arange(k.shape[0], device=dev)[None] >= limit[:, None]] = -math.inf
        e = torch.exp(s - s.max(dim=1, keepdim=True).values)
        return e / e.sum(dim=1, keepdim=True)

    if c["op"] in ("decode", "weights", "prefill"):
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device=dev)
        mass = st["mass"].double() if c["op"] == "weights" else None
        at = 0
        for b in range(c["batch"]):
            L = int(lens[b])
            n = int(rows[b]) if c["op"] == "prefill" else 1
            lo, at = at, at + n
            if L == 0 or n == 0:
                continue
            k, v = values("k", b, L), values("v", b, L)
            limit = L - n + 1 + torch.arange(n, device=dev)
            for g in range(Hkv):
                sums = torch.zeros(L, dtype=torch.float64, device=dev)
                for h in range(g * G, (g + 1) * G):
                    p = softmax(st["q"][lo:at, h].double(), k[g], limit)
                    out[lo:at, h] = p @ v[g]
                    sums += p.sum(dim=0)
                if mass is not None:
                    t = torch.arange(L, device=dev)
                    mass[torch.from_numpy(tables[b]).to(dev)[t // bs], g, t % bs] += sums
        return [out] if mass is None else [out, mass]

    if c["op"] == "write":
        outs = []
        for which in ("k", "v"):
            got, at = [], 0
            for b in range(c["batch"]):
                L, n = int(lens[b]), int(rows[b])
                old = values(which, b, L)
                fresh = st[which + "_rows"][at:at + n].double().view(n, Hkv, d).transpose(0, 1)
                at += n
                res = old.clone()
                res[:, L - n:] = fresh
                for p in range((L - n) // bs, -(-L // bs)) if n else []:
                    a, z = p * bs, min(L, (p + 1) * bs)
                    start = max(a, L - n)
                    s = fresh[:, start - (L - n):z - (L - n)].abs().amax(dim=(1, 2)) / 127
                    if start > a:
                        s0 = st[which + "s"][int(tables[b, p])].double()
                        grown = torch.maximum(s, s0)
                        step = torch.round(old[:, a:start] / s0[:, None, None])  # whole steps of the old scale
                        res[:, a:start] = torch.round(step * (s0 / grown)[:, None, None]) * grown[:, None, None]
                        s = grown
                    res[:, start:z] = torch.round(res[:, start:z] / s[:, None, None]) * s[:, None, None]
                got.append(res.transpose(0, 1).reshape(L, Hkv * d))
            outs.append(torch.cat(got))
        return outs

    # evict
    mass, keep, recent = st["mass"].clone(), c["keep"], c["recent"]
    kept = torch.full((c["batch"], Hkv, keep), -1, dtype=torch.int32)
    dst = st["dst_tables"].cpu().numpy().astype(np.int64)
    new = {w: ([] if q8 else st[w].double()) for w in ("k", "v")}
    for b in range(c["batch"]):
        L = int(lens[b])
        m = min(keep, L)
        moved = {w: torch.zeros(m, Hkv, d, dtype=torch.float64, device=dev) for w in ("k", "v")}
        vals = {w: values(w, b, L) for w in ("k", "v")}
        t = np.arange(L)
        src_page = torch.from_numpy(tables[b][t // bs]).to(dev)
        i = torch.arange(m, device=dev)
        to_page = torch.from_numpy(dst[b]).to(dev)[i // bs]
        for g in range(Hkv):
            w = st["mass"][src_page, g, torch.from_numpy(t % bs).to(dev)].cpu().numpy()
            old = max(0, L - recent)
            best = np.lexsort((np.arange(old), -w[:old].astype(np.float64)))[:max(0, m - min(recent, L))]
            pick = np.sort(np.concatenate([best, np.arange(old, L)]).astype(np.int64))[:m]
            kept[b, g, :m] = torch.from_numpy(pick.astype(np.int32))
            p = torch.from_numpy(pick).to(dev)
            mass[to_page, g, i % bs] = torch.from_numpy(w).to(dev)[p]
            for n in ("k", "v"):
                x = vals[n][g][p]
                if q8 and m:
                    s = st[n + "s"][src_page[p], g].double()
                    top = torch.zeros(-(-m // bs), dtype=torch.float64, device=dev)
                    top.scatter_reduce_(0, i // bs, s, "amax")
                    top = top[i // bs][:, None]
                    x = torch.round(x / top) * top
                moved[n][:, g] = x
        for n in ("k", "v"):
            if q8:
                new[n].append(moved[n].reshape(m, Hkv * d))
            else:
                new[n][to_page * bs + i % bs] = moved[n].reshape(m, Hkv * d)
    return [kept] + [torch.cat(new[n]) if q8 else new[n] for n in ("k", "v")] + [mass.double()]

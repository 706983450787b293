"""Batched serving over a paged cache (lt_paged_append, lt_paged_attn_decode, lt_paged_attn_prompt, lt_kv_evict)
against plain 64-bit implementations.

Bars, from the arithmetic: queries, weights and f32 caches enter the products as two terms of 11 bits each (relative
error 2^-22), the sums are f32, so a score of magnitude s is off by about s * 2^-21 and a weight, relatively, by as
much plus 2^-22 of the exponential; with |s| up to about 10 that is 5e-6 at worst and less in a sum.  Attention
outputs: rel-L2 < 1e-5.  Accumulated weights: the same on what was added.  Rotations: the angle p / theta^(2i/hd) is
rounded in f32 (three roundings, p * 1.8e-7), plus 1e-6 for the norm.  Copies and choices are exact.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ATTN_BAR = 1e-5


def i32(v):
    return torch.as_tensor(np.asarray(v, dtype=np.int64).astype(np.uint32).view(np.int32)).cuda()


class Cache:
    """A pool with page tables for sequences of the given capacities; what no sequence holds is NaN."""

    def __init__(self, pkg, rng, lens, kv, hd, f16, page, layout="nhd", extra_pages=2, spare=0):
        self.lens, self.kv, self.hd, self.page, self.f16 = lens, kv, hd, page, f16
        need = [-(-n // page) for n in lens]
        self.width = max(1, max(need)) + spare
        self.n_pages = sum(need) + extra_pages
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), self.width), 0xFFFFFFFF, dtype=np.int64)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.free = order[at:]
        dt = np.float16 if f16 else np.float32
        shape = (self.n_pages, page, kv, hd) if layout == "nhd" else (self.n_pages, kv, page, hd)
        k, v = np.full(shape, np.nan, dt), np.full(shape, np.nan, dt)
        self.hk, self.hv = (x if layout == "nhd" else x.swapaxes(1, 2) for x in (k, v))  # [page][slot][head][hd] views
        for s, n in enumerate(lens):
            for j in range(n):
                p = self.table[s, j // page]
                self.hk[p, j % page] = rng.normal(0, 1, (kv, hd))
                self.hv[p, j % page] = rng.normal(0, 1, (kv, hd))
        self._k, self._v = k, v
        self.layout = layout
        self.upload(pkg)

    def upload(self, pkg):
        self.dk, self.dv, self.dtable = torch.from_numpy(self._k).cuda(), torch.from_numpy(self._v).cuda(), i32(self.table)
        p, kv, hd = self.page, self.kv, self.hd
        st = (0, 0, 0) if self.layout == "nhd" else (kv * p * hd, hd, p * hd)
        self.desc = pkg.PagedKV(n_kv_heads=kv, head_dim=hd, kv_f16=int(self.f16), page_size=p, n_pages=self.n_pages,
                                max_pages=self.width, page_stride=st[0], slot_stride=st[1], head_stride=st[2],
                                k=self.dk.data_ptr(), v=self.dv.data_ptr())

    def seq(self, s, n=None):
        """K and V [n][kv][hd] of sequence s in 64 bits."""
        n = self.lens[s] if n is None else n
        j = np.arange(n)
        p = self.table[s, j // self.page]
        return self.hk[p, j % self.page].astype(np.float64), self.hv[p, j % self.page].astype(np.float64)


def attend(q, K, V, i, seen, scale, cap=0.0, slopes=None):
    """q [m][H][hd] at positions i [m], K and V [n][kv][hd], seen [m][n] -> out [m][H][hd], weights [m][H][n]."""
    m, H, hd = q.shape
    n, kv = K.shape[:2]
    out, W = np.zeros((m, H, hd)), np.zeros((m, H, n))
    if n == 0:
        return out, W
    for h in range(H):
        s = q[:, h].astype(np.float64) @ K[:, h // (H // kv)].T * scale
        if cap:
            s = cap * np.tanh(s / cap)
        if slopes is not None:
            s = s - float(slopes[h]) * np.abs(i[:, None] - np.arange(n)[None])
        for r in range(m):
            v = seen[r]
            if v.any():
                e = np.exp(s[r, v] - s[r, v].max())
                W[r, h, v] = e / e.sum()
                out[r, h] = W[r, h, v] @ V[v, h // (H // kv)]
    return out, W


def rel(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30))


SHAPES = [(14, 2, 64), (32, 4, 128), (16, 8, 256), (4, 4, 128), (16, 1, 64), (40, 2, 128)]


# ── append ───────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (32, 4, 128), (16, 8, 256), (3, 1, 128)])
@pytest.mark.parametrize("f16,neox,v_norm,norms,page", [(True, True, False, True, 16), (False, False, True, True, 7),
                                                        (True, False, True, False, 1)])
def test_append(pkg, ctx, heads, kv, hd, f16, neox, v_norm, norms, page):
    rng = np.random.default_rng(hd + page)
    lens = [40, 1, 301]
    c = Cache(pkg, rng, lens, kv, hd, f16, page)
    tok = [(0, 39), (1, 0), (2, 300), (2, 12), (2, 13), (0, 0)]
    seq, pos = np.array([s for s, _ in tok]), np.array([p for _, p in tok])
    theta, eps = 1e5, 1e-6
    qkv = rng.normal(0, 2, (len(tok), heads + 2 * kv, hd)).astype(np.float32)
    qn, kn = (rng.normal(1, 0.2, hd).astype(np.float32) for _ in range(2))
    cfg = pkg.AttnCfg(n_heads=heads, n_kv_heads=kv, head_dim=hd, rope_neox=int(neox), rope_theta=theta, eps=eps, scale=1.0,
                      kv_cap=1, window=0, v_norm=int(v_norm), kv_f16=int(f16))
    d = [torch.from_numpy(x).cuda() for x in (qkv, qn, kn)]
    q = torch.zeros(len(tok), heads, hd, device="cuda")
    ctx.paged_append(cfg, c.desc, d[0], len(tok), d[1] if norms else None, d[2] if norms else None, i32(seq), i32(pos), None,
                     c.dtable, len(lens), q)
    ctx.sync()
    x = qkv.astype(np.float64)
    inv = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    y = x.copy()
    if norms:
        y[:, :heads] = x[:, :heads] * inv[:, :heads] * qn
        y[:, heads:heads + kv] = x[:, heads:heads + kv] * inv[:, heads:heads + kv] * kn
    if v_norm:
        y[:, heads + kv:] = x[:, heads + kv:] * inv[:, heads + kv:]
    half = hd // 2
    ang = pos[:, None] * theta ** (-2.0 * np.arange(half) / hd)
    cs, sn = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = (slice(0, half), slice(half, hd)) if neox else (slice(0, hd, 2), slice(1, hd, 2))
    z = y.copy()
    r = slice(0, heads + kv)
    z[:, r, a] = y[:, r, a] * cs - y[:, r, b] * sn
    z[:, r, b] = y[:, r, a] * sn + y[:, r, b] * cs
    bar = 1.8e-7 * 300 + 1e-6
    assert rel(q.cpu().numpy(), z[:, :heads]) < bar
    gk, gv = (t.cpu().numpy().astype(np.float64) for t in (c.dk, c.dv))
    half_ulp = 2.0 ** -11 if f16 else 0.0
    for t, (s, p) in enumerate(tok):
        page_id, inside = c.table[s, p // page], p % page
        assert rel(gk[page_id, inside], z[t, heads:heads + kv]) < bar + half_ulp
        assert rel(gv[page_id, inside], z[t, heads + kv:]) < 1e-6 + half_ulp
    # nothing else is touched
    touched = np.zeros(c._k.shape[:2], bool)
    for s, p in tok:
        touched[c.table[s, p // page], p % page] = True
    assert np.array_equal(c._k[~touched], c.dk.cpu().numpy()[~touched], equal_nan=True)


def test_append_agrees_with_one_token_prep(pkg, ctx):
    """The same rotation as lt_attn_prep at long positions, into a slot of its own."""
    rng = np.random.default_rng(5)
    heads, kv, hd, pos = 32, 4, 128, 100003
    c = Cache(pkg, rng, [20], kv, hd, False, 16)
    qkv = rng.normal(0, 2, (1, heads + 2 * kv, hd)).astype(np.float32)
    cfg = pkg.AttnCfg(n_heads=heads, n_kv_heads=kv, head_dim=hd, rope_neox=1, rope_theta=1e6, eps=1e-6, scale=1.0, kv_cap=1,
                      window=0, v_norm=0, kv_f16=0)
    w = torch.from_numpy(rng.normal(1, 0.2, hd).astype(np.float32)).cuda()
    x, q = torch.from_numpy(qkv).cuda(), torch.zeros(heads * hd, device="cuda")
    one, k1, v1 = x.clone(), torch.zeros(kv * hd, device="cuda"), torch.zeros(kv * hd, device="cuda")
    ctx.paged_append(cfg, c.desc, x, 1, w, w, i32([0]), i32([pos]), i32([17]), c.dtable, 1, q)
    ctx.attn_prep(cfg, one, w, w, i32([pos]), k1, v1)
    ctx.sync()
    assert rel(q.cpu(), one.view(-1)[:heads * hd].cpu()) < 1e-6
    page = c.table[0, 1]
    assert rel(c.dk[page, 1].cpu().reshape(-1), k1.cpu()) < 1e-6
    assert torch.equal(c.dv[page, 1].reshape(-1), v1)


def test_append_bad_index_reported(pkg, ctx):
    rng = np.random.default_rng(6)
    c = Cache(pkg, rng, [16], 2, 64, True, 16)
    cfg = pkg.AttnCfg(n_heads=2, n_kv_heads=2, head_dim=64, rope_neox=1, rope_theta=1e4, eps=1e-6, scale=1.0, kv_cap=1)
    qkv, q = torch.zeros(1, 6 * 64, device="cuda"), torch.zeros(1, 2 * 64, device="cuda")
    for seq, pos in ((0, 16), (1, 0), (0, 1 << 20)):  # past the table, no such sequence, far past
        ctx.paged_append(cfg, c.desc, qkv, 1, None, None, i32([seq]), i32([pos]), None, c.dtable, 1, q)
        with pytest.raises(pkg.LtError) as e:
            ctx.sync()
        assert e.value.status == 1
    assert np.array_equal(c.dk.cpu().numpy(), c._k, equal_nan=True)
    ctx.sync()


# ── decode ───────────────────────────────────────────────────────────────────

def run_decode(pkg, ctx, c, q, heads, cap=0.0, window=0, slopes=None, mass=None, q_pad=0):
    S, hd = len(c.lens), c.hd
    qd = torch.zeros(S, heads * hd + q_pad, device="cuda")
    qd[:, :heads * hd] = torch.from_numpy(q.reshape(S, -1)).cuda()
    out = torch.full((S, heads * hd + q_pad), 7.0, device="cuda")
    sl = None if slopes is None else torch.from_numpy(slopes).cuda()
    cfg = pkg.PagedAttnCfg(n_heads=heads, window=window, causal=1, scale=1 / math.sqrt(hd), softcap=cap,
                           slopes=None if sl is None else sl.data_ptr(), q_stride=heads * hd + q_pad,
                           out_stride=heads * hd + q_pad)
    most = max(1, max(c.lens))
    lens = i32(c.lens)
    ctx.paged_attn_decode(cfg, c.desc, qd, S, c.dtable, lens, most, out, mass, 0 if mass is None else mass.shape[-1])
    ctx.sync()
    if q_pad:
        assert (out[:, heads * hd:] == 7.0).all()
    return out[:, :heads * hd].cpu().numpy().reshape(S, heads, hd)


def check_decode(pkg, ctx, heads, kv, hd, f16, page, lens, cap=0.0, window=0, alibi=False, with_mass=False, layout="nhd",
                 q_pad=0, seed=0):
    rng = np.random.default_rng(seed)
    c = Cache(pkg, rng, lens, kv, hd, f16, page, layout)
    if window:  # what lies before every window may hold anything
        for s, n in enumerate(lens):
            for j in range(max(0, n - window)):
                c.hk[c.table[s, j // page], j % page] = np.inf if j % 2 else np.nan
                c.hv[c.table[s, j // page], j % page] = np.nan if j % 2 else -np.inf
        c.upload(pkg)
    q = (rng.normal(0, 1.5, (len(lens), heads, hd))).astype(np.float32)
    slopes = (2.0 ** (-8.0 * (np.arange(heads) + 1) / heads)).astype(np.float32) if alibi else None
    most = max(1, max(lens))
    m0 = rng.uniform(0, 1, (len(lens), kv, most + 3)).astype(np.float32)
    mass = torch.from_numpy(m0).cuda() if with_mass else None
    got = run_decode(pkg, ctx, c, q, heads, cap, window, slopes, mass, q_pad)
    want, added = np.zeros(got.shape), np.zeros(m0.shape)
    for s, n in enumerate(lens):
        K, V = c.seq(s)
        seen = np.ones((1, n), bool)
        if window:
            seen[0, :max(0, n - window)] = False
        o, W = attend(q[s][None], K, V, np.array([n - 1]), seen, 1 / math.sqrt(hd), cap, slopes)
        want[s] = o[0]
        added[s, :, :n] = W[0].reshape(kv, heads // kv, n).sum(1)
        assert n or not got[s].any()
    assert np.isfinite(got).all()
    assert rel(got, want) < ATTN_BAR
    if with_mass:
        g = mass.cpu().numpy().astype(np.float64)
        assert np.array_equal(g[added == 0], m0[added == 0])
        # the cells round to f32 when they are added to (2^-24 of at most 1 + group)
        assert rel(g - m0, added) < ATTN_BAR + 6e-8 * (1 + heads // kv) * math.sqrt(added.size) / np.linalg.norm(added)


EDGES = [0, 1, 2, 15, 16, 17, 63, 64, 65, 130]


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("f16", [True, False])
def test_decode_edge_lengths(pkg, ctx, heads, kv, hd, f16):
    check_decode(pkg, ctx, heads, kv, hd, f16, 16, EDGES, seed=heads)


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("page,layout", [(1, "nhd"), (7, "hnd"), (64, "hnd"), (128, "nhd")])
def test_decode_pages_and_strides(pkg, ctx, heads, kv, hd, f16, page, layout):
    check_decode(pkg, ctx, heads, kv, hd, f16, page, [301, 5, 0, 77], layout=layout, q_pad=12, with_mass=True, seed=page)


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("cap,window,alibi", [(50.0, 0, False), (0.0, 1, False), (0.0, 33, True), (5.0, 100, True), (0.0, 0, True)])
def test_decode_scores_and_windows(pkg, ctx, heads, kv, hd, f16, cap, window, alibi):
    check_decode(pkg, ctx, heads, kv, hd, f16, 16, [200, 33, 1, 0, 99], cap, window, alibi, with_mass=True, seed=window)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("lens", [[9000], [3, 4000, 0, 0, 1, 700]])
def test_decode_split_and_joined(pkg, ctx, f16, lens):
    check_decode(pkg, ctx, 32, 4, 128, f16, 16, lens, with_mass=True, seed=3)


def test_decode_many_sequences(pkg, ctx):
    """More sequences than threads in a block, most of them short."""
    rng = np.random.default_rng(4)
    check_decode(pkg, ctx, 14, 2, 64, True, 16, [int(n) for n in rng.integers(0, 40, 300)], seed=4)


def test_decode_extreme_queries(pkg, ctx):
    """Query rows of very small and very large magnitude keep their relative precision."""
    rng = np.random.default_rng(8)
    heads, kv, hd = 8, 2, 128
    for f16 in (True, False):
        c = Cache(pkg, rng, [150], kv, hd, f16, 16)
        q = rng.normal(0, 1, (1, heads, hd)) * (10.0 ** np.arange(-38, -38 + heads)[None, :, None] if f16 else 1.0)
        q[0, -1] = 0
        q[0, 0] = rng.normal(0, 1, hd) * 3e3
        q = q.astype(np.float32)
        got = run_decode(pkg, ctx, c, q, heads)
        K, V = c.seq(0)
        want, _ = attend(q[0][None], K, V, np.array([149]), np.ones((1, 150), bool), 1 / math.sqrt(hd))
        assert np.isfinite(got).all()
        # head 0's scores reach about 1e4: an f32 score is off by up to 1e4 * 2^-22, and so is its weight
        assert rel(got[0, 1:], want[0, 1:]) < ATTN_BAR
        assert rel(got[0, 0], want[0, 0]) < 1e4 * 2.0 ** -20


def test_decode_offsets_past_32_bits(pkg, ctx):
    """Pages more than 4 GiB apart."""
    rng = np.random.default_rng(9)
    heads, kv, hd, page = 8, 1, 64, 16
    stride = 1 << 30  # elements: 2 GiB in f16
    pool = torch.empty(3 * stride + page * hd, dtype=torch.float16, device="cuda")
    c = Cache(pkg, rng, [48 + 15], kv, hd, True, page, extra_pages=0)
    for p in range(4):
        pool[p * stride:p * stride + page * hd] = torch.from_numpy(np.nan_to_num(c._k[p])).cuda().reshape(-1)
    vpool = c.dv  # V stays contiguous in a pool with the same strides: its own copy
    vp = torch.empty_like(pool)
    for p in range(4):
        vp[p * stride:p * stride + page * hd] = torch.from_numpy(np.nan_to_num(c._v[p])).cuda().reshape(-1)
    c.desc = pkg.PagedKV(n_kv_heads=kv, head_dim=hd, kv_f16=1, page_size=page, n_pages=4, max_pages=c.width,
                         page_stride=stride, slot_stride=hd, head_stride=hd, k=pool.data_ptr(), v=vp.data_ptr())
    q = rng.normal(0, 1.5, (1, heads, hd)).astype(np.float32)
    got = run_decode(pkg, ctx, c, q, heads)
    K, V = c.seq(0)
    want, _ = attend(q, K, V, np.array([62]), np.ones((1, 63), bool), 1 / math.sqrt(hd))
    assert rel(got, want) < ATTN_BAR
    del pool, vp, vpool


def test_decode_same_result_twice_and_in_a_graph(pkg, ctx):
    """No result depends on timing; a captured step follows its device-side lengths."""
    rng = np.random.default_rng(10)
    heads, kv, hd, lens = 32, 4, 128, [2000, 17, 900]
    c = Cache(pkg, rng, lens, kv, hd, True, 16)
    q = torch.from_numpy(rng.normal(0, 1.5, (3, heads * hd)).astype(np.float32)).cuda()
    cfg = pkg.PagedAttnCfg(n_heads=heads, scale=1 / math.sqrt(hd))
    out, ln = torch.zeros(3, heads * hd, device="cuda"), i32(lens)
    torch.cuda.synchronize()
    seen = []
    for _ in range(5):
        ctx.paged_attn_decode(cfg, c.desc, q, 3, c.dtable, ln, 2000, out)
        ctx.sync()
        seen.append(out.clone())
    assert all(torch.equal(seen[0], x) for x in seen)
    ctx.capture_begin()
    ctx.paged_attn_decode(cfg, c.desc, q, 3, c.dtable, ln, 2000, out)
    graph = ctx.capture_end()
    for new in (lens, [1500, 1, 0], lens):
        ln.copy_(i32(new))
        torch.cuda.synchronize()
        graph.launch()
        ctx.sync()
        c.lens = new
        want = run_decode(pkg, ctx, c, q.cpu().numpy(), heads)
        assert np.array_equal(out.cpu().numpy().reshape(want.shape), want)
    graph.free()


def test_decode_on_callers_stream(pkg):
    rng = np.random.default_rng(11)
    heads, kv, hd = 14, 2, 64
    c = Cache(pkg, rng, [333], kv, hd, True, 16)
    q = rng.normal(0, 1.5, (1, heads, hd)).astype(np.float32)
    with pkg.Context(0) as other:
        base = run_decode(pkg, other, c, q, heads)
        s = torch.cuda.Stream()
        other.set_stream(s)
        with torch.cuda.stream(s):
            qd = torch.zeros(1, heads * hd, device="cuda")
            out = torch.zeros(1, heads * hd, device="cuda")
            ln, cfg = i32([333]), pkg.PagedAttnCfg(n_heads=heads, scale=1 / math.sqrt(hd))
            qd.copy_(torch.from_numpy(q.reshape(1, -1)).pin_memory(), non_blocking=True)  # orders with the op on s
            other.paged_attn_decode(cfg, c.desc, qd, 1, c.dtable, ln, 333, out)
            got = out.cpu().numpy()
        other.set_stream(None)
    assert np.array_equal(got.reshape(base.shape), base)


@pytest.mark.parametrize("what", ["page", "len"])
def test_decode_bad_index_reported(pkg, ctx, what):
    rng = np.random.default_rng(12)
    c = Cache(pkg, rng, [40, 40], 2, 64, True, 16)
    if what == "page":
        c.table[0, 1] = c.n_pages
        c.dtable = i32(c.table)
        lens = [40, 40]
    else:
        lens = [41 + 16, 40]
    out = torch.zeros(2, 4 * 64, device="cuda")
    cfg = pkg.PagedAttnCfg(n_heads=4, scale=0.125)
    q, ln = torch.ones(2, 4 * 64, device="cuda"), i32(lens)
    ctx.paged_attn_decode(cfg, c.desc, q, 2, c.dtable, ln, 40, out)
    with pytest.raises(pkg.LtError) as e:
        ctx.sync()
    assert e.value.status == 1
    assert torch.isfinite(out[1]).all()
    ctx.sync()


def test_attention_refusals(pkg, ctx):
    rng = np.random.default_rng(13)
    c = Cache(pkg, rng, [40], 2, 64, True, 16)
    q = torch.zeros(1, 4 * 64, device="cuda")
    ln, cu = i32([40]), i32([0, 1])

    def refused(kv=None, cfg=None, max_len=40, n_seq=1, **kw):
        d = pkg.PagedKV.from_buffer_copy(c.desc)
        for k, v in (kv or {}).items():
            setattr(d, k, v)
        a = pkg.PagedAttnCfg(**{**dict(n_heads=4, scale=0.125), **(cfg or {})})
        for op in ("decode",) if "mass" in kw else ("decode", "prompt"):
            with pytest.raises(pkg.LtError) as e:
                if op == "decode":
                    ctx.paged_attn_decode(a, d, kw.get("q", q), n_seq, c.dtable, ln, max_len, q, kw.get("mass"), kw.get("ms", 0))
                else:
                    ctx.paged_attn_prompt(a, d, kw.get("q", q), n_seq, cu, 1, 1, c.dtable, ln, max_len, q)
            assert e.value.status == 1 and str(e.value)

    refused(kv=dict(head_dim=96))
    refused(kv=dict(n_kv_heads=0))
    refused(kv=dict(n_kv_heads=3))
    refused(kv=dict(page_size=0))
    refused(kv=dict(n_pages=0))
    refused(kv=dict(max_pages=0))
    refused(kv=dict(slot_stride=128))
    refused(kv=dict(page_stride=2048, slot_stride=132, head_stride=64))
    refused(kv=dict(k=c.dk.data_ptr() + 2))
    refused(kv=dict(v=None))
    refused(cfg=dict(n_heads=0))
    refused(cfg=dict(n_heads=5))
    refused(cfg=dict(softcap=-1.0))
    refused(cfg=dict(softcap=float("nan")))
    refused(cfg=dict(scale=float("inf")))
    refused(cfg=dict(q_stride=128))
    refused(cfg=dict(out_stride=258))
    refused(max_len=0)
    refused(max_len=(1 << 30) + 1)
    refused(n_seq=70000)
    refused(q=q.data_ptr() + 4)
    refused(q=None)
    refused(mass=q, ms=39)
    with pytest.raises(pkg.LtError):  # document numbers must cover max_len
        ctx.paged_attn_prompt(pkg.PagedAttnCfg(n_heads=4, scale=0.125), c.desc, q, 1, cu, 1, 1, c.dtable, ln, 40, q, None, ln, 39)
    ctx.paged_attn_decode(pkg.PagedAttnCfg(n_heads=4, scale=0.125), c.desc, q, 0, c.dtable, ln, 40, q)  # nothing to do
    ctx.sync()


# ── prompts ──────────────────────────────────────────────────────────────────

def check_prompt(pkg, ctx, heads, kv, hd, f16, page, new, lens, causal=True, cap=0.0, window=0, alibi=False, prefix=None,
                 docs=None, layout="nhd", seed=0, q_pad=0):
    rng = np.random.default_rng(seed)
    c = Cache(pkg, rng, lens, kv, hd, f16, page, layout)
    total = sum(new)
    q = rng.normal(0, 1.5, (total, heads, hd)).astype(np.float32)
    slopes = (2.0 ** (-8.0 * (np.arange(heads) + 1) / heads)).astype(np.float32) if alibi else None
    sl = None if slopes is None else torch.from_numpy(slopes).cuda()
    row = heads * hd + q_pad
    qd = torch.zeros(total, row, device="cuda")
    qd[:, :heads * hd] = torch.from_numpy(q.reshape(total, -1)).cuda()
    out = torch.full((total, row), 7.0, device="cuda")
    most = max(1, max(lens))
    cfg = pkg.PagedAttnCfg(n_heads=heads, window=window, causal=int(causal), scale=1 / math.sqrt(hd), softcap=cap,
                           slopes=None if sl is None else sl.data_ptr(), q_stride=row, out_stride=row)
    cu, ln = i32(np.concatenate([[0], np.cumsum(new)])), i32(lens)
    pf = None if prefix is None else i32(prefix)
    dn = None
    if docs is not None:
        dn = np.zeros((len(lens), most + 1), np.int64)
        for s, n in enumerate(lens):
            dn[s, :n] = docs(np.arange(n))
    dd = None if dn is None else i32(dn)
    ctx.paged_attn_prompt(cfg, c.desc, qd, len(lens), cu, total, max(new), c.dtable, ln, most, out, pf, dd, most + 1)
    ctx.sync()
    if q_pad:
        assert (out[:, heads * hd:] == 7.0).all()
    got = out[:, :heads * hd].cpu().numpy().reshape(total, heads, hd)
    want = np.zeros(got.shape)
    first = 0
    for s, (m, n) in enumerate(zip(new, lens)):
        K, V = c.seq(s)
        i, j = np.arange(n - m, n)[:, None], np.arange(n)[None]
        seen = np.ones((m, n), bool)
        if causal:
            seen &= (j <= i) | (j < (prefix[s] if prefix is not None else 0))
        if window:
            seen &= i - j < window
        if docs is not None:
            seen &= np.where(i >= 0, dn[s][np.clip(i, 0, None)], -1) == dn[s, :n][None]
        want[first:first + m], _ = attend(q[first:first + m], K, V, i[:, 0], seen, 1 / math.sqrt(hd), cap, slopes)
        empty = ~seen.any(1) if n else np.ones(m, bool)
        assert not got[first:first + m][empty].any()
        first += m
    assert np.isfinite(got).all()
    assert rel(got, want) < ATTN_BAR
    return got, want


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new,lens", [([1, 3, 130, 0, 17], [1, 40, 130, 9, 200])])
def test_prompt_causal(pkg, ctx, heads, kv, hd, f16, new, lens):
    check_prompt(pkg, ctx, heads, kv, hd, f16, 16, new, lens, seed=hd)


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("kw", [
    dict(causal=False), dict(window=1), dict(window=20, alibi=True), dict(cap=20.0, alibi=True),
    dict(prefix=[0, 31, 150]), dict(prefix=[2, 200, 10], window=40), dict(docs=lambda j: j // 23),
    dict(docs=lambda j: j % 3, causal=False), dict(docs=lambda j: j // 50, prefix=[9, 70, 150], cap=30.0, window=60),
])
def test_prompt_masks(pkg, ctx, heads, kv, hd, f16, kw):
    check_prompt(pkg, ctx, heads, kv, hd, f16, 24, [40, 90, 151], [40, 140, 151], seed=3, **kw)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_more_queries_than_positions(pkg, ctx, f16, causal):
    """Queries before position 0 see nothing of a causal cache; an empty cache gives zeros."""
    check_prompt(pkg, ctx, 8, 2, 128, f16, 16, [30, 12, 5], [10, 0, 5], causal=causal, seed=5)


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (32, 4, 128), (16, 8, 256)])
def test_prompt_longer(pkg, ctx, heads, kv, hd):
    check_prompt(pkg, ctx, heads, kv, hd, True, 16, [300, 700], [900, 700], seed=6, layout="hnd", q_pad=8)


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (32, 4, 128), (16, 8, 256)])
@pytest.mark.parametrize("page,layout", [(1, "nhd"), (8, "hnd"), (20, "nhd"), (64, "hnd"), (128, "nhd"), (200, "hnd")])
def test_prompt_pages(pkg, ctx, heads, kv, hd, page, layout):
    """Pages smaller and larger than a tile of keys, a multiple of 8 slots or not, in both layouts."""
    check_prompt(pkg, ctx, heads, kv, hd, True, page, [70, 150], [333, 150], seed=page, layout=layout)
    check_prompt(pkg, ctx, heads, kv, hd, True, page, [90], [421], seed=page, layout=layout, window=130)


def test_prompt_offsets_past_32_bits(pkg, ctx):
    """Pages more than 4 GiB apart, on the way that copies them by tensor maps and on the other."""
    rng = np.random.default_rng(19)
    heads, kv, hd = 8, 1, 64
    for page in (32, 9):
        stride = 1 << 30  # elements: 2 GiB in f16
        n = 4 * page - 3
        c = Cache(pkg, rng, [n], kv, hd, True, page, extra_pages=0)
        pools = []
        for src in (c._k, c._v):
            t = torch.empty(3 * stride + page * hd, dtype=torch.float16, device="cuda")
            for p in range(4):
                t[p * stride:p * stride + page * hd] = torch.from_numpy(np.nan_to_num(src[p])).cuda().reshape(-1)
            pools.append(t)
        desc = pkg.PagedKV(n_kv_heads=kv, head_dim=hd, kv_f16=1, page_size=page, n_pages=4, max_pages=c.width,
                           page_stride=stride, slot_stride=hd, head_stride=hd, k=pools[0].data_ptr(), v=pools[1].data_ptr())
        q = rng.normal(0, 1.5, (n, heads, hd)).astype(np.float32)
        qd, out = torch.from_numpy(q.reshape(n, -1)).cuda(), torch.zeros(n, heads * hd, device="cuda")
        cu, ln = i32([0, n]), i32([n])
        cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=1 / math.sqrt(hd))
        ctx.paged_attn_prompt(cfg, desc, qd, 1, cu, n, n, c.dtable, ln, n, out)
        ctx.sync()
        K, V = c.seq(0)
        i = np.arange(n)
        want, _ = attend(q, K, V, i, i[None] <= i[:, None], 1 / math.sqrt(hd))
        assert rel(out.cpu().numpy().reshape(want.shape), want) < ATTN_BAR
        del pools, t


@pytest.mark.parametrize("f16", [True, False])
def test_serving_step_in_a_graph(pkg, ctx, f16):
    """Append, prompt attention, decode with weights and eviction, recorded once and replayed on other contents."""
    rng = np.random.default_rng(20)
    heads, kv, hd, page, m = 14, 2, 64, 16, 40
    lens = [60, 120]
    c = Cache(pkg, rng, [n + 1 for n in lens], kv, hd, f16, page, extra_pages=12)
    acfg = pkg.AttnCfg(n_heads=heads, n_kv_heads=kv, head_dim=hd, rope_neox=1, rope_theta=1e4, eps=1e-6, scale=1.0, kv_cap=1,
                       kv_f16=int(f16))
    cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=1 / math.sqrt(hd))
    qkv = torch.zeros(2, (heads + 2 * kv) * hd, device="cuda")
    q, out = torch.zeros(2, heads * hd, device="cuda"), torch.zeros(2, heads * hd, device="cuda")
    pq, pout = torch.zeros(2 * m, heads * hd, device="cuda"), torch.zeros(2 * m, heads * hd, device="cuda")
    cu, seq, pos, ln = i32([0, m, 2 * m]), i32([0, 1]), i32(lens), i32([n + 1 for n in lens])
    mass, mass2 = torch.zeros(2, kv, 128, device="cuda"), torch.zeros(2, kv, 50, device="cuda")
    kept, ln2 = torch.zeros(2, kv, 50, dtype=torch.int32, device="cuda"), i32([0, 0])
    dst = np.full_like(c.table, 0xFFFFFFFF)
    dst[0, :4], dst[1, :4] = c.free[:4], c.free[4:8]
    dd = i32(dst)
    torch.cuda.synchronize()

    def step():
        ctx.paged_append(acfg, c.desc, qkv, 2, None, None, seq, pos, None, c.dtable, 2, q)
        ctx.paged_attn_prompt(cfg, c.desc, pq, 2, cu, 2 * m, m, c.dtable, ln, 121, pout)
        ctx.paged_attn_decode(cfg, c.desc, q, 2, c.dtable, ln, 121, out, mass, 128)
        ctx.kv_evict(c.desc, 2, c.dtable, ln, 121, mass, 128, 50, 10, dd, ln2, mass2, 50, kept)

    def fill(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in (qkv, pq):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        mass.zero_()
        torch.cuda.synchronize()

    fill(1)
    step()  # the arena grows here
    ctx.sync()
    ctx.capture_begin()
    step()
    graph = ctx.capture_end()
    for seed in (2, 3):
        fill(seed)
        step()
        ctx.sync()
        want = [t.clone() for t in (out, pout, mass, mass2, kept, ln2, c.dk, c.dv)]
        for t in (out, pout, mass2, kept, ln2):
            t.zero_()
        fill(seed)
        graph.launch()
        ctx.sync()
        got = (out, pout, mass, mass2, kept, ln2, c.dk, c.dv)
        assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(got, want))
        assert ln2.tolist() == [50, 50] and float(mass.sum()) == pytest.approx(2 * heads, rel=1e-5)
    graph.free()


def test_prompt_few_tokens_long_cache(pkg, ctx):
    """A handful of queries per sequence over long caches, as in checking drafted tokens."""
    for f16 in (True, False):
        check_prompt(pkg, ctx, 32, 4, 128, f16, 16, [4, 5, 1], [3000, 777, 1200], seed=7)


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (32, 4, 128), (16, 8, 256)])
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("mask", ["causal", "window", "docs", "split"])
def test_prompt_masked_values_may_be_anything(pkg, ctx, heads, kv, hd, f16, mask):
    """Infinities and NaN in K and V of positions that a query does not see do not reach it."""
    rng = np.random.default_rng(21)
    n, m = (1300, 40) if mask == "split" else (230, 230)
    c = Cache(pkg, rng, [n], kv, hd, f16, 16)
    bad = n - 7 if mask in ("causal", "split") else 100
    for j, x in ((bad, np.nan), (bad + 1, np.inf)):
        c.hk[c.table[0, j // 16], j % 16] = x
        c.hv[c.table[0, j // 16], j % 16] = -x
    c.upload(pkg)
    q = rng.normal(0, 1.5, (m, heads, hd)).astype(np.float32)
    docs = np.zeros((1, n), np.int64)
    docs[0, 90:110] = 1
    window = 50 if mask == "window" else 0
    cfg = pkg.PagedAttnCfg(n_heads=heads, window=window, causal=1, scale=1 / math.sqrt(hd))
    qd, out = torch.from_numpy(q.reshape(m, -1)).cuda(), torch.zeros(m, heads * hd, device="cuda")
    cu, ln, dd = i32([0, m]), i32([n]), i32(docs)
    ctx.paged_attn_prompt(cfg, c.desc, qd, 1, cu, m, m, c.dtable, ln, n, out, None, dd if mask == "docs" else None, n)
    ctx.sync()
    got = out.cpu().numpy().reshape(m, heads, hd)
    i, j = np.arange(n - m, n)[:, None], np.arange(n)[None]
    seen = j <= i
    if window:
        seen = seen & (i - j < window)
    if mask == "docs":
        seen = seen & (docs[0][i] == docs[0][j])
    clean = ~seen[:, bad:bad + 2].any(1)
    assert clean.any() and not clean.all()
    K, V = c.seq(0)
    K, V = np.nan_to_num(K, nan=0, posinf=0, neginf=0), np.nan_to_num(V, nan=0, posinf=0, neginf=0)
    want, _ = attend(q[clean], K, V, i[clean, 0], seen[clean], 1 / math.sqrt(hd))
    assert rel(got[clean], want) < ATTN_BAR
    assert np.isnan(got[~clean]).any(axis=(1, 2)).all()


def test_prompt_bad_ranges_reported(pkg, ctx):
    rng = np.random.default_rng(14)
    c = Cache(pkg, rng, [40, 40], 2, 64, True, 16)
    cfg = pkg.PagedAttnCfg(n_heads=4, scale=0.125, causal=1)
    q, out, ln = torch.zeros(8, 4 * 64, device="cuda"), torch.zeros(8, 4 * 64, device="cuda"), i32([40, 40])
    for cu, most in (([0, 4, 9], 5), ([0, 6, 8], 5), ([5, 4, 8], 5)):
        ctx.paged_attn_prompt(cfg, c.desc, q, 2, i32(cu), 8, most, c.dtable, ln, 40, out)
        with pytest.raises(pkg.LtError) as e:
            ctx.sync()
        assert e.value.status == 1
    ctx.sync()


# ── eviction ─────────────────────────────────────────────────────────────────

def evict_ref(mass, n, budget, recent):
    if n <= budget:
        return np.arange(n)
    old = n - recent
    m = np.where(np.isnan(mass[:old]), np.inf, mass[:old].astype(np.float64))
    nan_first = ~np.isnan(mass[:old])
    best = np.lexsort((np.arange(old), -m, nan_first))[:budget - recent]
    return np.concatenate([np.sort(best), np.arange(old, n)]).astype(np.int64)


def check_evict(pkg, ctx, kv, hd, f16, page, lens, budget, recent, fill, in_place, layout="nhd", seed=0, kept_out=True):
    rng = np.random.default_rng(seed)
    extra = len(lens) * -(-budget // page) + 1
    c = Cache(pkg, rng, lens, kv, hd, f16, page, layout, extra_pages=extra, spare=2)
    most, S = max(1, max(lens)), len(lens)
    mass = fill(rng, (S, kv, most + 5)).astype(np.float32)
    dst = np.full_like(c.table, 0xFFFFFFFF)
    at = 0
    for s, n in enumerate(lens):
        k = -(-min(n, budget) // page)
        dst[s, :k] = c.free[at:at + k]
        at += k
    dm, ln, dd = torch.from_numpy(mass).cuda(), i32(lens), i32(dst)
    lens_out = ln if in_place else torch.full((S,), -1, dtype=torch.int32, device="cuda")
    out_stride = mass.shape[2] if in_place else budget + 1
    mass_out = dm if in_place else torch.full((S, kv, out_stride), -5.0, device="cuda")
    kept = torch.full((S, kv, budget), -1, dtype=torch.int32, device="cuda")
    ctx.kv_evict(c.desc, S, c.dtable, ln, most, dm, mass.shape[2], budget, recent, None if in_place else dd, lens_out, mass_out,
                 out_stride, kept if kept_out else None)
    ctx.sync()
    gk, gv = (t.cpu().numpy() for t in (c.dk, c.dv))
    if layout == "hnd":
        gk, gv = gk.swapaxes(1, 2), gv.swapaxes(1, 2)
    table = c.table if in_place else dst
    got_mass, got_kept = mass_out.cpu().numpy(), kept.cpu().numpy()
    touched = np.zeros((c.n_pages, page, kv), bool)
    for s, n in enumerate(lens):
        m = min(n, budget)
        assert int(lens_out[s]) == m
        for h in range(kv):
            want = evict_ref(mass[s, h, :n], n, budget, recent)
            if kept_out:
                assert np.array_equal(got_kept[s, h, :m], want)
                assert (got_kept[s, h, m:] == -1).all()
            assert np.array_equal(got_mass[s, h, :m], mass[s, h, want], equal_nan=True)
            i = np.arange(m)
            src, to = c.table[s, want // page], table[s, i // page]
            assert np.array_equal(gk[to, i % page, h], c.hk[src, want % page, h])
            assert np.array_equal(gv[to, i % page, h], c.hv[src, want % page, h])
            touched[to, i % page, h] = True
    if not in_place:
        assert (got_mass[:, :, budget:] == -5.0).all()
    # slots that nothing moved to keep their bits
    assert np.array_equal(gk[~touched], c.hk[~touched], equal_nan=True)


FILLS = {
    "random": lambda rng, sh: rng.uniform(0, 3, sh),
    "zeros": lambda rng, sh: np.zeros(sh),
    "ties": lambda rng, sh: rng.integers(0, 4, sh) * 0.25,
    "skewed": lambda rng, sh: np.exp(rng.normal(0, 30, sh).clip(-87, 87)),
    "special": lambda rng, sh: rng.choice([0.0, -0.0, 1e-45, 1.0, -1.0, np.inf, np.nan, 3e38], sh),
}


@pytest.mark.parametrize("fill", sorted(FILLS))
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kv,hd,f16,page,layout", [(2, 64, True, 16, "nhd"), (1, 128, False, 7, "hnd"), (3, 256, False, 32, "nhd")])
def test_evict(pkg, ctx, fill, in_place, kv, hd, f16, page, layout):
    check_evict(pkg, ctx, kv, hd, f16, page, [0, 1, 60, 61, 62, 190], 61, 9, FILLS[fill], in_place, layout)


@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (40, 40), (40, 0), (500, 100)])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_budgets(pkg, ctx, budget, recent, in_place):
    check_evict(pkg, ctx, 2, 64, True, 16, [100, 39, 40, 41], budget, recent, FILLS["random"], in_place, seed=2, kept_out=False)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("fill", ["random", "ties", "zeros"])
def test_evict_long(pkg, ctx, in_place, fill):
    """Several passes of the selection and of the moving CTAs over one row."""
    check_evict(pkg, ctx, 1, 64, True, 64, [21000, 9000], 5000, 100, FILLS[fill], in_place, seed=4)


def test_evict_refusals_and_bad_pages(pkg, ctx):
    rng = np.random.default_rng(15)
    c = Cache(pkg, rng, [40], 2, 64, True, 16)
    m, ln, kept = torch.zeros(1, 2, 40, device="cuda"), i32([40]), torch.zeros(1, 2, 8, dtype=torch.int32, device="cuda")
    mo, lo = torch.zeros(1, 2, 8, device="cuda"), i32([0])

    def call(budget=8, recent=2, max_len=40, ms=40, mos=8, lens=ln, table=c.dtable, mass=m, out=mo, lens_out=lo):
        ctx.kv_evict(c.desc, 1, table, lens, max_len, mass, ms, budget, recent, None, lens_out, out, mos, kept)

    for bad in (dict(budget=0), dict(recent=9), dict(max_len=0), dict(ms=39), dict(mos=7), dict(mass=None), dict(lens=None),
                dict(lens_out=None), dict(out=m)):
        with pytest.raises(pkg.LtError) as e:
            call(**bad)
        assert e.value.status == 1
    c.table[0, 2] = 1 << 20
    before = c.dk.clone()
    call(table=i32(c.table))
    with pytest.raises(pkg.LtError):
        ctx.sync()
    call(lens=i32([1 << 20]))
    with pytest.raises(pkg.LtError):
        ctx.sync()
    ctx.sync()
    assert before.shape == c.dk.shape

"""A paged cache in 8 bits (lt_paged_q8_append, lt_paged_q8_attn_decode, lt_paged_q8_attn_prompt) against plain 64-bit
implementations.

Bars, from the arithmetic.  Attention: codes are exact in the products, scales are f32; queries and weights enter as two
terms of 11 bits each (2^-22), sums are f32, so a score of magnitude s is off by about s * 2^-21 and a weight by as much;
the logarithm of V's scale, |log2 vs| <= 10 here, adds 10 * 2^-24.  With |s| up to about 10: 5e-6 at worst and less in a
sum: rel-L2 < 1e-5.
Append: a value is off by 1e-6 of its block's largest (the norm's f32 sum and quotients, 4 roundings, the angle's 2^-23; what
a rotation mixes is no larger than twice that), and that is 127 steps: 2.6e-4 steps, the quotient's rounding 127 * 2^-24 of one.
A code is within 0.5 + 2e-3 steps of its value, a scale within 2e-6.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ATTN_BAR = 1e-5
CODE_BAR = 0.5 + 2e-3


def i32(v):
    return torch.as_tensor(np.asarray(v, dtype=np.int64).astype(np.uint32).view(np.int32)).cuda()


def rel(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30))


class Cache:
    """Codes and scales of sequences of the given lengths; what no sequence holds is any byte, on scales that are no numbers."""

    def __init__(self, pkg, rng, lens, kv, hd, page, block, layout="hnd", extra_pages=2, spare=0, spread=0.0):
        self.lens, self.kv, self.hd, self.page, self.block, self.layout = lens, kv, hd, page, block, layout
        need = [-(-n // page) for n in lens]
        self.width = max(1, max(need)) + spare
        self.n_pages = sum(need) + extra_pages
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), self.width), 0xFFFFFFFF, dtype=np.int64)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.free = order[at:].tolist()
        shape = (self.n_pages, page, kv, hd) if layout == "nhd" else (self.n_pages, kv, page, hd)
        self._c = [rng.integers(-128, 128, shape).astype(np.int8) for _ in range(2)]
        self.hc = [x.swapaxes(1, 2) if layout == "nhd" else x for x in self._c]      # [page][head][slot][hd] views
        self.hs = [np.full((self.n_pages, kv, page // block), np.nan, np.float32) for _ in range(2)]
        for x, y in zip(self.hs, (np.inf, -1.0)):
            x[::2] = y
        for s, n in enumerate(lens):
            for j0 in range(0, n, block):
                p = self.table[s, j0 // page]
                for t in range(2):
                    scale = np.exp(rng.normal(0, spread, kv)) * rng.uniform(2.5, 4.0, kv) / 127 * (0.7 if t else 1.0)
                    x = np.clip(np.rint(rng.normal(0, 1, (kv, block, hd)) / scale[:, None, None]), -127, 127)
                    m = min(block, n - j0)
                    self.hc[t][p, :, j0 % page:j0 % page + m] = x[:, :m]
                    self.hs[t][p, :, j0 % page // block] = scale
        self.upload(pkg)

    def upload(self, pkg):
        self.dc = [torch.from_numpy(x).cuda() for x in self._c]
        self.ds = [torch.from_numpy(x).cuda() for x in self.hs]
        self.dtable = i32(self.table)
        p, kv, hd = self.page, self.kv, self.hd
        st = (0, 0, 0) if self.layout == "hnd" else (kv * p * hd, kv * hd, hd)
        self.desc = pkg.PagedQ8(n_kv_heads=kv, head_dim=hd, page_size=p, block=self.block, n_pages=self.n_pages,
                                max_pages=self.width, page_stride=st[0], slot_stride=st[1], head_stride=st[2],
                                k=self.dc[0].data_ptr(), v=self.dc[1].data_ptr(), k_scale=self.ds[0].data_ptr(),
                                v_scale=self.ds[1].data_ptr())
        torch.cuda.synchronize()

    def download(self):
        """The device's codes and scales as [page][head][slot][hd] and [page][head][block]."""
        c = [x.cpu().numpy() for x in self.dc]
        return [x.swapaxes(1, 2) if self.layout == "nhd" else x for x in c], [x.cpu().numpy() for x in self.ds]

    def seq(self, s, n=None):
        """K and V [n][kv][hd] of sequence s in 64 bits."""
        j = np.arange(self.lens[s] if n is None else n)
        p = self.table[s, j // self.page]
        return [self.hc[t][p, :, j % self.page].astype(np.float64) *
                self.hs[t][p, :, j % self.page // self.block].astype(np.float64)[..., None] for t in range(2)]


def attend(q, K, V, i, seen, scale, cap=0.0, slopes=None):
    """q [m][H][hd] at positions i [m], K and V [n][kv][hd], seen [m][n] -> out [m][H][hd]."""
    m, H, hd = q.shape
    n, kv = K.shape[:2]
    out = np.zeros((m, H, hd))
    if n == 0:
        return out
    for h in range(H):
        s = q[:, h].astype(np.float64) @ K[:, h // (H // kv)].T * scale
        if cap:
            s = cap * np.tanh(s / cap)
        if slopes is not None:
            s = s - float(slopes[h]) * np.abs(i[:, None] - np.arange(n)[None])
        s = np.where(seen, s, -np.inf)
        some = seen.any(1)
        e = np.exp(s[some] - s[some].max(1, keepdims=True))
        out[some, h] = e / e.sum(1, keepdims=True) @ V[:, h // (H // kv)]
    return out


SHAPES = [(14, 2, 64), (32, 4, 128), (16, 8, 256), (4, 4, 128), (16, 1, 64), (40, 2, 128)]


# ── append ───────────────────────────────────────────────────────────────────

def turned(x, heads, kv, pos, theta, eps, qn, kn, v_norm, neox):
    """Rows [t][H + 2 kv][hd] normalised and rotated, in 64 bits."""
    x = x.astype(np.float64)
    hd = x.shape[-1]
    inv = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    y = x.copy()
    if qn is not None:
        y[:, :heads] = x[:, :heads] * inv[:, :heads] * qn
        y[:, heads:heads + kv] = x[:, heads:heads + kv] * inv[:, heads:heads + kv] * kn
    if v_norm:
        y[:, heads + kv:] = x[:, heads + kv:] * inv[:, heads + kv:]
    half = hd // 2
    ang = np.asarray(pos, np.float64)[:, None] * theta ** (-2.0 * np.arange(half) / hd)
    cs, sn = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = (slice(0, half), slice(half, hd)) if neox else (slice(0, hd, 2), slice(1, hd, 2))
    z, r = y.copy(), slice(0, heads + kv)
    z[:, r, a] = y[:, r, a] * cs - y[:, r, b] * sn
    z[:, r, b] = y[:, r, a] * sn + y[:, r, b] * cs
    return z


class Appends:
    """A cache and calls of lt_paged_q8_append into it, checked against the rules of the format."""

    def __init__(self, pkg, ctx, c, rng, heads, neox=True, v_norm=False, norms=True, theta=1e5):
        self.pkg, self.ctx, self.c, self.rng, self.heads = pkg, ctx, c, rng, heads
        self.neox, self.v_norm, self.theta, self.eps = neox, v_norm, theta, 1e-6
        self.qn, self.kn = (rng.normal(1, 0.2, c.hd).astype(np.float32) for _ in range(2)) if norms else (None, None)
        self.dn = [None if w is None else torch.from_numpy(w).cuda() for w in (self.qn, self.kn)]
        self.cfg = pkg.AttnCfg(n_heads=heads, n_kv_heads=c.kv, head_dim=c.hd, rope_neox=int(neox), rope_theta=theta, eps=self.eps,
                               scale=1.0, kv_cap=1, window=0, v_norm=int(v_norm), kv_f16=0)

    def call(self, qkv, new, lens, pos=None, extra=2):
        """lens with the new rows; returns q, with `extra` rows of marks behind the last."""
        c, total = self.c, len(qkv)
        x = torch.from_numpy(np.concatenate([qkv, np.full((extra,) + qkv.shape[1:], np.nan, np.float32)])).cuda()
        q = torch.full((total + extra, self.heads, c.hd), 7.0, device="cuda")
        cu, ln = i32(np.concatenate([[0], np.cumsum(new)])), i32(lens)
        dp = None if pos is None else i32(list(pos) + [0] * extra)
        torch.cuda.synchronize()
        self.ctx.paged_q8_append(self.cfg, c.desc, x, len(new), cu, total + extra, max(new) + 1, self.dn[0], self.dn[1], dp,
                                 c.dtable, ln, q)
        self.ctx.sync()
        assert (q[total:] == 7.0).all()
        return q[:total].cpu().numpy()

    def check(self, new, lens, pos=None, scale_of=2.0):
        c, heads, kv, hd, B = self.c, self.heads, self.c.kv, self.c.hd, self.c.block
        qkv = (self.rng.normal(0, scale_of, (sum(new), heads + 2 * kv, hd))).astype(np.float32)
        places = np.concatenate([np.arange(n - m, n) for m, n in zip(new, lens)]).astype(np.int64)
        want = turned(qkv, heads, kv, places if pos is None else pos, self.theta, self.eps, self.qn, self.kn, self.v_norm, self.neox)
        c0, s0 = [x.copy() for x in c.hc], [x.copy() for x in c.hs]
        q = self.call(qkv, new, lens, pos)
        assert rel(q, want[:, :heads]) < 1e-6
        got, scales = c.download()
        touched = np.zeros((c.n_pages, c.page), bool)
        blocks = np.zeros((c.n_pages, c.page // B), bool)
        first = 0
        for s, (m, n) in enumerate(zip(new, lens)):
            for j0 in range((n - m) // B * B, n if m else 0, B):
                p, b, i0 = c.table[s, j0 // c.page], j0 % c.page // B, j0 % c.page
                lo, hi = max(j0, n - m), min(j0 + B, n)
                rows = slice(first + lo - (n - m), first + hi - (n - m))
                old = lo - j0
                for t in range(2):
                    x = want[rows, heads + t * kv:heads + (t + 1) * kv].swapaxes(0, 1)      # [kv][rows][hd]
                    fresh = np.abs(x).max((1, 2)) / 127
                    was = s0[t][p, :, b].astype(np.float64)
                    now = scales[t][p, :, b].astype(np.float64)
                    expect = np.maximum(fresh, was) if old else fresh
                    assert np.allclose(now, expect, rtol=2e-6, atol=0)
                    code = got[t][p, :, i0 + old:i0 + hi - j0].astype(np.float64)
                    assert (np.abs(code) <= 127).all()
                    assert (np.abs(code * now[:, None, None] - x) <= now[:, None, None] * CODE_BAR).all()
                    if old:
                        before = c0[t][p, :, i0:i0 + old].astype(np.float64)
                        after = got[t][p, :, i0:i0 + old].astype(np.float64)
                        same = now == was
                        assert (after[same] == before[same]).all()
                        assert (np.abs(after * now[:, None, None] - before * was[:, None, None]) <= now[:, None, None] * CODE_BAR).all()
                touched[p, i0:i0 + hi - j0] = True
                blocks[p, b] = True
            first += m
        for t in range(2):  # nothing else is touched
            assert np.array_equal(c0[t].swapaxes(1, 2)[~touched], got[t].swapaxes(1, 2)[~touched])
            assert np.array_equal(s0[t].swapaxes(1, 2)[~blocks], scales[t].swapaxes(1, 2)[~blocks], equal_nan=True)
            c.hc[t][...] = got[t]
            c.hs[t][...] = scales[t]


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (32, 4, 128), (16, 8, 256), (3, 1, 128)])
@pytest.mark.parametrize("neox,v_norm,norms,page,block,layout", [
    (True, False, True, 16, 16, "hnd"), (False, True, True, 48, 16, "nhd"), (True, True, False, 64, 32, "hnd"),
    (False, False, False, 128, 128, "nhd"), (True, False, True, 192, 64, "hnd")])
def test_append(pkg, ctx, heads, kv, hd, neox, v_norm, norms, page, block, layout):
    """Prompts, single tokens into fresh and into begun blocks, and a sequence without rows."""
    rng = np.random.default_rng(hd + page)
    c = Cache(pkg, rng, [40, 1, 301, 0, 33, 129], kv, hd, page, block, layout)
    a = Appends(pkg, ctx, c, rng, heads, neox, v_norm, norms)
    a.check([39, 1, 140, 0, 1, 2], [40, 1, 301, 0, 33, 129])
    a.check([1, 1, 301, 0, 33, 17], [17, 1, 301, 0, 33, 128], scale_of=5.0)
    a.check([1, 0, 1, 0, 0, 1], [40, 1, 64, 0, 33, 129], pos=[1000003, 7, 0], scale_of=0.1)


@pytest.mark.parametrize("block", [16, 64])
def test_append_token_by_token(pkg, ctx, block):
    """A sequence grown by single tokens of growing and falling size stays within the steps that its scales took."""
    rng = np.random.default_rng(block)
    heads, kv, hd = 4, 2, 64
    c = Cache(pkg, rng, [130], kv, hd, block, block)
    a = Appends(pkg, ctx, c, rng, heads, norms=False)
    for n in range(1, 131):
        a.check([1], [n], scale_of=1.0 + (n % 7))


@pytest.mark.parametrize("heads,kv,hd,page,block,new,past", [
    (4, 8, 256, 32, 32, [4001, 1001, 2001], [0, 700, 41]), (6, 2, 64, 128, 128, [6000], [3]), (2, 4, 128, 48, 16, [3000, 1], [7, 15])])
def test_append_long(pkg, ctx, heads, kv, hd, page, block, new, past):
    """More blocks than the device runs at once, thousands of rows to a sequence."""
    rng = np.random.default_rng(31)
    lens = [a + b for a, b in zip(new, past)]
    c = Cache(pkg, rng, lens, kv, hd, page, block)
    Appends(pkg, ctx, c, rng, heads, neox=hd != 256, v_norm=hd != 128, theta=1e6).check(new, lens)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_append_without_eps(pkg, ctx, hd, block):
    """eps = 0: rows that a warp's share of a block lacks are no rows of zeros to be normalised.  Sequences that end at every
    kind of place in their blocks, shares of a block with some rows, one and none; begun blocks, too."""
    rng = np.random.default_rng(32)
    heads, kv, new = 3, 2, [17, 1, 0, 31, 7, 130]
    c = Cache(pkg, rng, [20, 1, 5, 32, 70, 131], kv, hd, 128, block)
    a = Appends(pkg, ctx, c, rng, heads, v_norm=True)
    a.eps = a.cfg.eps = 0.0
    a.check(new, c.lens)
    a.check([2, 1, 0, 15, 1, 9], c.lens, scale_of=5.0)


def test_append_twice_changes_nothing(pkg, ctx):
    rng = np.random.default_rng(1)
    heads, kv, hd, new, lens = 8, 2, 128, [5, 33, 1], [21, 40, 64]
    c = Cache(pkg, rng, lens, kv, hd, 32, 16)
    a = Appends(pkg, ctx, c, rng, heads)
    qkv = rng.normal(0, 3, (39, heads + 2 * kv, hd)).astype(np.float32)
    q1 = a.call(qkv, new, lens)
    first = c.download()
    q2 = a.call(qkv, new, lens)
    again = c.download()
    assert np.array_equal(q1, q2)
    for x, y in zip(first[0] + first[1], again[0] + again[1]):
        assert np.array_equal(x, y, equal_nan=True)


def test_append_zeros_and_tiny_values(pkg, ctx):
    """Rows of zeros give a scale of 0 and codes of 0; values near the least f32 numbers stay finite."""
    rng = np.random.default_rng(2)
    heads, kv, hd = 2, 2, 64
    for size in (0.0, 1e-44, 1e-38, 1e-30):
        c = Cache(pkg, rng, [20], kv, hd, 16, 16)
        a = Appends(pkg, ctx, c, rng, heads, norms=False)
        qkv = (rng.normal(0, 1, (20, heads + 2 * kv, hd)) * size).astype(np.float32)
        a.call(qkv, [20], [20])
        codes, scales = c.download()
        for t in range(2):
            for j in range(20):
                p = c.table[0, j // 16]
                x = codes[t][p, :, j % 16].astype(np.float64) * scales[t][p][..., 0].astype(np.float64)[:, None]
                w = turned(qkv, heads, kv, np.arange(20), a.theta, a.eps, None, None, False, True)[j, heads + t * kv:heads + (t + 1) * kv]
                # half a step, and what a number below 2^-126 is rounded by: 2^-150 for the scale, times the code
                assert (np.abs(x - w) <= 0.51 * scales[t][p][..., 0][:, None] + 130 * 2.0 ** -149).all()


def test_append_poison(pkg, ctx):
    """A value that is no number, or beyond 2^60, makes its block's scale NaN until the block starts afresh; other heads,
    blocks and the other of K and V are as without it."""
    rng = np.random.default_rng(3)
    heads, kv, hd = 2, 2, 64
    for bad in (np.nan, np.inf, -np.inf, 2e18):
        c = Cache(pkg, rng, [40], kv, hd, 32, 16)
        a = Appends(pkg, ctx, c, rng, heads, norms=False)
        qkv = rng.normal(0, 1, (40, heads + 2 * kv, hd)).astype(np.float32)
        a.call(qkv, [40], [40])
        c1, s1 = c.download()
        spoilt = qkv.copy()
        spoilt[20, heads + kv + 1, 5] = bad     # V, head 1, position 20: block 1
        a.call(spoilt, [40], [40])
        c2, s2 = c.download()
        p = c.table[0, 0]
        assert np.isnan(s2[1][p, 1, 1])
        s2[1][p, 1, 1] = s1[1][p, 1, 1]
        c2[1] = c2[1].copy()
        c2[1][p, 1, 16:32] = c1[1][p, 1, 16:32]
        for x, y in zip(c1 + s1, c2 + s2):
            assert np.array_equal(x, y, equal_nan=True)
        a.call(qkv[21:22], [1], [22])           # behind it in the block: still NaN
        assert np.isnan(c.download()[1][1][p, 1, 1])
        a.call(qkv[16:17], [1], [17])           # the block starts afresh
        assert np.isfinite(c.download()[1][1][p, 1, 1])


def test_append_bad_index_reported(pkg, ctx):
    rng = np.random.default_rng(6)
    c = Cache(pkg, rng, [16, 16], 2, 64, 16, 16)
    cfg = pkg.AttnCfg(n_heads=2, n_kv_heads=2, head_dim=64, rope_neox=1, rope_theta=1e4, eps=1e-6, scale=1.0, kv_cap=1)
    qkv, q = torch.zeros(4, 6 * 64, device="cuda"), torch.full((4, 2 * 64), 7.0, device="cuda")
    before = c.download()
    # past the table, more rows than positions, rows out of order, past total_q, more than max_q in a sequence
    for cu, lens in (([0, 1, 2], [17, 0]), ([0, 2, 2], [1, 0]), ([2, 1, 1], [16, 0]), ([0, 5, 5], [16, 0]), ([0, 4, 4], [16, 0])):
        dcu, ln = i32(cu), i32(lens)
        torch.cuda.synchronize()
        ctx.paged_q8_append(cfg, c.desc, qkv, 2, dcu, 4, 3, None, None, None, c.dtable, ln, q)
        with pytest.raises(pkg.LtError) as e:
            ctx.sync()
        assert e.value.status == 1
    d = pkg.PagedQ8.from_buffer_copy(c.desc)
    d.n_pages = int(c.table[0, 0])              # the page's number is past the pool
    dcu, ln = i32([0, 1, 1]), i32([1, 0])
    torch.cuda.synchronize()
    if d.n_pages:
        ctx.paged_q8_append(cfg, d, qkv, 2, dcu, 4, 3, None, None, None, c.dtable, ln, q)
        with pytest.raises(pkg.LtError):
            ctx.sync()
    after = c.download()
    for x, y in zip(before[0] + before[1], after[0] + after[1]):
        assert np.array_equal(x, y, equal_nan=True)
    ctx.sync()


def test_append_refusals(pkg, ctx):
    rng = np.random.default_rng(7)
    c = Cache(pkg, rng, [16], 2, 64, 32, 16)
    good = dict(n_heads=2, n_kv_heads=2, head_dim=64, rope_neox=1, rope_theta=1e4, eps=1e-6, scale=1.0, kv_cap=1)
    qkv, q = torch.zeros(1, 6 * 64, device="cuda"), torch.zeros(1, 2 * 64, device="cuda")
    cu, ln = i32([0, 1]), i32([16])
    torch.cuda.synchronize()

    def refused(kv=None, cfg=None, x=qkv, n_seq=1, total=1, table=c.dtable):
        d = pkg.PagedQ8.from_buffer_copy(c.desc)
        for k, v in (kv or {}).items():
            setattr(d, k, v)
        with pytest.raises(pkg.LtError) as e:
            ctx.paged_q8_append(pkg.AttnCfg(**{**good, **(cfg or {})}), d, x, n_seq, cu, total, 1, None, None, None, table, ln, q)
        assert e.value.status == 1 and str(e.value)

    for kv in (dict(head_dim=96), dict(block=8), dict(block=24), dict(block=0), dict(block=256), dict(page_size=24), dict(page_size=0),
               dict(n_kv_heads=0), dict(n_pages=0), dict(max_pages=0), dict(slot_stride=64), dict(page_stride=4096, slot_stride=72, head_stride=64),
               dict(page_stride=1 << 32, slot_stride=64, head_stride=64), dict(k=c.dc[0].data_ptr() + 4), dict(v=None), dict(k_scale=None), dict(v_scale=c.ds[1].data_ptr() + 2)):
        refused(kv=kv)
    for cfg in (dict(n_heads=0), dict(n_kv_heads=1), dict(head_dim=128), dict(rope_theta=0.0), dict(rope_theta=float("inf")),
                dict(rope_theta=float("nan"))):
        refused(cfg=cfg)
    refused(x=None)
    refused(x=qkv.data_ptr() + 4)
    refused(table=None)
    refused(n_seq=65536)
    refused(total=(1 << 30) + 1)
    ctx.paged_q8_append(pkg.AttnCfg(**good), c.desc, qkv, 0, cu, 1, 1, None, None, None, c.dtable, ln, q)  # nothing to do
    ctx.sync()


# ── decode ───────────────────────────────────────────────────────────────────

def slopes_of(heads):
    return (2.0 ** (-8.0 * (np.arange(heads) + 1) / heads)).astype(np.float32)


def run_decode(pkg, ctx, c, q, heads, cap=0.0, window=0, slopes=None, q_pad=0):
    S, hd = len(c.lens), c.hd
    qd = torch.zeros(S, heads * hd + q_pad, device="cuda")
    qd[:, :heads * hd] = torch.from_numpy(q.reshape(S, -1)).cuda()
    out = torch.full((S, heads * hd + q_pad), 7.0, device="cuda")
    sl = None if slopes is None else torch.from_numpy(slopes).cuda()
    cfg = pkg.PagedAttnCfg(n_heads=heads, window=window, causal=1, scale=1 / math.sqrt(hd), softcap=cap,
                           slopes=None if sl is None else sl.data_ptr(), q_stride=heads * hd + q_pad, out_stride=heads * hd + q_pad)
    lens = i32(c.lens)
    torch.cuda.synchronize()
    ctx.paged_q8_attn_decode(cfg, c.desc, qd, S, c.dtable, lens, max(1, max(c.lens)), out)
    ctx.sync()
    if q_pad:
        assert (out[:, heads * hd:] == 7.0).all()
    return out[:, :heads * hd].cpu().numpy().reshape(S, heads, hd)


def check_decode(pkg, ctx, heads, kv, hd, page, block, lens, cap=0.0, window=0, alibi=False, layout="hnd", q_pad=0, seed=0, spread=0.0,
                 bar=ATTN_BAR):
    rng = np.random.default_rng(seed)
    c = Cache(pkg, rng, lens, kv, hd, page, block, layout, spread=spread)
    if window:  # blocks before every window have scales that are no numbers
        for s, n in enumerate(lens):
            for j in range(0, max(0, n - window) // block * block, block):
                c.hs[0][c.table[s, j // page], :, j % page // block] = np.inf if j % 64 else np.nan
                c.hs[1][c.table[s, j // page], :, j % page // block] = np.nan if j % 64 else -np.inf
        c.upload(pkg)
    q = rng.normal(0, 1.5, (len(lens), heads, hd)).astype(np.float32)
    slopes = slopes_of(heads) if alibi else None
    got = run_decode(pkg, ctx, c, q, heads, cap, window, slopes, q_pad)
    want = np.zeros(got.shape)
    for s, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        K, V = (x[lo:] for x in c.seq(s))
        want[s] = attend(q[s][None], K, V, np.array([n - 1 - lo]), np.ones((1, n - lo), bool), 1 / math.sqrt(hd), cap, slopes)[0]
        assert n or not got[s].any()
    assert np.isfinite(got).all()
    assert rel(got, want) < bar
    return got, want


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 255, 257]


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("page,block", [(16, 16), (128, 128)])
def test_decode_edge_lengths(pkg, ctx, heads, kv, hd, page, block):
    check_decode(pkg, ctx, heads, kv, hd, page, block, EDGES, seed=heads)


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
@pytest.mark.parametrize("page,block,layout", [(32, 16, "nhd"), (48, 16, "hnd"), (64, 64, "hnd"), (128, 32, "nhd"), (320, 64, "hnd")])
def test_decode_pages_and_strides(pkg, ctx, heads, kv, hd, page, block, layout):
    check_decode(pkg, ctx, heads, kv, hd, page, block, [701, 5, 0, 77], layout=layout, q_pad=12, seed=page)


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
@pytest.mark.parametrize("cap,window,alibi", [(50.0, 0, False), (0.0, 1, False), (0.0, 33, True), (5.0, 100, True), (0.0, 0, True), (0.0, 16, False)])
def test_decode_scores_and_windows(pkg, ctx, heads, kv, hd, cap, window, alibi):
    check_decode(pkg, ctx, heads, kv, hd, 16, 16, [200, 33, 1, 0, 99, 160], cap, window, alibi, seed=window)
    check_decode(pkg, ctx, heads, kv, hd, 64, 32, [200, 33, 1, 0, 99, 160], cap, window, alibi, seed=window)


@pytest.mark.parametrize("lens", [[9000], [3, 4000, 0, 0, 1, 700], [20000, 1]])
@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
def test_decode_split_and_joined(pkg, ctx, heads, kv, hd, lens):
    check_decode(pkg, ctx, heads, kv, hd, 64, 64, lens, seed=3)


def test_decode_many_sequences(pkg, ctx):
    """More sequences than threads in a block, most of them short."""
    rng = np.random.default_rng(4)
    check_decode(pkg, ctx, 14, 2, 64, 16, 16, [int(n) for n in rng.integers(0, 40, 300)], seed=4)


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
def test_decode_scales_of_many_sizes(pkg, ctx, heads, kv, hd):
    """Blocks whose scales differ by orders of magnitude: exp(N(0, 3)), so |log2 scale| up to about 20: twice the bar's share
    of the logarithm; scores are up to e^9 larger, and capped for that."""
    check_decode(pkg, ctx, heads, kv, hd, 32, 16, [300, 17, 64], cap=10.0, seed=9, spread=3.0)


def test_decode_extreme_scales(pkg, ctx):
    """V scales at both ends of their range, all alike: log2 off by 60 * 2^-24, 2.5e-6 of a weight, alike for all."""
    rng = np.random.default_rng(10)
    heads, kv, hd = 8, 2, 128
    for size in (2.0 ** 60, 2.0 ** -60):
        c = Cache(pkg, rng, [150], kv, hd, 16, 16)
        for t in range(10):
            c.hs[1][c.table[0, t]] = size
        c.upload(pkg)
        q = rng.normal(0, 1, (1, heads, hd)).astype(np.float32)
        got = run_decode(pkg, ctx, c, q, heads)
        K, V = c.seq(0)
        want = attend(q, K, V, np.array([149]), np.ones((1, 150), bool), 1 / math.sqrt(hd))
        assert rel(got.astype(np.float64) / size, want / size) < ATTN_BAR


def test_decode_blocks_of_zeros(pkg, ctx):
    """Blocks of scale 0 weigh in with values of 0 (their codes are 0, as append leaves them)."""
    rng = np.random.default_rng(11)
    heads, kv, hd = 8, 2, 64
    c = Cache(pkg, rng, [100, 30], kv, hd, 16, 16)
    for s, b in ((0, 1), (0, 4), (1, 0), (1, 1)):
        for t in range(2):
            c.hs[t][c.table[s, b]] = 0
            c.hc[t][c.table[s, b]] = 0
    c.upload(pkg)
    q = rng.normal(0, 1.5, (2, heads, hd)).astype(np.float32)
    got = run_decode(pkg, ctx, c, q, heads)
    K, V = c.seq(0)
    want = attend(q[:1], K, V, np.array([99]), np.ones((1, 100), bool), 1 / math.sqrt(hd))
    assert rel(got[0], want[0]) < ATTN_BAR
    assert not got[1].any()


@pytest.mark.parametrize("which,value", [(0, np.nan), (0, np.inf), (0, -1.0), (1, np.nan), (1, np.inf), (1, -1.0), (1, 2e18)])
def test_scales_that_are_no_numbers_are_seen(pkg, ctx, which, value):
    """The heads that read such a block are NaN, the others are not; nor is a sequence or a row that does not see it."""
    rng = np.random.default_rng(12)
    heads, kv, hd = 8, 2, 128
    c = Cache(pkg, rng, [100, 60], kv, hd, 16, 16)
    c.hs[which][c.table[0, 2], 1] = value     # positions 32 .. 47 of KV head 1
    c.upload(pkg)
    q = rng.normal(0, 1, (2, heads, hd)).astype(np.float32)
    got = run_decode(pkg, ctx, c, q, heads)
    assert np.isnan(got[0, 4:]).all() and np.isfinite(got[0, :4]).all() and np.isfinite(got[1]).all()
    got = run_decode(pkg, ctx, c, q, heads, window=52)   # positions 48 ..
    assert np.isfinite(got).all()
    rows = rng.normal(0, 1, (100, heads, hd)).astype(np.float32)
    qd, out = torch.from_numpy(rows).cuda(), torch.zeros(100, heads, hd, device="cuda")
    cu, ln, cfg = i32([0, 100]), i32([100]), pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=1 / math.sqrt(hd))
    torch.cuda.synchronize()
    ctx.paged_q8_attn_prompt(cfg, c.desc, qd, 1, cu, 100, 100, c.dtable, ln, 100, out)
    ctx.sync()
    got = out.cpu().numpy()
    assert np.isfinite(got[:32]).all() and np.isfinite(got[:, :4]).all() and np.isnan(got[32:, 4:]).all()


@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (8, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("seqs,rows", [(1, 100), (90, 100), (3, 3)])
@pytest.mark.parametrize("cap,slope", [(0.0, 0.7), (20.0, 0.7), (0.0, 3e4), (0.0, 0.0), (20.0, 0.0)])
def test_scales_that_are_no_numbers_are_seen_from_far(pkg, ctx, heads, kv, hd, seqs, rows, cap, slope):
    """A distance bias that leaves nothing of a far block's weights leaves the NaN of its scale; prompts that share their keys
    among CTAs (one sequence), that do not (many), and few rows; a row whose window has passed the block is as without it."""
    rng = np.random.default_rng(33)
    n, group = 700, heads // kv
    c = Cache(pkg, rng, [n], kv, hd, 16, 16)
    c.hs[0][c.table[0, 2], 1] = np.nan        # positions 32 .. 47 of KV head 1
    c.hs[1][c.table[0, 20], 0] = np.inf       # positions 320 .. 335 of KV head 0
    c.upload(pkg)
    table = c.dtable.repeat(seqs, 1).contiguous()
    q, out = torch.randn(seqs * rows, heads, hd, device="cuda"), torch.zeros(seqs * rows, heads, hd, device="cuda")
    cu, ln, sl = i32(np.arange(seqs + 1) * rows), i32([n] * seqs), torch.full((heads,), slope, device="cuda")
    for window in (0, 330, 400):
        cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, window=window, scale=1 / math.sqrt(hd), softcap=cap, slopes=sl.data_ptr())
        out.fill_(7.0)
        torch.cuda.synchronize()
        ctx.paged_q8_attn_prompt(cfg, c.desc, q, seqs, cu, seqs * rows, rows, table, ln, n, out)
        ctx.sync()
        got = out.cpu().numpy().reshape(seqs, rows, heads, hd)
        lo = np.maximum(0, np.arange(n - rows, n) - window + 1) if window else np.zeros(rows, np.int64)
        for h, end in ((0, 336), (1, 48)):
            part = got[:, :, h * group:(h + 1) * group]
            assert np.isnan(part[:, lo < end]).all(), (window, h)
            assert np.isfinite(part[:, lo >= end]).all(), (window, h)


@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (8, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("alibi", [False, True])
def test_prompt_scores_near_the_largest_numbers(pkg, ctx, heads, kv, hd, alibi):
    """A score of 2e38 in units of log2 is a number like others: its value is the row.  All keys but that one are zeros, and its
    product is a power of two times the factor, so that it is exact."""
    rng = np.random.default_rng(34)
    n = 300
    c = Cache(pkg, rng, [n], kv, hd, 16, 16)
    for s in (c.hs[0], c.hc[0]):
        s[c.table[0, :-(-n // 16)]] = 0
    p = c.table[0, 5]                          # position 80: a key of ones
    c.hs[0][p], c.hc[0][p, :, 0] = 1.0, 1
    c.upload(pkg)
    q, sl = torch.ones(n, heads, hd, device="cuda"), torch.full((heads,), 1e-3, device="cuda")
    cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=2e38 / 1.4426950408889634 / hd, slopes=sl.data_ptr() if alibi else None)
    out, cu, ln = torch.zeros(n, heads, hd, device="cuda"), i32([0, n]), i32([n])
    torch.cuda.synchronize()
    ctx.paged_q8_attn_prompt(cfg, c.desc, q, 1, cu, n, n, c.dtable, ln, n, out)
    ctx.sync()
    got, V = out.cpu().numpy(), c.seq(0)[1]
    want = np.broadcast_to(V[80].repeat(heads // kv, 0), (n - 80, heads, hd))
    assert np.isfinite(got).all()
    assert rel(got[80:], want) < ATTN_BAR


def test_decode_extreme_queries(pkg, ctx):
    """Query rows of very small and very large magnitude keep their relative precision."""
    rng = np.random.default_rng(8)
    heads, kv, hd = 8, 2, 128
    c = Cache(pkg, rng, [150], kv, hd, 16, 16)
    q = rng.normal(0, 1, (1, heads, hd)) * 10.0 ** np.arange(-38, -38 + heads)[None, :, None]
    q[0, -1] = 0
    q[0, 0] = rng.normal(0, 1, hd) * 3e3
    q = q.astype(np.float32)
    got = run_decode(pkg, ctx, c, q, heads)
    K, V = c.seq(0)
    want = attend(q, K, V, np.array([149]), np.ones((1, 150), bool), 1 / math.sqrt(hd))
    assert np.isfinite(got).all()
    # head 0's scores reach about 1e4: an f32 score is off by up to 1e4 * 2^-22, and so is its weight
    assert rel(got[0, 1:], want[0, 1:]) < ATTN_BAR
    assert rel(got[0, 0], want[0, 0]) < 1e4 * 2.0 ** -20


def spread_pools(pkg, c, stride):
    """The cache's codes with its pages `stride` bytes apart."""
    pools = []
    for src in c._c:
        t = torch.empty((c.n_pages - 1) * stride + src[0].size, dtype=torch.int8, device="cuda")
        for p in range(c.n_pages):
            t[p * stride:p * stride + src[p].size] = torch.from_numpy(src[p]).cuda().reshape(-1)
        pools.append(t)
    d = pkg.PagedQ8.from_buffer_copy(c.desc)
    d.page_stride, d.slot_stride, d.head_stride = stride, c.hd, c.page * c.hd
    d.k, d.v = (t.data_ptr() for t in pools)
    torch.cuda.synchronize()
    return pools, d


def test_offsets_past_32_bits(pkg, ctx):
    """Pages 2 GiB apart, the pool more than 4 GiB: decode, prompt and append."""
    rng = np.random.default_rng(9)
    heads, kv, hd, page, n = 8, 1, 64, 16, 61
    c = Cache(pkg, rng, [n], kv, hd, page, 16, extra_pages=0)
    pools, c.desc = spread_pools(pkg, c, 2 << 30)
    q = rng.normal(0, 1.5, (1, heads, hd)).astype(np.float32)
    K, V = c.seq(0)
    want = attend(q, K, V, np.array([n - 1]), np.ones((1, n), bool), 1 / math.sqrt(hd))
    assert rel(run_decode(pkg, ctx, c, q, heads), want) < ATTN_BAR
    rows = rng.normal(0, 1.5, (n, heads, hd)).astype(np.float32)
    qd, out = torch.from_numpy(rows).cuda(), torch.zeros(n, heads, hd, device="cuda")
    cu, ln, cfg = i32([0, n]), i32([n]), pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=1 / math.sqrt(hd))
    torch.cuda.synchronize()
    ctx.paged_q8_attn_prompt(cfg, c.desc, qd, 1, cu, n, n, c.dtable, ln, n, out)
    ctx.sync()
    i = np.arange(n)
    assert rel(out.cpu(), attend(rows, K, V, i, i[None] <= i[:, None], 1 / math.sqrt(hd))) < ATTN_BAR
    a = Appends(pkg, ctx, c, rng, heads)
    qkv = rng.normal(0, 2, (n, heads + 2 * kv, hd)).astype(np.float32)
    a.call(qkv, [n], [n])
    w = turned(qkv, heads, kv, np.arange(n), a.theta, a.eps, a.qn, a.kn, False, True)
    for j in (0, 17, 35, 60):
        p = int(c.table[0, j // page])
        for t in range(2):
            code = pools[t][p * (2 << 30) + j % page * hd:][:hd].cpu().numpy().astype(np.float64)
            step = float(c.ds[t][p, 0, 0])
            assert (np.abs(code * step - w[j, heads + t]) <= step * CODE_BAR).all()


def test_decode_same_result_twice_and_in_a_graph(pkg, ctx):
    """No result depends on timing; a captured step follows its device-side lengths."""
    rng = np.random.default_rng(10)
    heads, kv, hd, lens = 32, 4, 128, [2000, 17, 900]
    c = Cache(pkg, rng, lens, kv, hd, 16, 16)
    q = torch.from_numpy(rng.normal(0, 1.5, (3, heads * hd)).astype(np.float32)).cuda()
    cfg = pkg.PagedAttnCfg(n_heads=heads, scale=1 / math.sqrt(hd))
    out, ln = torch.zeros(3, heads * hd, device="cuda"), i32(lens)
    torch.cuda.synchronize()
    seen = []
    for _ in range(5):
        ctx.paged_q8_attn_decode(cfg, c.desc, q, 3, c.dtable, ln, 2000, out)
        ctx.sync()
        seen.append(out.cpu().numpy().copy())
    assert all(np.array_equal(seen[0], x) for x in seen)
    ctx.capture_begin()
    ctx.paged_q8_attn_decode(cfg, c.desc, q, 3, c.dtable, ln, 2000, out)
    g = ctx.capture_end()
    g.launch()
    ctx.sync()
    assert np.array_equal(seen[0], out.cpu().numpy())
    for now in ([1500, 1, 0], [3, 17, 900]):
        ln.copy_(i32(now))
        torch.cuda.synchronize()
        g.launch()
        ctx.sync()
        got = out.cpu().numpy().reshape(3, heads, hd)
        for s, n in enumerate(now):
            K, V = c.seq(s, n)
            want = attend(q[s].cpu().numpy().reshape(1, heads, hd), K, V, np.array([n - 1]), np.ones((1, n), bool), 1 / math.sqrt(hd))
            assert rel(got[s], want[0]) < ATTN_BAR or (n == 0 and not got[s].any())


def test_attention_bad_pages_and_lengths_reported(pkg, ctx):
    rng = np.random.default_rng(11)
    lens = [40, 30]
    c = Cache(pkg, rng, lens, 2, 64, 16, 16)
    heads, hd = 4, 64
    cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=0.125)
    q = torch.ones(2, heads * hd, device="cuda")
    for what in ("page", "length", "length past max_len"):
        for op in ("decode", "prompt"):
            table, ln, out = c.dtable.clone(), i32(lens), torch.zeros(2, heads * hd, device="cuda")
            if what == "page":
                table[0, 1] = c.n_pages
            else:
                ln[0] = 49 if what == "length" else 45
            cu, most = i32([0, 1, 2]), 48 if what == "length" else 44
            torch.cuda.synchronize()
            if op == "decode":
                ctx.paged_q8_attn_decode(cfg, c.desc, q, 2, table, ln, most, out)
            else:
                ctx.paged_q8_attn_prompt(cfg, c.desc, q, 2, cu, 2, 1, table, ln, most, out)
            with pytest.raises(pkg.LtError) as e:
                ctx.sync()
            assert e.value.status == 1
            assert torch.isfinite(out[1]).all() and out[1].abs().sum() > 0
    for cu in ([0, 3, 3], [1, 0, 1], [0, 2, 2]):  # past total_q, descending, more than max_q
        dcu, ln, out = i32(cu), i32(lens), torch.zeros(2, heads * hd, device="cuda")
        torch.cuda.synchronize()
        ctx.paged_q8_attn_prompt(cfg, c.desc, q, 2, dcu, 2, 1, c.dtable, ln, 48, out)
        with pytest.raises(pkg.LtError):
            ctx.sync()
    ctx.sync()


def test_attention_refusals(pkg, ctx):
    rng = np.random.default_rng(13)
    c = Cache(pkg, rng, [40], 2, 64, 32, 16)
    q = torch.zeros(1, 4 * 64, device="cuda")
    ln, cu = i32([40]), i32([0, 1])
    torch.cuda.synchronize()

    def refused(kv=None, cfg=None, max_len=40, n_seq=1, **kw):
        d = pkg.PagedQ8.from_buffer_copy(c.desc)
        for k, v in (kv or {}).items():
            setattr(d, k, v)
        a = pkg.PagedAttnCfg(**{**dict(n_heads=4, scale=0.125), **(cfg or {})})
        for op in ("decode", "prompt"):
            with pytest.raises(pkg.LtError) as e:
                if op == "decode":
                    ctx.paged_q8_attn_decode(a, d, kw.get("q", q), n_seq, c.dtable, ln, max_len, q)
                else:
                    ctx.paged_q8_attn_prompt(a, d, kw.get("q", q), n_seq, cu, 1, 1, c.dtable, ln, max_len, q)
            assert e.value.status == 1 and str(e.value)

    for kv in (dict(head_dim=96), dict(n_kv_heads=0), dict(n_kv_heads=3), dict(page_size=0), dict(page_size=40), dict(block=8), dict(block=48),
               dict(n_pages=0), dict(max_pages=0), dict(slot_stride=64), dict(page_stride=2048, slot_stride=72, head_stride=64),
               dict(k=c.dc[0].data_ptr() + 8), dict(v=None), dict(k_scale=None), dict(v_scale=None)):
        refused(kv=kv)
    for cfg in (dict(n_heads=0), dict(n_heads=5), dict(softcap=-1.0), dict(softcap=float("nan")), dict(scale=float("inf")), dict(q_stride=128),
                dict(out_stride=258)):
        refused(cfg=cfg)
    refused(max_len=0)
    refused(max_len=(1 << 30) + 1)
    refused(n_seq=70000)
    refused(q=q.data_ptr() + 4)
    refused(q=None)
    with pytest.raises(pkg.LtError):  # document numbers must cover max_len
        ctx.paged_q8_attn_prompt(pkg.PagedAttnCfg(n_heads=4, scale=0.125), c.desc, q, 1, cu, 1, 1, c.dtable, ln, 40, q, None, ln, 39)
    ctx.paged_q8_attn_decode(pkg.PagedAttnCfg(n_heads=4, scale=0.125), c.desc, q, 0, c.dtable, ln, 40, q)  # nothing to do
    ctx.sync()


# ── prompts ──────────────────────────────────────────────────────────────────

def check_prompt(pkg, ctx, heads, kv, hd, page, block, new, lens, causal=True, cap=0.0, window=0, alibi=False, prefix=None, docs=None,
                 layout="hnd", seed=0, q_pad=0, spread=0.0):
    rng = np.random.default_rng(seed)
    c = Cache(pkg, rng, lens, kv, hd, page, block, layout, spread=spread)
    total = sum(new)
    q = rng.normal(0, 1.5, (total, heads, hd)).astype(np.float32)
    slopes = slopes_of(heads) if alibi else None
    sl = None if slopes is None else torch.from_numpy(slopes).cuda()
    row = heads * hd + q_pad
    qd = torch.zeros(total, row, device="cuda")
    qd[:, :heads * hd] = torch.from_numpy(q.reshape(total, -1)).cuda()
    out = torch.full((total + 3, row), 7.0, device="cuda")
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
    torch.cuda.synchronize()
    ctx.paged_q8_attn_prompt(cfg, c.desc, qd, len(lens), cu, total, max(new), c.dtable, ln, most, out, pf, dd, most + 1)
    ctx.sync()
    assert (out[total:] == 7.0).all()
    if q_pad:
        assert (out[:, heads * hd:] == 7.0).all()
    got = out[:total, :heads * hd].cpu().numpy().reshape(total, heads, hd)
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
        want[first:first + m] = attend(q[first:first + m], K, V, i[:, 0], seen, 1 / math.sqrt(hd), cap, slopes)
        empty = ~seen.any(1) if n else np.ones(m, bool)
        assert not got[first:first + m][empty].any()
        first += m
    assert np.isfinite(got).all()
    assert rel(got, want) < ATTN_BAR
    return got, want


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("page,block", [(16, 16), (64, 64)])
def test_prompt_causal(pkg, ctx, heads, kv, hd, page, block):
    check_prompt(pkg, ctx, heads, kv, hd, page, block, [1, 3, 130, 0, 17], [1, 40, 130, 9, 200], seed=hd)


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
@pytest.mark.parametrize("page,block", [(48, 16), (32, 32)])
@pytest.mark.parametrize("kw", [
    dict(causal=False), dict(window=1), dict(window=20, alibi=True), dict(cap=20.0, alibi=True),
    dict(prefix=[0, 31, 150]), dict(prefix=[2, 200, 10], window=40), dict(docs=lambda j: j // 23),
    dict(docs=lambda j: j % 3, causal=False), dict(docs=lambda j: j // 50, prefix=[9, 70, 150], cap=30.0, window=60),
    dict(prefix=[0, 0xFFFFFFFF, 7])])
def test_prompt_masks(pkg, ctx, heads, kv, hd, page, block, kw):
    check_prompt(pkg, ctx, heads, kv, hd, page, block, [40, 90, 151], [40, 140, 151], seed=3, **kw)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (8, 2, 256), (2, 2, 64)])
def test_prompt_more_queries_than_positions(pkg, ctx, heads, kv, hd, causal):
    """Queries before position 0 see nothing of a causal cache; an empty cache gives zeros."""
    check_prompt(pkg, ctx, heads, kv, hd, 16, 16, [30, 12, 5], [10, 0, 5], causal=causal, seed=5)


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_prompt_longer(pkg, ctx, heads, kv, hd, cap):
    check_prompt(pkg, ctx, heads, kv, hd, 32, 16, [300, 700], [900, 700], seed=6, layout="nhd", q_pad=8, cap=cap)


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
@pytest.mark.parametrize("page,block,layout", [(16, 16, "nhd"), (48, 16, "hnd"), (64, 32, "nhd"), (128, 128, "hnd"), (192, 64, "hnd"), (256, 16, "nhd")])
def test_prompt_pages(pkg, ctx, heads, kv, hd, page, block, layout):
    """Pages smaller and larger than a tile of keys, in both layouts; windows that begin inside blocks."""
    check_prompt(pkg, ctx, heads, kv, hd, page, block, [70, 150], [333, 150], seed=page, layout=layout)
    check_prompt(pkg, ctx, heads, kv, hd, page, block, [90], [421], seed=page, layout=layout, window=130)


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
def test_prompt_few_rows(pkg, ctx, heads, kv, hd):
    """A few drafted tokens of many sequences on long caches."""
    check_prompt(pkg, ctx, heads, kv, hd, 64, 64, [4, 1, 2, 4, 3], [1000, 77, 2, 333, 3000], seed=7)
    check_prompt(pkg, ctx, heads, kv, hd, 16, 16, [2, 2, 2], [100, 5, 33], seed=8, window=30, cap=20.0, alibi=True)


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
def test_prompt_scales_of_many_sizes(pkg, ctx, heads, kv, hd):
    check_prompt(pkg, ctx, heads, kv, hd, 32, 16, [150, 17], [300, 64], cap=10.0, seed=9, spread=3.0)
    check_prompt(pkg, ctx, heads, kv, hd, 32, 32, [150, 17], [300, 64], cap=10.0, seed=9, spread=3.0, docs=lambda j: j // 40)


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
@pytest.mark.parametrize("largest", [300, 13, 10, 5])
def test_smaller_calls_need_no_more_scratch(pkg, heads, kv, hd, largest):
    """Each op run once with its largest sizes, then recorded with smaller ones: fewer rows, or shorter caches, go to another
    kernel or are shared among more CTAs, and the arena has to hold what either needs.  Each graph is launched, too."""
    rng = np.random.default_rng(25)
    S, n, most = 9, 250, 4096
    c = Cache(pkg, rng, [n] * S, kv, hd, 16, 16, spare=most // 16)
    cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=1 / math.sqrt(hd))
    q, out, ln = torch.randn(S * 300, heads * hd, device="cuda"), torch.zeros(S * 300, heads * hd, device="cuda"), i32([n] * S)
    ms = [m for m in (300, 64, 13, 10, 9, 5, 3, 1) if m <= largest]
    cus = {(s, m): i32(np.arange(s + 1) * m) for s in (S, 3, 1) for m in ms}
    torch.cuda.synchronize()

    def prompt(ctx, s, m, max_len):
        ctx.paged_q8_attn_prompt(cfg, c.desc, q, s, cus[s, m], s * m, m, c.dtable, ln, max_len, out)

    calls = [(s, m, l) for s in (S, 3, 1) for m in ms for l in (n, 600, most)]
    want = []
    with pkg.Context(0) as ctx:
        prompt(ctx, S, largest, most)
        ctx.paged_q8_attn_decode(cfg, c.desc, q, S, c.dtable, ln, most, out)
        ctx.sync()
        for a in calls:
            ctx.capture_begin()
            prompt(ctx, *a)
            ctx.paged_q8_attn_decode(cfg, c.desc, q, a[0], c.dtable, ln, a[2], out)
            ctx.capture_end().free()
            ctx.capture_begin()
            prompt(ctx, *a)
            graph = ctx.capture_end()
            out.zero_()
            torch.cuda.synchronize()
            graph.launch()
            ctx.sync()
            want.append(out.clone())
            graph.free()
    with pkg.Context(0) as ctx:  # and they compute what they do without a graph
        for a, w in zip(calls, want):
            out.zero_()
            torch.cuda.synchronize()
            prompt(ctx, *a)
            ctx.sync()
            assert torch.equal(out, w), a


@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
@pytest.mark.parametrize("scale", [-0.1, 0.0])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_scale_of_any_sign(pkg, ctx, heads, kv, hd, scale, cap):
    """A scale below zero turns the scores round, 0 makes all weights alike; a block of zeros for keys among the others."""
    rng = np.random.default_rng(24)
    n = 150
    c = Cache(pkg, rng, [n], kv, hd, 16, 16)
    c.hs[0][c.table[0, 3]] = 0.0
    c.upload(pkg)
    K, V = c.seq(0)
    rows = rng.normal(0, 1.0, (n, heads, hd)).astype(np.float32)
    qd, out, one = torch.from_numpy(rows).cuda(), torch.zeros(n, heads, hd, device="cuda"), torch.zeros(1, heads, hd, device="cuda")
    cu, ln, cfg = i32([0, n]), i32([n]), pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=scale, softcap=cap)
    torch.cuda.synchronize()
    ctx.paged_q8_attn_prompt(cfg, c.desc, qd, 1, cu, n, n, c.dtable, ln, n, out)
    ctx.paged_q8_attn_decode(cfg, c.desc, qd[n - 1:], 1, c.dtable, ln, n, one)
    ctx.sync()
    i = np.arange(n)
    want = attend(rows, K, V, i, i[None] <= i[:, None], scale, cap)
    assert rel(out.cpu(), want) < ATTN_BAR
    assert rel(one.cpu(), want[n - 1:]) < ATTN_BAR


def test_most_sequences(pkg, ctx):
    """65535 sequences of one position each: appended, then attended to by one query (its result is the value), as single
    tokens and as rows."""
    rng = np.random.default_rng(22)
    S, heads, kv, hd, page = 65535, 2, 1, 64, 16
    codes = torch.zeros(2, S, kv, page, hd, dtype=torch.int8, device="cuda")
    scales = torch.full((2, S, kv, 1), float("nan"), device="cuda")
    desc = pkg.PagedQ8(n_kv_heads=kv, head_dim=hd, page_size=page, block=16, n_pages=S, max_pages=1, k=codes[0].data_ptr(),
                       v=codes[1].data_ptr(), k_scale=scales[0].data_ptr(), v_scale=scales[1].data_ptr())
    cfg = pkg.AttnCfg(n_heads=heads, n_kv_heads=kv, head_dim=hd, rope_neox=1, rope_theta=1e5, eps=1e-6, scale=1.0, kv_cap=1)
    acfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=0.125)
    x = torch.from_numpy(rng.normal(0, 1, (S, heads + 2 * kv, hd)).astype(np.float32)).cuda()
    order = rng.permutation(S)
    table, lens, cu = i32(order), i32(np.ones(S)), i32(np.arange(S + 1))
    q, one, rows = (torch.full((S, heads, hd), 7.0, device="cuda") for _ in range(3))
    torch.cuda.synchronize()
    ctx.paged_q8_append(cfg, desc, x, S, cu, S, 1, None, None, None, table, lens, q)
    ctx.paged_q8_attn_decode(acfg, desc, q, S, table, lens, 1, one)
    ctx.paged_q8_attn_prompt(acfg, desc, q, S, cu, S, 1, table, lens, 1, rows)
    ctx.sync()
    at = torch.from_numpy(order).cuda()
    held = codes[1, at, 0, 0].double() * scales[1, at, 0].double()
    v = x[:, heads + kv].double()
    assert ((held - v).abs() <= scales[1, at, 0].double() * CODE_BAR).all()
    for got in (one, rows):
        # one weight over itself: the scale's inverse, 1 / l and the product are off by 2^-23 each at most, times two
        assert ((got.double() - held[:, None]).abs() <= held[:, None].abs() * 2.0 ** -20).all()


def test_two_contexts_at_once(pkg, ctx):
    """A second context on a stream of its own, both with decode and prompt calls in flight: workspaces are a context's."""
    rng = np.random.default_rng(23)
    heads, kv, hd, lens = 32, 4, 128, [3000, 17, 900, 2500]
    other, streams = pkg.Context(0), [torch.cuda.Stream() for _ in range(2)]
    other.set_stream(streams[1])
    ctx.set_stream(streams[0])
    try:
        sides = []
        for k, c0 in enumerate((ctx, other)):
            c = Cache(pkg, rng, lens, kv, hd, 16, 16)
            n = sum(min(x, 200) for x in lens)
            cu = np.concatenate([[0], np.cumsum([min(x, 200) for x in lens])])
            q, o = torch.from_numpy(rng.normal(0, 1.5, (n, heads, hd)).astype(np.float32)).cuda(), torch.zeros(n, heads, hd, device="cuda")
            sides.append((c0, c, q, o, torch.zeros(4, heads, hd, device="cuda"), i32(cu), i32(lens), n))
        cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=1 / math.sqrt(hd))

        def calls(side):
            c0, c, q, o, d, cu, ln, n = side
            c0.paged_q8_attn_decode(cfg, c.desc, q, 4, c.dtable, ln, 3000, d)
            c0.paged_q8_attn_prompt(cfg, c.desc, q, 4, cu, n, 200, c.dtable, ln, 3000, o)

        alone = []
        for side in sides:
            torch.cuda.synchronize()
            calls(side)
            torch.cuda.synchronize()
            alone.append((side[3].clone(), side[4].clone()))
            side[3].zero_()
            side[4].zero_()
        torch.cuda.synchronize()
        for _ in range(30):
            for side in sides:
                calls(side)
        torch.cuda.synchronize()
        for side, (o, d) in zip(sides, alone):
            assert torch.equal(side[3], o) and torch.equal(side[4], d) and o.any() and d.any()
            side[0].sync()
    finally:
        ctx.set_stream(None)
        other.close()


# ── together ─────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("heads,kv,hd", SHAPES[:3])
def test_plan_append_attend(pkg, ctx, heads, kv, hd):
    """A batch served step by step from one pool: prompts, single tokens, a draft cut back, a sequence ended and its pages
    taken over by another; every step recorded in a graph once and replayed, against attention over the values themselves."""
    rng = np.random.default_rng(21)
    page = block = 16
    S, n_pages, width, most, room = 3, 24, 10, 160, 64
    c = Cache(pkg, rng, [0] * S, kv, hd, page, block, extra_pages=n_pages, spare=width - 1)
    lens, table = torch.zeros(S, dtype=torch.int32, device="cuda"), i32(np.full((S, width), 0xFFFFFFFF))
    free, n_free = i32(np.arange(n_pages)), i32([n_pages])
    state = pkg.PagedState(n_seq=S, page_size=page, n_pages=n_pages, max_pages=width, lens=lens.data_ptr(), page_table=table.data_ptr(),
                           free=free.data_ptr(), n_free=n_free.data_ptr())
    cfg = pkg.AttnCfg(n_heads=heads, n_kv_heads=kv, head_dim=hd, rope_neox=1, rope_theta=1e5, eps=1e-6, scale=1.0, kv_cap=1)
    acfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=1 / math.sqrt(hd))
    keep, new, cu = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (S, S, S + 1))
    qkv, q, out = (torch.zeros(room, w, device="cuda") for w in ((heads + 2 * kv) * hd, heads * hd, heads * hd))
    torch.cuda.synchronize()

    def step():
        ctx.paged_plan(state, keep, new, room, cu)
        ctx.paged_q8_append(cfg, c.desc, qkv, S, cu, room, room, None, None, None, table, lens, q)
        ctx.paged_q8_attn_prompt(acfg, c.desc, q, S, cu, room, room, table, lens, most, out)

    step()
    ctx.sync()
    ctx.capture_begin()
    step()
    g = ctx.capture_end()
    rows = [np.zeros((0, heads + 2 * kv, hd)) for _ in range(S)]
    steps = [([0, 0, 0], [20, 1, 0]), ([20, 1, 0], [1, 1, 33]), ([21, 2, 33], [4, 4, 4]), ([23, 2, 37], [1, 1, 1]), ([24, 0, 38], [1, 50, 1]),
             ([25, 50, 10], [1, 1, 40]), ([0, 51, 50], [30, 1, 1])]
    for k, n in steps:
        x = rng.normal(0, 1.5, (sum(n), heads + 2 * kv, hd)).astype(np.float32)
        keep.copy_(i32(k))
        new.copy_(i32(n))
        qkv[:sum(n)] = torch.from_numpy(x.reshape(sum(n), -1)).cuda()
        out.fill_(7.0)
        torch.cuda.synchronize()
        g.launch()
        ctx.sync()
        got, at = out.cpu().numpy(), 0
        assert (got[sum(n):] == 7.0).all()
        for s in range(S):
            rows[s] = np.concatenate([rows[s][:k[s]], x[at:at + n[s]]])
            L = k[s] + n[s]
            y = turned(rows[s], heads, kv, np.arange(L), 1e5, 1e-6, None, None, False, True)
            i = np.arange(k[s], L)
            want = attend(y[k[s]:, :heads], y[:, heads:heads + kv], y[:, heads + kv:], i, np.arange(L)[None] <= i[:, None], 1 / math.sqrt(hd))
            have = got[at:at + n[s]].reshape(n[s], heads, hd)
            # Values are off by up to a step or two (re-rounded codes) of max / 127 each: relative to values of about max / 3.5,
            # 3.5 / 127 / sqrt(12) = 0.008 per rounding in V; scores of deviation 1.5^2 = 2.25 from K as much, 0.018: 3 %.
            if n[s]:
                assert rel(have, want) < 0.05
            at += n[s]

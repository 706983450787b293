"""Paged attention and eviction where numbers get large, small or strange: positions past 2^24, prefixes past 2^31,
budgets without a limit, scales of zero and below, capped scores over their whole range, sums that are not finite.

Bars as in test_gpu_paged.py unless a test derives its own."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_gpu_paged import ATTN_BAR, Cache, attend, check_prompt, evict_ref, i32, rel

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).cuda()


# ── positions ────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [[4, 3], [60, 40]])
@pytest.mark.parametrize("window", [0, 30])
def test_prefix_past_31_bits(pkg, ctx, f16, new, window):
    """A prefix longer than any sequence: everything cached is seen in both directions."""
    for prefix in ([0xFFFFFFFF, 1 << 31], [(1 << 31) - 1, (1 << 31) + 50]):
        check_prompt(pkg, ctx, 8, 2, 64, f16, 16, new, [100, 90], prefix=prefix, window=window, seed=1)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("m", [0, 1, 5, 40])
def test_distances_past_24_bits(pkg, ctx, f16, m):
    """The distance bias of a window near position 2^25 (m = 0: decode, else m rows of a prompt): differences of
    positions are exact, whatever the positions."""
    rng = np.random.default_rng(2)
    heads, kv, hd, page, window = 8, 2, 64, 1 << 12, 24
    n = (1 << 25) + 5
    width = -(-n // page)
    near = window + max(m, 1)  # positions that any query sees, and one
    K, V = (rng.normal(0, 1, (near, kv, hd)).astype(np.float16) for _ in range(2))
    pools = [torch.zeros(2, page, kv, hd, dtype=torch.float16 if f16 else torch.float32, device="cuda") for _ in range(2)]
    table = np.full((1, width), 0xFFFFFFFF, np.int64)  # the pages before the window are gone
    table[0, -2:] = [1, 0]
    j = np.arange(n - near, n)
    for pool, x in zip(pools, (K, V)):
        pool[table[0, j // page], j % page] = torch.from_numpy(x).cuda().to(pool.dtype)
    desc = pkg.PagedKV(n_kv_heads=kv, head_dim=hd, kv_f16=int(f16), page_size=page, n_pages=2, max_pages=width,
                       k=pools[0].data_ptr(), v=pools[1].data_ptr())
    slopes = (2.0 ** -np.arange(heads)).astype(np.float32)
    sl = dev(slopes)
    cfg = pkg.PagedAttnCfg(n_heads=heads, window=window, causal=1, scale=1 / math.sqrt(hd), slopes=sl.data_ptr())
    rows = max(m, 1)
    q = rng.normal(0, 1.5, (rows, heads, hd)).astype(np.float32)
    qd, out, dt, ln = dev(q), torch.zeros(rows, heads * hd, device="cuda"), i32(table), i32([n])
    cu = i32([0, rows])
    torch.cuda.synchronize()
    if m == 0:
        ctx.paged_attn_decode(cfg, desc, qd, 1, dt, ln, n, out)
    else:
        ctx.paged_attn_prompt(cfg, desc, qd, 1, cu, m, m, dt, ln, n, out)
    ctx.sync()
    i = np.arange(n - rows, n)
    seen = (j[None] <= i[:, None]) & (i[:, None] - j[None] < window)
    want, _ = attend(q, K.astype(np.float64), V.astype(np.float64), i - (n - near), seen, 1 / math.sqrt(hd), slopes=slopes)
    assert rel(out.cpu().numpy().reshape(want.shape), want) < ATTN_BAR


# ── scores ───────────────────────────────────────────────────────────────────

def run_scaled(pkg, ctx, heads, kv, hd, f16, n, m, scale, q, cap=0.0, seed=0, layout_page=16):
    """Decode (m = 0) or a causal prompt of m rows over n positions; got, want."""
    rng = np.random.default_rng(seed)
    c = Cache(pkg, rng, [n], kv, hd, f16, layout_page)
    rows = max(m, 1)
    q = np.asarray(q(rng, (rows, heads, hd)), np.float32)
    cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=scale, softcap=cap)
    qd, out, ln, cu = dev(q), torch.zeros(rows, heads * hd, device="cuda"), i32([n]), i32([0, rows])
    torch.cuda.synchronize()
    if m == 0:
        ctx.paged_attn_decode(cfg, c.desc, qd, 1, c.dtable, ln, n, out)
    else:
        ctx.paged_attn_prompt(cfg, c.desc, qd, 1, cu, m, m, c.dtable, ln, n, out)
    ctx.sync()
    K, V = c.seq(0)
    i = np.arange(n - rows, n)
    # the scale as the call takes it, in 32 bits
    want, _ = attend(q, K, V, i, np.arange(n)[None] <= i[:, None], float(np.float32(scale)), cap)
    return out.cpu().numpy().reshape(want.shape), want


SHAPES = [(14, 2, 64), (32, 4, 128), (16, 8, 256)]


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("m", [0, 2, 150])
@pytest.mark.parametrize("scale,size,cap", [(0.0, 1.5, 0.0), (-0.125, 1.5, 0.0), (-0.125, 1.5, 2.0), (0.0, 1.5, 2.0),
                                            (1e-30, 1e-20, 0.0), (1e-38, 1e-38, 0.0), (1e20, 1e-20, 0.0)])
def test_scales(pkg, ctx, heads, kv, hd, f16, m, scale, size, cap):
    got, want = run_scaled(pkg, ctx, heads, kv, hd, f16, 200, m, scale, lambda r, sh: r.normal(0, size, sh), cap, seed=hd)
    assert np.isfinite(got).all()
    assert rel(got, want) < ATTN_BAR


def prompt_ms(pkg, ctx, hd, scale, size):
    """Shortest of three causal prompts of 1024 tokens over an f16 cache, in ms."""
    heads, kv, n = 8, 2, 1024
    c = Cache(pkg, np.random.default_rng(3), [n], kv, hd, True, 128)
    cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=scale)
    q, out = torch.randn(n, heads * hd, device="cuda") * size, torch.zeros(n, heads * hd, device="cuda")
    ln, cu = i32([n]), i32([0, n])
    torch.cuda.synchronize()
    ctx.profile(True)
    best = []
    for _ in range(3):
        ctx.profile_reset()
        ctx.paged_attn_prompt(cfg, c.desc, q, 1, cu, n, n, c.dtable, ln, n, out)
        ctx.sync()
        best.append(sum(r["total_ms"] for r in ctx.profile_read().values()))
    ctx.profile(False)
    ctx.profile_reset()
    return min(best)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_scores_of_zero_take_no_longer(pkg, ctx, hd):
    """Rows without finite results are done again one by one, hundreds of times slower; scores of zero are finite."""
    usual = prompt_ms(pkg, ctx, hd, 0.125, 1.0)
    for scale, size in ((0.0, 1.0), (1e-38, 1e-38), (0.125, 0.0)):
        assert prompt_ms(pkg, ctx, hd, scale, size) < 5 * usual


def test_weights_of_a_row_that_is_not_finite(pkg, ctx):
    """A score that overflows makes the row's output NaN, and NaN is what it adds to every position that it sees."""
    heads, kv, hd, n = 4, 2, 64, 90
    rng = np.random.default_rng(5)
    c = Cache(pkg, rng, [n, n], kv, hd, False, 16)
    c.hk[c.table[0, 1], 4, 0, 7] = 1e30  # position 20 of the first sequence, KV head 0
    c.upload(pkg)
    q = rng.normal(0, 1, (2, heads, hd)).astype(np.float32)
    q[0, 1, 7] = 1e30
    cfg = pkg.PagedAttnCfg(n_heads=heads, window=80, scale=0.125)
    qd, out, ln = dev(q), torch.zeros(2, heads * hd, device="cuda"), i32([n, n])
    mass = torch.zeros(2, kv, n, device="cuda")
    torch.cuda.synchronize()
    ctx.paged_attn_decode(cfg, c.desc, qd, 2, c.dtable, ln, n, out, mass, n)
    ctx.sync()
    got, m = out.cpu().numpy().reshape(2, heads, hd), mass.cpu().numpy()
    assert np.isnan(got[0, 1]).any()
    assert np.isnan(m[0, 0, n - 80:]).all() and not m[0, 0, :n - 80].any()
    for s, h in ((0, 1), (1, 0), (1, 1)):  # the others are as they would be
        assert np.isfinite(got[s, 2 * h:2 * h + 2]).all()
        assert m[s, h].sum() == pytest.approx(2.0, rel=1e-5)


# ── eviction ─────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("budget", [0xFFFFFFFF, 1 << 31, 41])
def test_evict_without_a_limit(pkg, ctx, in_place, budget):
    """A budget past every length keeps everything, and needs no room for more."""
    rng = np.random.default_rng(7)
    kv, hd, lens = 16, 64, [40, 0, 17]
    c = Cache(pkg, rng, lens, kv, hd, True, 16, extra_pages=6)
    mass = rng.uniform(0, 1, (3, kv, 40)).astype(np.float32)
    dm, ln, out, lens_out = dev(mass), i32(lens), torch.zeros(3, kv, 40, device="cuda"), i32([9, 9, 9])
    dst = np.full_like(c.table, 0xFFFFFFFF)
    dst[0, :3], dst[2, :2] = c.free[:3], c.free[3:5]
    dd = i32(dst)
    torch.cuda.synchronize()
    ctx.kv_evict(c.desc, 3, c.dtable, ln, 40, dm, 40, budget, 5, None if in_place else dd, lens_out, out, 40)
    ctx.sync()
    assert lens_out.tolist() == lens
    gk = c.dk.cpu().numpy()
    for s, n in enumerate(lens):
        assert np.array_equal(out[s, :, :n].cpu().numpy(), mass[s, :, :n])
        j = np.arange(n)
        t = c.table if in_place else dst
        assert np.array_equal(gk[t[s, j // 16], j % 16], c.hk[c.table[s, j // 16], j % 16])

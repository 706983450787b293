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


def prompt_ms(pkg, ctx, hd, scale, size, spoil=None):
    """Shortest of three causal prompts of 1024 tokens over an f16 cache, in ms."""
    heads, kv, n = 8, 2, 1024
    c = Cache(pkg, np.random.default_rng(3), [n], kv, hd, True, 128)
    cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=scale)
    q, out = torch.randn(n, heads * hd, device="cuda") * size, torch.zeros(n, heads * hd, device="cuda")
    if spoil:
        spoil(q, c.dk[c.table[0, 0], 0], c.dv[c.table[0, 0], 0])  # the queries, K and V of position 0
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


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_rows_that_are_not_finite_end_soon(pkg, ctx, hd):
    """A prompt whose rows all come out infinite or NaN, as after an overflow in the model, must not hold the device.

    Every row is done again, 32 of them in turn by a warp.  Where the sum of the weights is NaN a row ends at the key
    that made it so: some five dependent accesses, 3 us, 0.1 ms for 32 rows beside the usual 0.03 to 0.05 ms.  Infinite
    values only: up to 1024 keys at some 80 clocks, 1.4 ms for 32 rows."""
    usual = prompt_ms(pkg, ctx, hd, 0.125, 1.0)
    assert prompt_ms(pkg, ctx, hd, 0.125, 1.0, lambda q, k, v: q.fill_(math.nan)) < 10 * usual
    assert prompt_ms(pkg, ctx, hd, 0.125, 1.0, lambda q, k, v: k.fill_(math.nan)) < 10 * usual
    assert prompt_ms(pkg, ctx, hd, 0.125, 1.0, lambda q, k, v: v[:, 3].fill_(math.inf)) < 60 * usual


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


def test_evict_bad_page_keeps_to_its_own(pkg, ctx):
    """A bad page id of one sequence: reported, the others' slots and the free pages are as they should be."""
    rng = np.random.default_rng(8)
    kv, hd, lens, budget, recent = 2, 64, [90, 90], 40, 8
    c = Cache(pkg, rng, lens, kv, hd, True, 16, extra_pages=3)
    mass = rng.uniform(0, 1, (2, kv, 90)).astype(np.float32)
    good = c.table.copy()
    c.table[0, 1] = 1 << 20
    dm, ln, dt = dev(mass), i32(lens), i32(c.table)
    torch.cuda.synchronize()
    ctx.kv_evict(c.desc, 2, dt, ln, 90, dm, 90, budget, recent, None, ln, dm, 90)
    with pytest.raises(pkg.LtError) as e:
        ctx.sync()
    assert e.value.status == 1
    for got, host in ((c.dk.cpu().numpy(), c.hk), (c.dv.cpu().numpy(), c.hv)):
        for p in [*c.free, good[0, 1]]:
            assert np.array_equal(got[p], host[p], equal_nan=True)
        for h in range(kv):
            keep, i = evict_ref(mass[1, h], 90, budget, recent), np.arange(budget)
            assert np.array_equal(got[good[1, i // 16], i % 16, h], host[good[1, keep // 16], keep % 16, h])
        # beyond the budget nothing of either sequence moved
        for s in (0, 1):
            i = np.arange(48, 90)
            assert np.array_equal(got[good[s, i // 16], i % 16], host[good[s, i // 16], i % 16])
    ctx.sync()


# ── what was not reached before ──────────────────────────────────────────────

@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [[90, 151], [2, 1]])
@pytest.mark.parametrize("cap", [0.05, 1.0, 4.0])
def test_prompt_caps_that_bite(pkg, ctx, heads, kv, hd, f16, new, cap):
    """Scores of standard deviation 1.5 under caps of that size and below: both ranges of the tanh."""
    check_prompt(pkg, ctx, heads, kv, hd, f16, 16, new, [140, 151], cap=cap, alibi=True, seed=4)


@pytest.mark.parametrize("op", ["decode", "prompt"])
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_capped_score_by_itself(pkg, ctx, op, f16, hd):
    """4096 heads with scores c tanh(x), x from -4 to 4, against a score of 0: the two weights' quotient is e^score.

    Error of log(p0 / p1) at a cap c of 10: the tanh 6.1e-8 (relative, below ln(3)/2 where it is at most 1/2) or
    1.5e-7, times c; the score in log2 units and its difference from the maximum, half an ulp of up to 14.4 each, 4.8e-7
    (below: of up to 7.3, 2.4e-7) times ln 2; two exponentials of 2^-22; two weights of 2^-22; x itself to 2^-23 times
    c x (1 - tanh^2) <= 0.45 c; two quotients of 2^-24.  In all 4.4e-6 and 2.6e-6."""
    heads, cap = 4096, 10.0
    x = np.linspace(-4, 4, heads).astype(np.float32)
    pools = [torch.zeros(1, 16, 1, hd, dtype=torch.float16 if f16 else torch.float32, device="cuda") for _ in range(2)]
    pools[0][0, 0, 0, 0] = 1.0          # the first key's score is the query's first element
    pools[1][0, 0, 0, 0] = pools[1][0, 1, 0, 1] = 1.0
    desc = pkg.PagedKV(n_kv_heads=1, head_dim=hd, kv_f16=int(f16), page_size=16, n_pages=1, max_pages=1,
                       k=pools[0].data_ptr(), v=pools[1].data_ptr())
    q = np.zeros((1, heads, hd), np.float32)
    q[0, :, 0] = x * np.float32(cap)
    cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=1.0, softcap=cap)
    qd, out, dt, ln, cu = dev(q), torch.zeros(1, heads * hd, device="cuda"), i32([[0]]), i32([2]), i32([0, 1])
    torch.cuda.synchronize()
    if op == "decode":
        ctx.paged_attn_decode(cfg, desc, qd, 1, dt, ln, 2, out)
    else:
        ctx.paged_attn_prompt(cfg, desc, qd, 1, cu, 1, 1, dt, ln, 2, out)
    ctx.sync()
    p = out.cpu().numpy().reshape(heads, hd).astype(np.float64)
    want = cap * np.tanh(q[0, :, 0].astype(np.float64) / cap)
    off = np.abs(np.log(p[:, 0] / p[:, 1]) - want)
    low = np.abs(x) < 0.549
    assert off[low].max() < 2.6e-6
    assert off.max() < 4.4e-6
    assert not p[:, 2:].any()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("extra", [False, True])
def test_prompts_over_f16_run_on_the_tensor_cores(pkg, ctx, hd, extra):
    """The other kernel gives the same results, many times slower, so a call that went there would not show."""
    heads, kv, n = 8, 2, 300
    c = Cache(pkg, np.random.default_rng(6), [n], kv, hd, True, 16)
    cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=0.125, softcap=30.0 if extra else 0.0)
    q, out, ln, cu = torch.randn(n, heads * hd, device="cuda"), torch.zeros(n, heads * hd, device="cuda"), i32([n]), i32([0, n])
    torch.cuda.synchronize()
    ctx.profile(True)
    ctx.profile_reset()
    ctx.paged_attn_prompt(cfg, c.desc, q, 1, cu, n, n, c.dtable, ln, n, out)
    ctx.sync()
    labels = set(ctx.profile_read())
    ctx.profile(False)
    ctx.profile_reset()
    assert "paged_prompt" in labels and "paged_attn_rows" not in labels

"""Rules on logits (lt_logits_process) against a 64-bit restatement.

Bar: a penalised value goes through at most four f32 roundings of quantities no larger than
max(|x|, |x| rep, |x| / rep, c freq + pres, |bias|), each 2^-24 of it; untouched and masked values are exact.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.as_tensor(np.asarray(v, dtype=np.int64).astype(np.uint32).view(np.int32)).cuda()


def reference(x, rules, history, ids, values, masks):
    """float64 values and the largest magnitude that was rounded on the way."""
    y, big = x.astype(np.float64), np.zeros(x.shape)
    for r, (rep, freq, pres, h0, hn, b0, bn, mask) in enumerate(rules):
        rep, freq, pres = (float(np.float32(v)) for v in (rep, freq, pres))
        h = np.asarray(history[h0:h0 + hn], np.int64)
        tok, c = np.unique(h[h < x.shape[1]], return_counts=True)
        v = y[r, tok]
        with np.errstate(invalid="ignore"):
            w = np.where(v > 0, v / rep, v * rep)
            big[r, tok] = np.abs(w) + np.abs(c * freq) + abs(pres)
            y[r, tok] = w - (c * freq + pres)
        last = {}
        for i in range(b0, b0 + bn):
            if ids[i] < x.shape[1]:
                last[int(ids[i])] = float(values[i])
        for t, b in last.items():
            with np.errstate(invalid="ignore"):
                y[r, t] += b
            big[r, t] += abs(b) + abs(x[r, t])
        if mask is not None:
            bits = np.unpackbits(masks[mask].view(np.uint8), bitorder="little")[:x.shape[1]]
            y[r, bits == 0] = -np.inf
    top = float(np.finfo(np.float32).max)  # past the f32 range a value is infinite
    y[np.isfinite(y) & (np.abs(y) > top)] *= np.inf
    return y, big


def rules_of(pkg, rules):
    a = np.zeros((len(rules), 8), np.uint32)
    for r, v in enumerate(rules):
        a[r, :3] = np.array(v[:3], np.float32).view(np.uint32)
        a[r, 3:7] = v[3:7]
        a[r, 7] = pkg.NO_MASK if v[7] is None else v[7]
    return torch.as_tensor(a.view(np.int32)).cuda()


def check(pkg, ctx, x, rules, history=(), ids=(), values=(), masks=None, in_place=False):
    rows, n = x.shape
    dx = torch.from_numpy(x).cuda()
    out = dx if in_place else torch.full_like(dx, 9.0)
    dr = rules_of(pkg, rules)
    dh = i32(history) if len(history) else None
    di = i32(ids) if len(ids) else None
    dv = torch.as_tensor(np.asarray(values, np.float32)).cuda() if len(ids) else None
    dm = None if masks is None else torch.as_tensor(masks.view(np.int32)).cuda()
    ctx.logits_process(dx, n, rows, dr, dh, di, dv, dm, out)
    ctx.sync()
    got = out.cpu().numpy()
    want, big = reference(x, rules, history, ids, values, masks)
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
    err = np.abs(got[fin] - want[fin])
    assert (err <= big[fin] * 5 * 2.0 ** -24).all()
    assert np.array_equal(got[fin & (big == 0)], x[fin & (big == 0)])
    return got


@pytest.mark.parametrize("n", [1, 31, 32, 33, 4095, 4097, 32003, 151936])
@pytest.mark.parametrize("in_place", [False, True])
def test_rules(pkg, ctx, n, in_place):
    rng = np.random.default_rng(n)
    rows = 5
    x = rng.normal(0, 5, (rows, n)).astype(np.float32)
    history = rng.integers(0, max(1, n // 3), 900)
    history[::50] = n + rng.integers(0, 5)  # padding past the vocabulary
    ids = rng.integers(0, n + 2, 120)
    values = rng.normal(0, 4, 120)
    masks = rng.integers(0, 1 << 32, (3, (n + 31) // 32), dtype=np.uint64).astype(np.uint32)
    masks[2] = 0  # leaves nothing
    rules = [(1.3, 0.2, 0.4, 0, 300, 0, 40, 0), (0.8, 0.0, -0.3, 300, 500, 40, 1, None), (1.0, 0.0, 0.0, 0, 0, 0, 0, 1),
             (1.1, 0.5, 0.0, 800, 100, 41, 79, 2), (2.0, 1.0, 1.0, 0, 900, 0, 120, 1)]
    got = check(pkg, ctx, x, rules, history, ids, values, masks, in_place)
    assert (got[3] == -np.inf).all()


def test_bias_named_twice_last_counts(pkg, ctx):
    x = np.zeros((1, 50), np.float32)
    got = check(pkg, ctx, x, [(1, 0, 0, 0, 0, 0, 6, None)], ids=[7, 8, 7, 7, 49, 8], values=[1, 2, 3, 4, 5, 6])
    assert got[0, 7] == 4 and got[0, 8] == 6 and got[0, 49] == 5


def test_special_values(pkg, ctx):
    x = np.array([[np.inf, -np.inf, np.nan, 0.0, -0.0, 3e38, -3e38, 1.0] * 2], np.float32)
    masks = np.array([[0xFF00]], np.uint32)
    check(pkg, ctx, x, [(1.5, 0.25, 0.5, 0, 16, 0, 0, None)], history=list(range(16)))
    check(pkg, ctx, x, [(1.5, 0.25, 0.5, 0, 16, 0, 0, 0)], history=list(range(16)), masks=masks)
    check(pkg, ctx, x, [(0.5, 0.0, 0.0, 0, 16, 0, 0, None)], history=list(range(16)))


def test_long_history_of_one_token(pkg, ctx):
    x = np.full((1, 40), 2.0, np.float32)
    check(pkg, ctx, x, [(1.2, 0.01, 0.1, 0, 100000, 0, 0, None)], history=np.full(100000, 33))


def test_batch_with_greedy_choice(pkg, ctx):
    """The masked arg-max is the allowed token with the largest logit."""
    rng = np.random.default_rng(3)
    rows, n = 9, 20000
    x = rng.normal(0, 5, (rows, n)).astype(np.float32)
    masks = np.zeros((rows, (n + 31) // 32), np.uint32)
    allowed = [np.sort(rng.choice(n, 12, replace=False)) for _ in range(rows)]
    for r, a in enumerate(allowed):
        np.bitwise_or.at(masks[r], a // 32, (1 << (a % 32)).astype(np.uint32))
    got = check(pkg, ctx, x, [(1, 0, 0, 0, 0, 0, 0, r) for r in range(rows)], masks=masks)
    d, idx = torch.from_numpy(got).cuda(), torch.zeros(rows, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.argmax(d, n, rows, idx)
    ctx.sync()
    assert idx.cpu().tolist() == [int(a[np.argmax(x[r, a])]) for r, a in enumerate(allowed)]


def test_refusals(pkg, ctx):
    x = torch.zeros(1, 8, device="cuda")
    r = rules_of(pkg, [(1, 0, 0, 0, 0, 0, 0, None)])
    for args in ((None, 8, 1, r, None, None, None, None, x), (x, 8, 1, None, None, None, None, None, x),
                 (x, 8, 1, r, None, None, None, None, None), (x, 8, 1, r, None, r, None, None, x), (x, 8, 70000, r, None, None, None, None, x)):
        with pytest.raises(pkg.LtError) as e:
            ctx.logits_process(*args)
        assert e.value.status == 1
    ctx.logits_process(x, 8, 0, r, None, None, None, None, x)
    ctx.logits_process(x, 0, 1, r, None, None, None, None, x)
    ctx.sync()

"""serving.BatchDecoder under a tight budget, call by call: what each layer's eviction keeps and moves, where the next
token's K and V go, what its attention sees and which weights it adds up."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from test_gpu_paged import ATTN_BAR, attend, evict_ref, rel

pytestmark = pytest.mark.gpu


def u32(t, n=None):
    a = t.cpu().numpy().reshape(-1).view(np.uint32).astype(np.int64)
    return a if n is None else a[:n]


class Checked:
    """The context, with the paged calls compared with plain restatements."""

    def __init__(self, ctx, dec):
        self._ctx, self._dec, self.evictions = ctx, dec, 0

    def __getattr__(self, name):
        return getattr(self._ctx, name)

    def _cache(self, kv):
        return next((k, v) for d, k, v in self._dec.caches if d is kv)

    def paged_append(self, cfg, kv, qkv, ntok, qn, kn, seq, pos, slot, *rest):
        if slot is not None:  # one token per sequence
            d = self._dec
            assert u32(pos, ntok).tolist() == [len(t) - 1 for t in d.tokens]       # its place in the text
            assert u32(slot, ntok).tolist() == [n - 1 for n in d.lens]             # its place in the cache
            assert u32(d.dlens, ntok).tolist() == d.lens
        self._ctx.paged_append(cfg, kv, qkv, ntok, qn, kn, seq, pos, slot, *rest)

    def paged_attn_decode(self, cfg, kv, q, n_seq, table, lens, max_len, out, mass, stride):
        self._ctx.sync()
        before = mass.cpu().numpy().astype(np.float64)
        self._ctx.paged_attn_decode(cfg, kv, q, n_seq, table, lens, max_len, out, mass, stride)
        self._ctx.sync()
        after = mass.cpu().numpy().astype(np.float64)
        K, V = (x.float().cpu().numpy().astype(np.float64) for x in self._cache(kv))
        H, nkv, hd, page = cfg.n_heads, kv.n_kv_heads, kv.head_dim, kv.page_size
        T = u32(table).reshape(n_seq, -1)
        qs, got = (t.cpu().numpy().reshape(n_seq, H, hd) for t in (q, out))
        for s, n in enumerate(u32(lens, n_seq)):
            j = np.arange(n)
            at = T[s, j // page], j % page
            want, W = attend(qs[s][None], K[at], V[at], np.array([n - 1]), np.ones((1, n), bool), cfg.scale)
            assert rel(got[s], want[0]) < ATTN_BAR
            assert not before[s, :, n - 1:].any()  # the new position, and those to come, start from nothing
            added = after[s] - before[s]
            # cells of up to the number of steps times the group round to f32 when they are added to
            assert np.abs(added[:, :n] - W[0].reshape(nkv, H // nkv, n).sum(1)).max() < 1e-5 + 2.0 ** -20
            assert not added[:, n:].any()

    def kv_evict(self, kv, n_seq, table, lens, max_len, mass, stride, budget, recent, dst, lens_out, mass_out, ms):
        self._ctx.sync()
        cache = self._cache(kv)
        old = [x.cpu().numpy() for x in cache]
        m0, L = mass.cpu().numpy(), u32(lens, n_seq)
        self._ctx.kv_evict(kv, n_seq, table, lens, max_len, mass, stride, budget, recent, dst, lens_out, mass_out, ms)
        self._ctx.sync()
        new, m1 = [x.cpu().numpy() for x in cache], mass_out.cpu().numpy()
        T, page = u32(table).reshape(n_seq, -1), kv.page_size
        assert u32(lens_out, n_seq).tolist() == np.minimum(L, budget).tolist()
        for s, n in enumerate(L):
            i = np.arange(min(n, budget))
            for h in range(kv.n_kv_heads):
                keep = evict_ref(m0[s, h, :n], n, budget, recent)
                assert np.array_equal(m1[s, h, i], m0[s, h, keep])
                for a, b in zip(old, new):
                    assert np.array_equal(b[T[s, i // page], i % page, h], a[T[s, keep // page], keep % page, h])
                self.evictions += n > budget


@pytest.mark.parametrize("kind,kv_f16", [("dense", True), ("moe", False)])
def test_tight_budget_call_by_call(ctx, kind, kv_f16):
    synth, decoder, serving = (importlib.import_module(f"llmtoy-zig_b200.{m}") for m in ("synth", "decoder", "serving"))
    make = synth.config0_model if kind == "dense" else synth.config2_model
    spec = decoder.upload_decoder(ctx, make(np.random.default_rng(1), n_layers=2, vocab=3000), kv_cap=256, kv_f16=kv_f16)
    dec = serving.BatchDecoder(ctx, spec, max_seqs=3, max_len=96, page_size=8, budget=24, recent=5)
    dec.ctx = Checked(ctx, dec)
    dec.start([[5, 17, 2999], list(range(100, 119)), list(range(40))])  # below the budget, near it, past it
    for _ in range(9):
        dec.step()
        assert max(dec.lens) <= 24 and [len(t) for t in dec.tokens] == [v + 1 for v in dec.pos]
    assert dec.ctx.evictions > 0 and dec.lens == [12, 24, 24]
    dec.close()

"""serving.Q8BatchDecoder: each of its calls against plain restatements on what its cache holds, and its pages."""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from test_gpu_paged_q8 import ATTN_BAR, CODE_BAR, attend, rel, turned

pytestmark = pytest.mark.gpu

PROMPTS = [[5, 17, 2999, 4, 80, 33], [1], list(range(100, 175)), [7, 7, 9]]


def mods():
    return (importlib.import_module(f"llmtoy-zig_b200.{m}") for m in ("synth", "decoder", "serving"))


def spec_of(ctx, kind):
    synth, decoder, serving = mods()
    rng = np.random.default_rng(0)
    m = synth.config0_model(rng, n_layers=2, vocab=3000, qkv_bias=True, norms_random=True) if kind == "dense" else \
        synth.config2_model(rng, n_layers=2, vocab=3000)
    return serving, decoder.upload_decoder(ctx, m, kv_cap=256, kv_f16=True)


def u32(t):
    return t.cpu().numpy().reshape(-1).view(np.uint32).astype(np.int64)


def f32(p):
    """A norm weight, or None."""
    return None if p is None else p.cpu().numpy().astype(np.float64)


class Checked:
    """The context, with the paged calls compared with plain restatements."""

    def __init__(self, ctx, dec):
        self._ctx, self._dec, self.calls = ctx, dec, []

    def __getattr__(self, name):
        return getattr(self._ctx, name)

    def _held(self, kv):
        """Values and scales of the layer's cache: [2][page][head][slot][hd], [2][page][head][block]."""
        codes, scales = next((c, s) for d, c, s in self._dec.caches if d is kv)
        c, s = codes.cpu().numpy().astype(np.float64), scales.cpu().numpy().astype(np.float64)
        return c * np.repeat(s, self._dec.block, 3)[..., None], s

    def paged_plan(self, state, keep, new, total, cu, *rest):
        d = self._dec
        self._ctx.sync()
        had, more = u32(d.dlens), u32(new)
        stay = had if keep is None else u32(keep)
        self._ctx.paged_plan(state, keep, new, total, cu, *rest)
        self._ctx.sync()
        assert u32(d.dlens).tolist() == (stay + more).tolist()
        assert u32(cu).tolist() == np.concatenate([[0], np.cumsum(more)]).tolist()
        rows = u32(d.table).reshape(d.max_seqs, d.width)
        held = [rows[s, :-(-int(n) // d.page)].tolist() for s, n in enumerate(stay + more)]
        flat = [p for r in held for p in r] + u32(d.free)[:u32(d.n_free)[0]].tolist()
        assert sorted(flat) == list(range(d.n_pages))  # every page is held once, or free
        self.calls.append("plan")

    def paged_q8_append(self, cfg, kv, qkv, n_seq, cu, total, most, qn, kn, pos, table, lens, q):
        d, L = self._dec, next(x for x, c in zip(self._dec.spec.layers, self._dec.caches) if c[0] is kv)
        self._ctx.sync()
        self._ctx.paged_q8_append(cfg, kv, qkv, n_seq, cu, total, most, qn, kn, pos, table, lens, q)
        self._ctx.sync()
        H, nkv, hd = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
        first, n, rows = u32(cu), u32(lens), u32(table).reshape(-1, d.width)
        new = first[1:n_seq + 1] - first[:n_seq]
        at = np.concatenate([np.arange(e - m, e) for m, e in zip(new, n)])
        assert int(new.max()) <= most and int(new.sum()) == total
        want = turned(qkv.cpu().numpy().reshape(total, H + 2 * nkv, hd), H, nkv, at, cfg.rope_theta, cfg.eps, f32(L.q_norm), f32(L.k_norm),
                      False, bool(cfg.rope_neox))
        if L.k_norm is None:
            assert L.q_norm is None
        assert rel(q.cpu().numpy().reshape(total, H, hd), want[:, :H]) < 1e-6
        held, scales = self._held(kv)
        seq = np.repeat(np.arange(n_seq), new)
        page, slot = rows[seq, at // d.page], at % d.page
        for t in range(2):
            step = scales[t][page, :, slot // d.block][..., None]
            assert (np.abs(held[t][page, :, slot] - want[:, H + t * nkv:H + (t + 1) * nkv]) <= step * CODE_BAR).all()
        self.calls.append("append")

    def _rows(self, cfg, kv, s, n, table):
        j = np.arange(n)
        held, _ = self._held(kv)
        p = u32(table).reshape(-1, self._dec.width)[s, j // self._dec.page]
        return held[0][p, :, j % self._dec.page], held[1][p, :, j % self._dec.page]

    def paged_q8_attn_decode(self, cfg, kv, q, n_seq, table, lens, max_len, out):
        self._ctx.paged_q8_attn_decode(cfg, kv, q, n_seq, table, lens, max_len, out)
        self._ctx.sync()
        assert u32(lens)[:n_seq].tolist() == self._dec.lens and max_len == max(self._dec.lens)
        qs, got = (t.cpu().numpy().reshape(n_seq, cfg.n_heads, kv.head_dim) for t in (q, out))
        for s, n in enumerate(self._dec.lens):
            K, V = self._rows(cfg, kv, s, n, table)
            assert rel(got[s], attend(qs[s][None], K, V, np.array([n - 1]), np.ones((1, n), bool), cfg.scale)[0]) < ATTN_BAR
        self.calls.append("decode")

    def paged_q8_attn_prompt(self, cfg, kv, q, n_seq, cu, total, most, table, lens, max_len, out, *rest):
        self._ctx.paged_q8_attn_prompt(cfg, kv, q, n_seq, cu, total, most, table, lens, max_len, out, *rest)
        self._ctx.sync()
        first, n = u32(cu), u32(lens)
        qs, got = (t.cpu().numpy().reshape(total, cfg.n_heads, kv.head_dim) for t in (q, out))
        for s in range(n_seq):
            K, V = self._rows(cfg, kv, s, int(n[s]), table)
            m = int(first[s + 1] - first[s])
            i = np.arange(n[s] - m, n[s])
            r = slice(first[s], first[s + 1])
            assert rel(got[r], attend(qs[r], K, V, i, np.arange(n[s])[None] <= i[:, None], cfg.scale)) < ATTN_BAR
        self.calls.append("prompt")


@pytest.mark.parametrize("kind", ["dense", "moe"])
@pytest.mark.parametrize("page,block", [(16, 16), (64, 32)])
def test_every_call(ctx, kind, page, block):
    serving, spec = spec_of(ctx, kind)
    dec = serving.Q8BatchDecoder(ctx, spec, max_seqs=5, max_len=128, page_size=page, block=block)
    plain = dec.generate(PROMPTS, 20)
    dec.ctx = check = Checked(ctx, dec)
    assert dec.generate(PROMPTS, 20) == plain          # and with a restatement beside every call
    assert check.calls.count("plan") == 20 and check.calls.count("append") == 40 and check.calls.count("decode") == 38
    assert dec.generate(PROMPTS[1:3], 3) == [p[:3] for p in plain[1:3]]  # a smaller batch on the same pages


def test_pages_are_counted(ctx):
    serving, spec = spec_of(ctx, "dense")
    dec = serving.Q8BatchDecoder(ctx, spec, max_seqs=2, max_len=64, n_pages=3)
    with pytest.raises(MemoryError):
        dec.start([list(range(1, 40)), list(range(1, 20))])
    first = dec.start([list(range(1, 31)), [3]])
    dec.step()
    dec.step()
    with pytest.raises(MemoryError):  # position 33 of the first needs a fourth page
        dec.step()
    dec.close()
    assert dec.start([list(range(1, 31)), [3]]) == first
    dec.close()


def test_refusals(ctx):
    serving, spec = spec_of(ctx, "dense")
    for page, block in ((16, 8), (24, 16), (16, 32), (0, 16)):
        with pytest.raises(ValueError):
            serving.Q8BatchDecoder(ctx, spec, max_seqs=2, max_len=64, page_size=page, block=block)
    dec = serving.Q8BatchDecoder(ctx, spec, max_seqs=2, max_len=32)
    with pytest.raises(ValueError):
        dec.step()
    with pytest.raises(ValueError):
        dec.start([[3000]])
    with pytest.raises(ValueError):
        dec.start([list(range(32))])

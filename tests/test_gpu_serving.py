"""Batched decoding over a paged cache (serving.BatchDecoder) against the single-sequence decoder.

Both run the same weights through the same matvecs and experts; attention and rotation differ by f32 rounding (f16
caches hold the same rounded values up to a half-ulp of K), so the greedy streams of random models, whose logits are
spread over several units, are the same."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def mods():
    return (importlib.import_module(f"llmtoy-zig_b200.{m}") for m in ("synth", "decoder", "serving"))


def model(synth, kind, seed=0):
    rng = np.random.default_rng(seed)
    if kind == "dense":  # 14/2 heads of 64 with biases
        return synth.config0_model(rng, n_layers=2, vocab=3000)
    return synth.config2_model(rng, n_layers=2, vocab=3000)  # 32/4 heads of 128, MoE


PROMPTS = [[5, 17, 2999, 4, 80, 33], [1], list(range(100, 175)), [7, 7, 9]]


@pytest.mark.parametrize("kind", ["dense", "moe"])
@pytest.mark.parametrize("kv_f16", [False, True])
def test_batch_equals_single_streams(ctx, kind, kv_f16):
    synth, decoder, serving = mods()
    spec = decoder.upload_decoder(ctx, model(synth, kind), kv_cap=256, kv_f16=kv_f16)
    with decoder.Decoder(ctx, spec) as one:
        want = [one.generate(p, 12) for p in PROMPTS]
    batch = serving.BatchDecoder(ctx, spec, max_seqs=4, max_len=256, page_size=16)
    assert batch.generate(PROMPTS, 12) == want
    # pages come back, and a batch of another make-up runs on them
    assert len(batch.pool.free) == batch.n_pages
    assert batch.generate(PROMPTS[2:], 12) == want[2:]


def test_rules_steer_the_stream(ctx):
    synth, decoder, serving = mods()
    spec = decoder.upload_decoder(ctx, model(synth, "dense"), kv_cap=256)
    batch = serving.BatchDecoder(ctx, spec, max_seqs=3, max_len=128)
    allowed = [11, 222, 1333]
    plain = batch.generate([PROMPTS[0]], 8)[0]
    out = batch.generate([serving.Request(PROMPTS[0], allowed=allowed), serving.Request(PROMPTS[0], bias={42: 1e4}),
                          serving.Request(PROMPTS[0], presence=1e6)], 8)
    assert set(out[0]) <= set(allowed)
    assert out[1] == [42] * 8
    assert len(set(out[2])) == 8 and not set(out[2]) & set(PROMPTS[0])
    assert out[2][0] == plain[0] or plain[0] in PROMPTS[0]


def test_budget_keeps_streams_bounded(ctx):
    """A budget above every length changes nothing; a tight one bounds the cache and the pages."""
    synth, decoder, serving = mods()
    spec = decoder.upload_decoder(ctx, model(synth, "moe"), kv_cap=256, kv_f16=True)
    free = serving.BatchDecoder(ctx, spec, max_seqs=4, max_len=128)
    want = free.generate(PROMPTS, 10)
    roomy = serving.BatchDecoder(ctx, spec, max_seqs=4, max_len=128, budget=100, recent=20)
    assert roomy.generate(PROMPTS, 10) == want
    tight = serving.BatchDecoder(ctx, spec, max_seqs=4, max_len=128, budget=40, recent=8)
    tight.start(PROMPTS)
    for _ in range(12):
        tight.step()
        assert max(tight.lens) <= 40
        assert all(len(p) == -(-n // tight.page) for p, n in zip(tight.pages, tight.lens))
    for (_, k, v), m in zip(tight.caches, tight.mass):
        assert bool(k.isfinite().all()) and bool(m.isfinite().all()) and float(m.min()) >= 0
    tight.close()
    assert len(tight.pool.free) == tight.n_pages

"""serving.BatchDecoder between torch's stream and the context's: no torch kernel runs while the context's stream has
work (its operands could come from blocks that this work still uses, and its results go to such blocks), and all work of
torch's has ended before a call launches anything.  A race shows in no output reliably, so the calls are recorded."""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu

ALLOCATE = {"empty", "empty_like", "empty_strided", "detach"}


class Recorder(TorchDispatchMode):
    def __init__(self, log):
        super().__init__()
        self.log = log

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.log.append(("torch", func.overloadpacket.__name__))
        return func(*args, **(kwargs or {}))


class RecordedContext:
    """A context that logs its calls."""

    def __init__(self, ctx, log):
        self._ctx, self._log = ctx, log

    def __getattr__(self, name):
        value = getattr(self._ctx, name)
        if not callable(value):
            return value

        def call(*a, **kw):
            self._log.append(("ctx", name))
            return value(*a, **kw)
        return call


def upload(ctx, kind, **kw):
    synth, decoder = (importlib.import_module(f"llmtoy-zig_b200.{m}") for m in ("synth", "decoder"))
    rng = np.random.default_rng(0)
    m = synth.config0_model(rng, n_layers=2, vocab=3000, qkv_bias=True, norms_random=True) if kind == "biases" else \
        synth.config2_model(rng, n_layers=2, vocab=3000)
    return decoder, decoder.upload_decoder(ctx, m, kv_cap=256, **kw)


@pytest.mark.parametrize("kind,budget", [("biases", 0), ("biases", 20), ("moe", 0)])
def test_no_torch_kernel_beside_the_contexts_work(ctx, monkeypatch, kind, budget):
    serving = importlib.import_module("llmtoy-zig_b200.serving")
    _, spec = upload(ctx, kind)
    assert (spec.layers[0].qkv_bias is not None) == (kind == "biases")
    dec = serving.BatchDecoder(ctx, spec, max_seqs=2, max_len=64, budget=budget, recent=budget // 4)
    log = []
    dec.ctx = RecordedContext(ctx, log)
    wait = torch.cuda.synchronize
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: (log.append(("wait", "device")), wait(*a))[1])
    with Recorder(log):
        dec.start([[5, 6, 7], list(range(30))])
        for _ in range(3):
            log.append(("call", "step"))
            dec.step()
    pending, torch_pending = False, True  # work on the context's stream; of torch's
    for where, name in log:
        if (where, name) == ("call", "step"):
            torch_pending = True  # whatever the caller ran in between
        elif where == "wait":
            pending = torch_pending = False
        elif where == "ctx":
            assert not torch_pending, name
            pending = name not in ("sync", "copy_to_device", "copy_to_host")  # these wait for the stream
        elif name not in ALLOCATE:
            assert not pending, name
            torch_pending = True
    assert not pending and ("ctx", "paged_attn_decode") in log and (not budget or ("ctx", "kv_evict") in log)
    dec.close()


@pytest.mark.parametrize("kv_f16", [False, True])
def test_biases_of_every_token(ctx, kv_f16):
    """A model with Q/K/V biases gives the single-sequence decoder's streams."""
    serving = importlib.import_module("llmtoy-zig_b200.serving")
    decoder, spec = upload(ctx, "biases", kv_f16=kv_f16)
    prompts = [[5, 17, 2999, 4, 80, 33], [1], list(range(100, 175))]
    with decoder.Decoder(ctx, spec) as one:
        want = [one.generate(p, 10) for p in prompts]
    assert serving.BatchDecoder(ctx, spec, max_seqs=3, max_len=128).generate(prompts, 10) == want


def test_biases_at_any_address(ctx):
    """A bias that is a view into something larger, at an odd address or with a stride."""
    serving = importlib.import_module("llmtoy-zig_b200.serving")
    _, spec = upload(ctx, "biases")
    prompts = [[5, 17, 2999], [1]]
    want = serving.BatchDecoder(ctx, spec, max_seqs=2, max_len=32).generate(prompts, 6)
    for i, L in enumerate(spec.layers):
        n = L.qkv_bias.numel()
        room = torch.zeros(2 * n + 1, device="cuda")
        view = room[1:n + 1] if i % 2 == 0 else room[1::2]
        view.copy_(L.qkv_bias)
        assert view.data_ptr() % 16
        L.qkv_bias = view
    torch.cuda.synchronize()
    assert serving.BatchDecoder(ctx, spec, max_seqs=2, max_len=32).generate(prompts, 6) == want

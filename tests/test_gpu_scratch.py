"""The context's scratch arena and recorded graphs: a graph goes on with the addresses it was recorded with, whatever
later ops need, and an op that cannot have its scratch while recording is refused without spoiling the recording."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_gpu_paged import Cache, i32

pytestmark = pytest.mark.gpu

HEADS, KV, HD, N = 8, 2, 128, 300


class Step:
    """A decode step that accumulates weights; its scratch holds HEADS scores per position up to max_len."""

    def __init__(self, pkg, seed=0):
        rng = np.random.default_rng(seed)
        self.cache = Cache(pkg, rng, [N], KV, HD, True, 16)
        self.cfg = pkg.PagedAttnCfg(n_heads=HEADS, scale=1 / math.sqrt(HD))
        self.q = torch.from_numpy(rng.normal(0, 1.5, (1, HEADS * HD)).astype(np.float32)).cuda()
        self.out, self.lens = torch.zeros_like(self.q), i32([N])
        self.mass = torch.zeros(KV << 22, device="cuda")
        torch.cuda.synchronize()

    def __call__(self, ctx, max_len):
        ctx.paged_attn_decode(self.cfg, self.cache.desc, self.q, 1, self.cache.dtable, self.lens, max_len, self.out, self.mass,
                              max_len)

    def result(self):
        torch.cuda.synchronize()
        return self.out.clone(), self.mass[:N].clone()

    def clear(self):
        self.out.zero_()
        self.mass.zero_()
        torch.cuda.synchronize()


def grow(ctx, step):
    """An op with four times the scratch; the bytes that it took from the device."""
    before = torch.cuda.mem_get_info()[0]
    step(ctx, 1 << 22)
    ctx.sync()
    return before - torch.cuda.mem_get_info()[0]


NEW = HEADS * 4 << 22  # bytes of the larger arena at least


def test_graph_outlives_a_larger_arena(pkg):
    step = Step(pkg)
    with pkg.Context(0) as ctx:
        step(ctx, 1 << 20)
        ctx.sync()
        want = step.result()
        ctx.capture_begin()
        step(ctx, 1 << 20)
        graph = ctx.capture_end()
        # the new arena comes on top of the one that the graph writes to
        assert grow(ctx, step) >= NEW
        for _ in range(2):
            step.clear()
            graph.launch()
            ctx.sync()
            assert all(torch.equal(a, b) for a, b in zip(step.result(), want))
        graph.free()


def test_unrecorded_arena_is_given_back(pkg):
    step = Step(pkg)
    with pkg.Context(0) as ctx:
        step(ctx, 1 << 20)
        ctx.sync()
        assert grow(ctx, step) < NEW


def test_graph_recorded_by_the_streams_owner(pkg):
    """torch records the stream that the context runs on."""
    step = Step(pkg)
    with pkg.Context(0) as ctx:
        s = torch.cuda.Stream()
        ctx.set_stream(s)
        step(ctx, 1 << 20)
        ctx.sync()
        want = step.result()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            graph.capture_begin()
            step(ctx, 1 << 20)
            with pytest.raises(pkg.LtError) as e:  # refused, and the recording goes on
                step(ctx, 1 << 22)
            graph.capture_end()
        assert e.value.status == 1
        assert grow(ctx, step) >= NEW
        step.clear()
        with torch.cuda.stream(s):
            graph.replay()
        ctx.sync()
        assert all(torch.equal(a, b) for a, b in zip(step.result(), want))
        del graph
        ctx.set_stream(None)


def test_a_failed_allocation_fails_its_own_call_only(pkg):
    """64 heads' scores at 2^30 positions are more than the device has; the next op is none the worse."""
    rng = np.random.default_rng(9)
    c = Cache(pkg, rng, [40], 2, 64, True, 16)
    q, out, ln = torch.randn(1, 64 * 64, device="cuda"), torch.zeros(1, 64 * 64, device="cuda"), i32([40])
    cfg, mass = pkg.PagedAttnCfg(n_heads=64, scale=0.125), torch.zeros(2 * 40, device="cuda")
    torch.cuda.synchronize()
    with pkg.Context(0) as ctx:
        ctx.paged_attn_decode(cfg, c.desc, q, 1, c.dtable, ln, 40, out)
        ctx.sync()
        want = out.clone()
        for _ in range(2):
            with pytest.raises(pkg.LtError) as e:
                ctx.paged_attn_decode(cfg, c.desc, q, 1, c.dtable, ln, 1 << 30, out, mass, 1 << 30)
            assert e.value.status == 3  # LT_ENOMEM
            out.zero_()
            torch.cuda.synchronize()
            ctx.paged_attn_decode(cfg, c.desc, q, 1, c.dtable, ln, 40, out)
            ctx.sync()
            assert torch.equal(out, want)

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


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (32, 4, 128), (16, 8, 256)])
@pytest.mark.parametrize("f16", [True, False])
def test_smaller_calls_need_no_more_scratch(pkg, heads, kv, hd, f16):
    """Each op run once with its largest sizes, then recorded with smaller ones: fewer rows are shared among more CTAs,
    the fewest go to another kernel, and the arena has to hold what either needs."""
    rng = np.random.default_rng(1)
    n, most = 600, 8192
    c = Cache(pkg, rng, [n] * 3, kv, hd, f16, 16, spare=most // 16)
    cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=1 / math.sqrt(hd))
    q, out = torch.randn(2048, heads * hd, device="cuda"), torch.zeros(2048, heads * hd, device="cuda")
    mass, ln = torch.zeros(3 * kv * most, device="cuda"), i32([n] * 3)
    kept, lens_out = torch.zeros(3 * kv * 512, dtype=torch.int32, device="cuda"), i32([0] * 3)
    cus = {(s, m): i32(np.arange(s + 1) * m) for s in (1, 2, 3) for m in (600, 300, 64, 9, 3, 1)}
    small = torch.zeros(3 * kv * 512, device="cuda")
    torch.cuda.synchronize()

    def prompt(ctx, s, m, max_q, max_len):
        ctx.paged_attn_prompt(cfg, c.desc, q, s, cus[s, m], s * m, max_q, c.dtable, ln, max_len, out)

    with pkg.Context(0) as ctx:
        prompt(ctx, 3, 600, most, most)
        ctx.sync()
        want = []
        calls = [(s, m, k, l) for s in (3, 1) for m in (600, 300, 64, 9, 3, 1) for k in {m, most} for l in (n, 1024, most)]
        for a in calls:
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
    with pkg.Context(0) as ctx:
        ctx.paged_attn_decode(cfg, c.desc, q, 3, c.dtable, ln, most, out, mass, most)
        ctx.kv_evict(c.desc, 3, c.dtable, ln, most, mass, most, 512, 8, None, lens_out, small, 512)
        ctx.sync()
        ctx.capture_begin()
        for s, l in ((3, n), (1, most), (2, 1000)):
            ctx.paged_attn_decode(cfg, c.desc, q, s, c.dtable, ln, l, out, mass, most)
            ctx.paged_attn_decode(cfg, c.desc, q, s, c.dtable, ln, l, out)
            ctx.kv_evict(c.desc, s, c.dtable, ln, l, mass, most, 512, 8, None, lens_out, small, 512)
            ctx.kv_evict(c.desc, s, c.dtable, ln, l, mass, most, 64, 8, None, lens_out, small, 64, kept)
        ctx.capture_end().free()


def test_leaving_a_stream_that_is_gone(pkg):
    """A caller may destroy its stream and then give the context another: the old one is not looked at again."""
    import ctypes
    rt = torch.cuda.cudart()
    step = Step(pkg)
    with pkg.Context(0) as ctx:
        step(ctx, 1 << 10)
        ctx.sync()
        want = step.result()
        handle = ctypes.c_void_p()
        assert int(rt.cudaStreamCreate(ctypes.addressof(handle))) == 0
        ctx.set_stream(handle.value)
        step.clear()
        step(ctx, 1 << 10)
        ctx.sync()
        assert all(torch.equal(a, b) for a, b in zip(step.result(), want))
        assert int(rt.cudaStreamDestroy(handle.value)) == 0
        ctx.set_stream(None)
        step.clear()
        step(ctx, 1 << 10)
        ctx.sync()
        assert all(torch.equal(a, b) for a, b in zip(step.result(), want))


def test_a_recording_asks_only_for_what_its_calls_need(pkg):
    """A long prompt shares no keys and needs no scratch: it can be recorded on a context that has run nothing."""
    rng = np.random.default_rng(3)
    heads, kv, hd, n = 32, 4, 128, 1300
    c = Cache(pkg, rng, [n] * 2, kv, hd, True, 16)
    cfg = pkg.PagedAttnCfg(n_heads=heads, causal=1, scale=1 / math.sqrt(hd))
    q, out = torch.randn(2 * n, heads * hd, device="cuda"), torch.zeros(2 * n, heads * hd, device="cuda")
    cu, ln = i32([0, n, 2 * n]), i32([n, n])
    torch.cuda.synchronize()
    with pkg.Context(0) as ctx:
        ctx.capture_begin()
        ctx.paged_attn_prompt(cfg, c.desc, q, 2, cu, 2 * n, n, c.dtable, ln, n, out)
        graph = ctx.capture_end()
        graph.launch()
        ctx.sync()
        got = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        ctx.paged_attn_prompt(cfg, c.desc, q, 2, cu, 2 * n, n, c.dtable, ln, n, out)  # the arena comes now
        ctx.sync()
        assert torch.equal(out, got) and bool(out.any())
        out.zero_()
        torch.cuda.synchronize()
        graph.launch()
        ctx.sync()
        assert torch.equal(out, got)
        graph.free()

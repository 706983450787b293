"""A context that was given no stream, and torch on its default stream: each sees the other's work in the order of the
calls, without a wait on the host.  The operands are appends to an 8-bit paged cache long enough to be under way still when
the host is back, and read or filled by torch right before and behind the calls."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from test_gpu_paged_q8 import i32

pytestmark = pytest.mark.gpu


class Append:
    """A prompt for a cache of one sequence: `fill` makes the rows from a seed on torch's stream, `read` takes what the
    call left there, queries, codes and scales, on the same stream."""

    def __init__(self, pkg, n=6000, heads=16, kv=8, hd=256, page=32):
        pages = -(-n // page)
        self.n, self.hd, self.heads, self.kv = n, hd, heads, kv
        self.x, self.q = torch.zeros(n, (heads + 2 * kv) * hd, device="cuda"), torch.zeros(n, heads * hd, device="cuda")
        self.codes = torch.zeros(2, pages, kv, page, hd, dtype=torch.int8, device="cuda")
        self.scales = torch.zeros(2, pages, kv, 1, device="cuda")
        self.cu, self.lens, self.table = i32([0, n]), i32([n]), i32(np.random.default_rng(1).permutation(pages))
        self.kv_desc = pkg.PagedQ8(n_kv_heads=kv, head_dim=hd, page_size=page, block=page, n_pages=pages, max_pages=pages,
                                   k=self.codes[0].data_ptr(), v=self.codes[1].data_ptr(), k_scale=self.scales[0].data_ptr(),
                                   v_scale=self.scales[1].data_ptr())
        self.cfg = pkg.AttnCfg(n_heads=heads, n_kv_heads=kv, head_dim=hd, rope_neox=1, rope_theta=1e5, eps=1e-6, scale=1.0, kv_cap=1)
        self.rows = [torch.randn(n, self.x.shape[1], device="cuda", generator=torch.Generator("cuda").manual_seed(s)) for s in range(2)]
        self.values = torch.zeros(self.codes.shape, device="cuda")
        torch.cuda.synchronize()

    def fill(self, s):
        torch.mul(self.rows[s], 2.0, out=self.x)

    def call(self, ctx):
        ctx.paged_q8_append(self.cfg, self.kv_desc, self.x, 1, self.cu, self.n, self.n, None, None, None, self.table, self.lens, self.q)

    def read(self):
        torch.mul(self.codes, self.scales[..., None], out=self.values)
        return self.q.clone(), self.values.clone(), self.scales.clone()


def test_calls_and_torch_take_turns(pkg):
    op = Append(pkg)
    with pkg.Context(0) as ctx:
        want = []
        for s in range(2):
            op.fill(s)
            torch.cuda.synchronize()
            op.call(ctx)
            ctx.sync()
            want.append(op.read())
            torch.cuda.synchronize()
        got = []
        for k in range(12):
            op.fill(k % 2)
            op.call(ctx)
            got.append(op.read())
        torch.cuda.synchronize()
        for k, three in enumerate(got):
            for x, y in zip(three, want[k % 2]):
                assert torch.equal(x, y), k


def test_replays_and_torch_take_turns(pkg):
    """The same of a graph that the context recorded."""
    op = Append(pkg)
    with pkg.Context(0) as ctx:
        op.fill(0)
        op.call(ctx)
        ctx.sync()
        ctx.capture_begin()
        op.call(ctx)
        g = ctx.capture_end()
        want = []
        for s in range(2):
            op.fill(s)
            torch.cuda.synchronize()
            op.call(ctx)
            ctx.sync()
            want.append(op.read())
            torch.cuda.synchronize()
        got = []
        for k in range(12):
            op.fill(k % 2)
            g.launch()
            got.append(op.read())
        torch.cuda.synchronize()
        for k, three in enumerate(got):
            for x, y in zip(three, want[k % 2]):
                assert torch.equal(x, y), k
        g.free()


@pytest.mark.parametrize("default", [False, True])
def test_torch_works_on_while_a_context_records(pkg, default):
    """torch's default stream, used by this thread and by another between the ends of a recording, is not part of it and
    does not break it; a second context works on, too."""
    op, side = Append(pkg, n=200), Append(pkg, n=200)
    with pkg.Context(0) as ctx, pkg.Context(0) as other:
        if default:
            ctx.set_stream(torch.cuda.current_stream())
        op.fill(0)
        op.call(ctx)
        ctx.sync()
        want = op.read()
        torch.cuda.synchronize()
        op.q.zero_()
        done = []

        def elsewhere():
            side.fill(0)
            side.call(other)
            done.append(side.read())
            torch.cuda.current_stream().synchronize()
            other.sync()

        ctx.capture_begin()
        op.call(ctx)
        t = threading.Thread(target=elsewhere)
        t.start()
        t.join()
        y = op.rows[0].sum()
        g = ctx.capture_end()
        torch.cuda.synchronize()
        assert len(done) == 1 and torch.isfinite(y) and not op.q.any()
        assert all(torch.equal(a, b) for a, b in zip(done[0], want))
        g.launch()
        assert torch.equal(op.q, want[0])
        ctx.sync()
        g.free()


def test_streams_changed_while_a_context_records(pkg):
    """The recording goes on and ends; the context is on the new stream then, also where that is the one it was on."""
    op = Append(pkg, n=200)
    with pkg.Context(0) as ctx:
        op.fill(0)
        op.call(ctx)
        ctx.sync()
        want = op.read()
        torch.cuda.synchronize()
        for stream in (None, torch.cuda.current_stream(), None, torch.cuda.Stream(), None):
            op.q.zero_()
            own = pkg.Context(0)
            try:
                own.capture_begin()
                own.set_stream(stream)
                op.call(own)
                g = own.capture_end()
                torch.cuda.synchronize()
                assert not op.q.any()
                g.launch()
                own.sync()
                assert torch.equal(op.q, want[0])
                g.free()
                op.q.zero_()
                torch.cuda.synchronize()
                op.call(own)
                own.sync()
                assert torch.equal(op.q, want[0])
            finally:
                own.close()


def test_a_context_closed_while_it_records(pkg):
    """An open recording ends with its context; the next context is none the worse."""
    op = Append(pkg, n=200)
    with pkg.Context(0) as ctx:
        op.fill(0)
        op.call(ctx)
        ctx.sync()
        want = op.read()
        ctx.capture_begin()
        op.call(ctx)
    with pkg.Context(0) as ctx:
        op.q.zero_()
        op.call(ctx)
        assert torch.equal(op.q, want[0])
        ctx.sync()

"""lt_paged_plan against a plain allocator of lists; every number is exact."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

GONE, MARK = 0xFFFFFFFF, 0xABCD1234


def dev(v):
    return torch.as_tensor(np.asarray(v, dtype=np.int64).astype(np.uint32).view(np.int32)).cuda()


def host(t):
    return t.cpu().numpy().view(np.uint32).astype(np.int64)


class Batch:
    """Lists of pages, as a host would keep them, and the same state on the device."""

    def __init__(self, pkg, rng, lens, page, n_pages, width):
        order = rng.permutation(n_pages).tolist()
        self.page, self.lens, self.width, self.n_pages = page, list(lens), width, n_pages
        self.pages = [[order.pop() for _ in range(-(-n // page))] for n in lens]
        self.free = order
        table = np.full((len(lens), width), GONE, np.int64)
        for s, p in enumerate(self.pages):
            table[s, :len(p)] = p
        self.dlens, self.dtable, self.dn = dev(lens), dev(table), dev([len(order)])
        self.dfree = dev(order + [GONE] * (n_pages - len(order)))
        self.state = pkg.PagedState(n_seq=len(lens), page_size=page, n_pages=n_pages, max_pages=width, lens=self.dlens.data_ptr(),
                                    page_table=self.dtable.data_ptr(), free=self.dfree.data_ptr(), n_free=self.dn.data_ptr())

    def want(self, keep, new):
        """The plain allocator; cu, seq, pos, slot of the coming tokens."""
        stay = [-(-k // self.page) for k in keep]
        for s in reversed(range(len(keep))):
            while len(self.pages[s]) > stay[s]:
                self.free.append(self.pages[s].pop())
        seq, pos, slot = [], [], []
        for s, (k, n) in enumerate(zip(keep, new)):
            while len(self.pages[s]) * self.page < k + n:
                self.pages[s].append(self.free.pop())
            self.lens[s] = k + n
            seq += [s] * n
            pos += range(k, k + n)
            slot += [self.pages[s][p // self.page] * self.page + p % self.page for p in range(k, k + n)]
        return np.concatenate([[0], np.cumsum(new)]), seq, pos, slot

    def run(self, ctx, keep, new, total, extra=3):
        """The call; its four outputs, with marks behind the tokens."""
        cu, seq, pos, slot = (torch.full((n,), MARK - (1 << 32), dtype=torch.int64).int().cuda()
                              for n in (len(new) + 1, total + extra, total + extra, total + extra))
        dkeep = None if keep is None else dev(keep)
        ctx.paged_plan(self.state, dkeep, dev(new), total, cu, seq, pos, slot)
        ctx.sync()
        return [host(t) for t in (cu, seq, pos, slot)]

    def same(self):
        assert host(self.dlens).tolist() == self.lens
        assert host(self.dn).tolist() == [len(self.free)]
        assert host(self.dfree)[:len(self.free)].tolist() == self.free
        table = host(self.dtable)
        for s, p in enumerate(self.pages):
            assert table[s, :len(p)].tolist() == p, s
            assert (table[s, len(p):] == GONE).all(), s


@pytest.mark.parametrize("n_seq,page,top,most", [
    (1, 1, 5, 3), (1, 16, 40, 0), (3, 16, 40, 1), (64, 16, 300, 1), (64, 24, 300, 50), (33, 128, 3000, 700), (1024, 16, 60, 9),
    (1025, 8, 60, 9), (5000, 3, 20, 4), (7, 64, 20000, 20000), (2, 1, 3000, 2500), (65535, 1, 2, 2)])
@pytest.mark.parametrize("room", [0, 5000])
def test_steps(pkg, ctx, n_seq, page, top, most, room):
    """Several steps in a row: grow, cut back, end, start again; with room for few tokens and for many, which take other launches."""
    rng = np.random.default_rng(n_seq * 131 + page)
    lens = rng.integers(0, top + 1, n_seq)
    width = -(-(top + 4 * max(1, most)) // page) + 1
    n_pages = int(sum(-(-n // page) for n in lens) + n_seq * (-(-most // page) + 1) * 4 + 3)
    b = Batch(pkg, rng, [int(n) for n in lens], page, n_pages, width)
    for step in range(4 if n_seq < 10000 else 1):
        keep = [int(n) if rng.random() < 0.6 else int(rng.integers(0, n + 1)) for n in b.lens]
        if step == 2:
            keep = list(b.lens)
        new = [int(x) for x in rng.integers(0, most + 1, n_seq)]
        if step == 3:
            new = [0] * n_seq
        total = sum(new) + int(rng.integers(0, 5)) + room
        got = b.run(ctx, None if step == 2 else keep, new, total)
        want = b.want(keep, new)
        assert got[0].tolist() == want[0].tolist()
        for g, w in zip(got[1:], want[1:]):
            assert g[:len(w)].tolist() == list(w)
            assert (g[len(w):] == MARK).all()
        b.same()


def test_repeat_gives_the_same(pkg, ctx):
    """Drafted tokens cut back and planned again land where they were."""
    b = Batch(pkg, np.random.default_rng(3), [5, 64, 0, 33], 16, 40, 12)
    keep, new = [5, 60, 0, 20], [30, 1, 17, 0]
    first = b.run(ctx, keep, new, 48)
    state = [host(t).copy() for t in (b.dlens, b.dtable, b.dfree, b.dn)]
    again = b.run(ctx, keep, new, 48)
    for x, y in zip(first, again):
        assert (x == y).all()
    for x, t in zip(state, (b.dlens, b.dtable, b.dfree, b.dn)):
        assert (x == host(t)).all()


def test_keep_may_be_the_lengths(pkg, ctx):
    b = Batch(pkg, np.random.default_rng(4), [5, 64, 0], 16, 40, 12)
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    new = dev([3, 0, 40])
    torch.cuda.synchronize()
    ctx.paged_plan(b.state, b.dlens, new, 43, cu)
    ctx.sync()
    b.want([5, 64, 0], [3, 0, 40])
    b.same()


# what is wrong, keep, new, total, pages taken from the stack's count, status
BAD = [("past the table and the pages", [5, 64, 0], [0, 0, 200], 200, 10, 1), ("too few pages", [5, 64, 0], [0, 0, 180], 200, 10, 3), ("keep past the length", [6, 64, 0], [1, 1, 1], 3, 0, 1),
       ("past the table", [5, 64, 0], [0, 129, 0], 129, 0, 1), ("more tokens than room", [5, 64, 0], [3, 3, 3], 8, 0, 1),
       ("a length that wraps", [5, 64, 0], [0xFFFFFFFF, 1, 0], 100, 0, 1)]


@pytest.mark.parametrize("room", [0, 5000])
@pytest.mark.parametrize("what,keep,new,total,less,status", BAD, ids=[b[0] for b in BAD])
def test_refused_plans_change_nothing(pkg, ctx, what, keep, new, total, less, status, room):
    if room and what == "more tokens than room":
        new = [room, 3, 3]
        total = room + 5
        b = Batch(pkg, np.random.default_rng(5), [5, 64, 0], 16, 400, 350)
    else:
        total += room
        b = Batch(pkg, np.random.default_rng(5), [5, 64, 0], 16, 25, 12)
    if less:
        b.dn.sub_(less)
        torch.cuda.synchronize()
    before = [host(t).copy() for t in (b.dlens, b.dtable, b.dfree, b.dn)]
    cu, seq = torch.full((4,), 7, dtype=torch.int32, device="cuda"), torch.full((total + 1,), 7, dtype=torch.int32, device="cuda")
    dkeep, dnew = dev(keep), dev(new)
    torch.cuda.synchronize()
    ctx.paged_plan(b.state, dkeep, dnew, total, cu, seq)
    with pytest.raises(pkg.LtError) as e:
        ctx.sync()
    assert e.value.status == status
    assert host(cu).tolist() == [0] * 4 and (host(seq) == 7).all()
    for x, t in zip(before, (b.dlens, b.dtable, b.dfree, b.dn)):
        assert (x == host(t)).all()
    ctx.sync()  # reported once


@pytest.mark.parametrize("room", [0, 5000])
@pytest.mark.parametrize("what", ["page id", "stack too long", "stack overflows"])
def test_broken_state_is_reported(pkg, ctx, what, room):
    b = Batch(pkg, np.random.default_rng(6), [5, 64, 0], 16, 25, 12)
    if what == "page id":
        b.dtable[1, 3] = 25
    else:
        b.dn.fill_(26 if what == "stack too long" else 24)
    torch.cuda.synchronize()
    before = [host(t).copy() for t in (b.dlens, b.dtable, b.dfree, b.dn)]
    cu = torch.full((4,), 7, dtype=torch.int32, device="cuda")
    keep, new = dev([0, 0, 0] if what == "stack overflows" else [5, 40, 0]), dev([1, 1, 1])
    torch.cuda.synchronize()
    ctx.paged_plan(b.state, keep, new, 3 + room, cu)
    with pytest.raises(pkg.LtError) as e:
        ctx.sync()
    assert e.value.status == 1
    assert host(cu).tolist() == [0] * 4
    for x, t in zip(before, (b.dlens, b.dtable, b.dfree, b.dn)):
        assert (x == host(t)).all()


@pytest.mark.parametrize("room", [0, 5000])
def test_captured_steps(pkg, ctx, room):
    """One captured plan replayed: a token more of every sequence each time."""
    b = Batch(pkg, np.random.default_rng(7), [5, 64, 0, 31], 16, 40, 12)
    one = dev([1, 1, 1, 1])
    cu, seq, pos, slot = (torch.zeros(5 + room, dtype=torch.int32, device="cuda") for _ in range(4))
    torch.cuda.synchronize()
    ctx.paged_plan(b.state, None, one, 4 + room, cu, seq, pos, slot)
    ctx.sync()
    b.want(list(b.lens), [1] * 4)
    ctx.capture_begin()
    ctx.paged_plan(b.state, None, one, 4 + room, cu, seq, pos, slot)
    g = ctx.capture_end()
    for _ in range(20):
        g.launch()
        ctx.sync()
        want = b.want(list(b.lens), [1] * 4)
        b.same()
        assert host(slot)[:4].tolist() == want[3] and host(pos)[:4].tolist() == want[2]


def test_rows_for_an_f16_cache(pkg, ctx):
    """Sequence, position and pool slot as they come, for lt_paged_append: values lie where pool_slot says."""
    rng = np.random.default_rng(11)
    page, kv, hd, heads = 24, 2, 64, 6
    b = Batch(pkg, rng, [0, 50, 7, 24], page, 40, 8)
    new = [33, 1, 0, 25]
    total = sum(new)
    cu, seq, pos, slot = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (len(new) + 1, total, total, total))
    k, v = (torch.zeros(40, page, kv, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    desc = pkg.PagedKV(n_kv_heads=kv, head_dim=hd, kv_f16=1, page_size=page, n_pages=40, max_pages=8, k=k.data_ptr(), v=v.data_ptr())
    cfg = pkg.AttnCfg(n_heads=heads, n_kv_heads=kv, head_dim=hd, rope_neox=1, rope_theta=1e5, eps=1e-6, scale=1.0, kv_cap=1, kv_f16=1)
    x = torch.from_numpy(rng.normal(0, 1, (total, heads + 2 * kv, hd)).astype(np.float32)).cuda()
    q = torch.zeros(total, heads, hd, device="cuda")
    want = b.want([0, 50, 3, 24], new)
    keep, more = dev([0, 50, 3, 24]), dev(new)
    torch.cuda.synchronize()
    ctx.paged_plan(b.state, keep, more, total, cu, seq, pos, slot)
    ctx.paged_append(cfg, desc, x, total, None, None, seq, pos, None, b.dtable, len(new), q)
    ctx.sync()
    for got, w in zip((cu, seq, pos, slot), want):
        assert host(got).tolist() == list(w)
    b.same()
    rows = host(slot)
    assert torch.equal(v.view(-1, kv, hd)[rows], x[:, heads + kv:].half())
    left = np.setdiff1d(np.arange(40 * page), rows)
    assert not v.view(-1, kv, hd)[left].any() and not k.view(-1, kv, hd)[left].any()


@pytest.mark.parametrize("room", [65535, 70000])
def test_most_sequences(pkg, ctx, room):
    """As many sequences as there may be: ends, cuts and growth of each, three steps."""
    rng = np.random.default_rng(12)
    S, page = 65535, 3
    lens = rng.integers(0, 10, S).tolist()
    b = Batch(pkg, rng, lens, page, 4 * S, 8)
    for _ in range(2):
        keep = [int(rng.integers(0, n + 1)) if rng.random() < 0.5 else n for n in b.lens]
        new = [1 if n < 20 else 0 for n in keep]
        want = b.want(keep, new)
        for got, w in zip(b.run(ctx, keep, new, room), want):
            assert got[:len(w)].tolist() == list(w)
            assert (got[len(w):] == MARK).all()
        b.same()


@pytest.mark.parametrize("room", [0, 5000])
@pytest.mark.parametrize("n_seq", [3, 2100])
@pytest.mark.parametrize("what", ["stack", "stack's deepest", "kept page", "kept page behind others that go"])
def test_page_ids_that_a_plan_would_use(pkg, ctx, what, n_seq, room):
    """A page number past the pool is refused wherever the plan would make a table entry or a slot of it: among the pages to
    be taken, and on the page that a sequence goes on with.  Where the plan has no use for it, it is nobody's business."""
    b = Batch(pkg, np.random.default_rng(13), [5, 64, 0] + [9] * (n_seq - 3), 16, n_seq + 30, 12)
    keep, new = [5, 64, 0] + [9] * (n_seq - 3), [20, 33, 1] + [1] * (n_seq - 3)   # takes 1 + 3 + 1 pages
    n = len(b.free)
    if what == "stack":
        at = b.dfree[n - 2:n - 1]
    elif what == "stack's deepest":
        at = b.dfree[n - 5:n - 4]
    elif what == "kept page":
        at = b.dtable[n_seq - 1 if n_seq > 3 else 0, 0:1]
    else:
        keep[1] = 33                                           # a page goes, the one before it holds one position of 16
        at = b.dtable[1, 2:3]
    good = at.clone()
    at.fill_(b.n_pages)
    torch.cuda.synchronize()
    before = [host(t).copy() for t in (b.dlens, b.dtable, b.dfree, b.dn)]
    total = sum(new) + room
    cu, seq, pos, slot = (torch.full((m,), 7, dtype=torch.int32, device="cuda") for m in (n_seq + 1, total, total, total))
    dkeep, dnew = dev(keep), dev(new)
    torch.cuda.synchronize()
    ctx.paged_plan(b.state, dkeep, dnew, total, cu, seq, pos, slot)
    with pytest.raises(pkg.LtError) as e:
        ctx.sync()
    assert e.value.status == 1
    assert not host(cu).any()
    assert all((host(t) == 7).all() for t in (seq, pos, slot))
    for x, t in zip(before, (b.dlens, b.dtable, b.dfree, b.dn)):
        assert (x == host(t)).all()
    # the same page number where this plan does not look
    at.copy_(good)
    b.dfree[0] = b.n_pages                                     # deeper in the stack than what is taken
    b.dtable[1, 0] = b.n_pages                                 # a page that stays and gets nothing
    torch.cuda.synchronize()
    got = b.run(ctx, keep, new, total)
    b.free[0] = b.n_pages
    b.pages[1][0] = b.n_pages
    for g, w in zip(got, b.want(keep, new)):
        assert g[:len(w)].tolist() == list(w)
    b.same()


def test_no_sequences(pkg, ctx):
    """The running sums of nothing: one 0, recorded or not."""
    b = Batch(pkg, np.random.default_rng(14), [5], 16, 10, 4)
    b.state.n_seq = 0
    cu, new = torch.full((2,), 7, dtype=torch.int32, device="cuda"), dev([1])
    torch.cuda.synchronize()
    ctx.paged_plan(b.state, None, new, 4, cu)
    ctx.sync()
    assert host(cu).tolist() == [0, 7]
    cu.fill_(7)
    torch.cuda.synchronize()
    ctx.capture_begin()
    ctx.paged_plan(b.state, None, new, 4, cu)
    g = ctx.capture_end()
    g.launch()
    ctx.sync()
    assert host(cu).tolist() == [0, 7]
    b.same()

"""The operators of batched serving over a paged cache held in 8 bits, case by case: pages and slots of the coming
tokens planned on the device, appending rotated keys and values as 8-bit codes with a scale for each block of positions
and head, and attention of one new token per sequence and of whole prompts over such a cache.

`own` false: each operator in its plain form, elementary torch operations in 32 bits.  `own` true: the package's
entry points.  Head shapes and windows are those of the package's decode configurations (14/2 heads of 64, 32/4 of
128, 16/8 of 256 with a window of 1024).
"""
import importlib
import math

import numpy as np
import torch

own = False

DEV = "cuda"
NO_PAGE = 0xFFFFFFFF
THETA = 1e6
EPS = 1e-6


# ── cases ────────────────────────────────────────────────────────────────────

def listed():
    return [
        # one step of a batch of chats: a token each, a few chats cut back or ended before it
        dict(name="plan, one step", op="plan", seqs=64, new_lo=1, new_hi=1, past_lo=100, past_hi=4000, cut=0.2, page=16),
        # a wave of prompts: pages and slots of a quarter of a million tokens
        dict(name="plan, prompts", op="plan", seqs=512, new_lo=100, new_hi=2000, past_lo=0, past_hi=1000, cut=0.5, page=32),
        # one decode step of a batch of chats: a token each, most into a block that holds others already
        dict(name="append, 64 sequences", op="append", seqs=64, new_lo=1, new_hi=1, past_lo=16, past_hi=250, heads=32,
             kv=4, hd=128, page=16, block=16, v_norm=False, neox=True),
        # three prompts of uneven length with normalised values, behind cached conversations
        dict(name="append, prompts", op="append", seqs=3, new_lo=1001, new_hi=4001, past_lo=0, past_hi=700, heads=16,
             kv=8, hd=256, page=32, block=32, v_norm=True, neox=False),
        # one chat on a sliding-window layer with capped scores: the call's latency is what counts
        dict(name="decode, one window", op="decode", seqs=1, lo=2345, hi=2345, heads=16, kv=8, hd=256, page=32, block=32,
             softcap=50.0, window=1024, alibi=False),
        # a batch of chats with histories of very different lengths
        dict(name="decode, 64 ragged", op="decode", seqs=64, lo=200, hi=8192, heads=32, kv=4, hd=128, page=16, block=16,
             softcap=0.0, window=0, alibi=False),
        # one long document
        dict(name="decode, one long", op="decode", seqs=1, lo=130001, hi=130001, heads=32, kv=4, hd=128, page=64, block=64,
             softcap=0.0, window=0, alibi=False),
        # a short follow-up question on a cached conversation
        dict(name="prompt, follow-up", op="prompt", seqs=1, new_lo=257, new_hi=257, past_lo=1243, past_hi=1243, heads=14,
             kv=2, hd=64, page=16, block=16, causal=True, softcap=0.0, window=0, alibi=False, prefix=0, doc=0),
        # one long prompt from its first token
        dict(name="prompt, 8192", op="prompt", seqs=1, new_lo=8192, new_hi=8192, past_lo=0, past_hi=0, heads=32, kv=4,
             hd=128, page=16, block=16, causal=True, softcap=0.0, window=0, alibi=False, prefix=0, doc=0),
        # packed documents, the first tokens seen in both directions, capped scores and a distance bias
        dict(name="prompt, documents", op="prompt", seqs=3, new_lo=1501, new_hi=2777, past_lo=0, past_hi=515, heads=16,
             kv=8, hd=256, page=32, block=32, causal=True, softcap=50.0, window=1024, alibi=True, prefix=300, doc=900),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def _shape(rng):
    heads, kv, hd = rng.choice([(14, 2, 64), (32, 4, 128), (16, 8, 256), (8, 8, 128), (16, 1, 128), (6, 2, 64)])
    block = rng.choice([16, 16, 32, 64, 128])
    return dict(heads=heads, kv=kv, hd=hd, block=block, page=block * rng.choice([1, 1, 1, 2, 3]))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "decode", "decode", "decode", "prompt", "prompt", "prompt"])
    if op == "plan":
        seqs = _log(rng, 1, 1024)
        hi = _log(rng, 1, max(1, 262144 // seqs))
        past = _log(rng, 1, 4000)
        return dict(op=op, seqs=seqs, new_lo=rng.choice([0, 1, hi // 3, hi]), new_hi=hi, past_lo=past // 4, past_hi=past,
                    cut=rng.choice([0.0, 0.1, 0.5, 1.0]), page=rng.choice([1, 16, 24, 32, 64, 128]))
    if op == "append":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, 6000 // seqs))
        past = _log(rng, 1, max(1, 16384 // seqs))
        return dict(op=op, seqs=seqs, new_lo=max(1, hi // 3), new_hi=hi, past_lo=past // 4, past_hi=past, v_norm=rng.random() < 0.3,
                    neox=rng.random() < 0.7, **_shape(rng))
    if op == "decode":
        s = _shape(rng)
        seqs = _log(rng, 1, 128)
        hi = _log(rng, 1, min(131072, max(64, (1 << 27) // (s["kv"] * s["hd"] * seqs))))
        return dict(op=op, seqs=seqs, lo=rng.choice([0, 1, hi // 20, hi]), hi=hi, softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                    window=rng.choice([0, 0, 0, 1024, _log(rng, 1, 4096)]), alibi=rng.random() < 0.25, **s)
    s = _shape(rng)
    seqs = _log(rng, 1, 8)
    hi = _log(rng, 1, 4096 // seqs)
    past = _log(rng, 1, 2048)
    return dict(op=op, seqs=seqs, new_lo=max(1, hi // 4), new_hi=hi, past_lo=past // 3, past_hi=past, causal=rng.random() < 0.85,
                softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), window=rng.choice([0, 0, 1024, _log(rng, 1, 2048)]),
                alibi=rng.random() < 0.25, prefix=rng.choice([0, 0, _log(rng, 1, 600)]),
                doc=rng.choice([0, 0, _log(rng, 30, 1500)]), **s)


def _spread(n, lo, hi, shift=0.0):
    """n lengths between lo and hi, even over their logarithm, in a mixed order; the case alone decides them."""
    if n == 1:
        return [hi]
    u = [((i + shift) * 0.6180339887498949) % 1.0 for i in range(n)]
    rank = sorted(range(n), key=u.__getitem__)
    out = [0] * n
    for k, i in enumerate(rank):
        f = k / (n - 1)
        out[i] = int(round(math.exp(math.log(lo + 1) * (1 - f) + math.log(hi + 1) * f))) - 1
    return out


def _new_past(case):
    new = _spread(case["seqs"], case["new_lo"], case["new_hi"])
    past = _spread(case["seqs"], case["past_lo"], case["past_hi"], 0.37)
    return new, past


def _keeps(case, past):
    """How many positions of each sequence stay: most all, some cut back a little, some ended."""
    cut = int(round(case["cut"] * case["seqs"]))
    return [n if i >= cut else (0 if i % 3 == 0 else max(0, n - 1 - i % 7)) for i, n in enumerate(past)]


def _docs_of(case, n):
    """Document number of each of n cached positions: document d holds about case["doc"] tokens."""
    if not case["doc"]:
        return None
    j = np.arange(n, dtype=np.int64)
    return (j + j // (2 * case["doc"]) * 37) // case["doc"]


# ── what a user's program has in hand ────────────────────────────────────────

def _pkg():
    return importlib.import_module("llmtoy-zig_b200")


_context = None


def _ctx():
    """The one device context that a program keeps."""
    global _context
    if _context is None:
        _context = _pkg().Context(0)
    return _context


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _i32(v):
    return torch.as_tensor(np.asarray(v, dtype=np.int64).astype(np.uint32).view(np.int32), device=DEV)


def _tables(g, caps, page):
    """Page tables of sequences of up to caps[s] positions over one pool, its pages handed out in no order."""
    need = [-(-c // page) for c in caps]
    total, width = max(1, sum(need)), max(1, max(need))
    order = torch.randperm(total, generator=g, device=DEV).cpu().numpy()
    table = np.zeros((len(caps), width), dtype=np.int64)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return _i32(table), total, width


def _pool(g, pages, case):
    """K and V of a pool as codes [2][page][head][slot][head_dim] and scales [2][page][head][block of the page]."""
    shape = (pages, case["kv"], case["page"] // case["block"], case["block"], case["hd"])
    codes = torch.empty((2,) + shape, dtype=torch.int8, device=DEV)
    scales = torch.empty((2,) + shape[:3], device=DEV)
    for i in range(2):
        x = torch.randn(shape, generator=g, device=DEV)
        if case["op"] != "append" and i == 0:  # some positions draw most heads, as the first tokens of a text do
            x.mul_(torch.where(torch.rand(pages, 1, shape[2], case["block"], 1, generator=g, device=DEV) < 0.01, 2.0, 1.0))
        scales[i] = x.abs().amax((3, 4)) / 127.0
        codes[i] = torch.round(x.div_(scales[i][..., None, None])).to(torch.int8)
    return codes.view(2, pages, case["kv"], case["page"], case["hd"]), scales


def _handle(st, case):
    """The descriptors of cache, batch and attention layer that a program builds once."""
    p = _pkg()
    if case["op"] == "plan":
        st["state"] = p.PagedState(n_seq=case["seqs"], page_size=case["page"], n_pages=st["pages"], max_pages=st["width"],
                                   lens=st["lens"].data_ptr(), page_table=st["table"].data_ptr(), free=st["free"].data_ptr(),
                                   n_free=st["n_free"].data_ptr())
        return
    st["kvh"] = p.PagedQ8(n_kv_heads=case["kv"], head_dim=case["hd"], page_size=case["page"], block=case["block"],
                          n_pages=st["pages"], max_pages=st["width"], k=st["codes"][0].data_ptr(), v=st["codes"][1].data_ptr(),
                          k_scale=st["scales"][0].data_ptr(), v_scale=st["scales"][1].data_ptr())
    if case["op"] == "append":
        st["cfg"] = p.AttnCfg(n_heads=case["heads"], n_kv_heads=case["kv"], head_dim=case["hd"], rope_neox=int(case["neox"]),
                              rope_theta=THETA, eps=EPS, scale=1.0, kv_cap=1, window=0, v_norm=int(case["v_norm"]), kv_f16=0)
    else:
        st["cfg"] = p.PagedAttnCfg(n_heads=case["heads"], window=case["window"], causal=int(case.get("causal", True)),
                                   scale=st["scale"], softcap=case["softcap"],
                                   slopes=st["slopes"].data_ptr() if case["alibi"] else None)


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case, "op": case["op"]}
    if case["op"] == "plan":
        _prepare_plan(case, g, st)
    else:
        _prepare_cache(case, g, st)
    if own:
        _handle(st, case)
    return st


def _prepare_plan(case, g, st):
    new, past = _new_past(case)
    keep = _keeps(case, past)
    lens = [max(a, b) for a, b in zip(keep, past)]
    table, _, width = _tables(g, lens, case["page"])
    held = sum(-(-n // case["page"]) for n in lens)
    width = max(width, max(-(-(a + b) // case["page"]) for a, b in zip(keep, new)) + 1)
    spare = sum(-(-n // case["page"]) + 1 for n in new) + 5
    pages = held + spare
    # which pages the sequences hold is as mixed as which are free
    order = torch.randperm(pages, generator=g, device=DEV).int()
    full = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEV)
    mine = torch.arange(table.shape[1], device=DEV) < _i32([-(-n // case["page"]) for n in lens])[:, None]
    full[:, :table.shape[1]] = torch.where(mine, order[table.long().clamp(0, max(0, held - 1))], full[:, :table.shape[1]])
    free = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
    free[:spare] = order[held:]
    total = sum(new)
    blank = torch.zeros(3, max(1, total), dtype=torch.int32, device=DEV)
    st.update(total=total, pages=pages, width=width, table=full, lens=_i32(lens), keep=_i32(keep), new=_i32(new), free=free,
              n_free=_i32([spare]), cu=torch.zeros(case["seqs"] + 1, dtype=torch.int32, device=DEV), seq=blank[0], pos=blank[1],
              slot=blank[2])


def _prepare_cache(case, g, st):
    if case["op"] in ("append", "prompt"):
        new, past = _new_past(case)
        lens = [a + b for a, b in zip(new, past)]
        cu = np.concatenate([[0], np.cumsum(new)])
        st.update(new=new, lens_host=lens, total=int(cu[-1]), max_q=max(new), cu=_i32(cu))
    else:
        lens = _spread(case["seqs"], case["lo"], case["hi"])
    # a program reserves room for the tokens to come
    table, pages, width = _tables(g, [n + (0 if case["op"] == "append" else 17) for n in lens], case["page"])
    st.update(table=table, pages=pages, width=width, lens=_i32(lens), max_len=max(1, max(lens)))
    st["codes"], st["scales"] = _pool(g, pages, case)
    if case["op"] == "append":
        nq, nkv = case["heads"] * case["hd"], case["kv"] * case["hd"]
        st["qkv"] = torch.randn(st["total"], nq + 2 * nkv, generator=g, device=DEV) * 2.0
        st["qn"] = 1.0 + 0.2 * torch.randn(case["hd"], generator=g, device=DEV)
        st["kn"] = 1.0 + 0.2 * torch.randn(case["hd"], generator=g, device=DEV)
        st["q"] = torch.empty(st["total"], nq, device=DEV)
        st["values"] = torch.empty(st["codes"].shape, dtype=torch.float16, device=DEV)
        return
    rows = case["seqs"] if case["op"] == "decode" else st["total"]
    st["scale"] = 1.0 / math.sqrt(case["hd"])
    st["q"] = torch.randn(rows, case["heads"], case["hd"], generator=g, device=DEV) * 1.5  # scores spread by about 1.5
    st["out"] = torch.empty(rows, case["heads"], case["hd"], device=DEV)
    st["slopes"] = _i32(np.zeros(1)) if not case["alibi"] else torch.tensor(
        [2.0 ** (-8.0 * (i + 1) / case["heads"]) for i in range(case["heads"])], device=DEV)
    if case["op"] == "prompt":
        st["prefix"] = _i32([min(case["prefix"], n) for n in lens]) if case["prefix"] else None
        docs = _docs_of(case, st["max_len"])
        st["docs"] = None if docs is None else _i32(np.tile(docs, (case["seqs"], 1)))


# ── one pass ─────────────────────────────────────────────────────────────────

def run(st):
    return (_OWN if own else _PLAIN)[st["op"]](st)


def _own_plan(st):
    _ctx().paged_plan(st["state"], st["keep"], st["new"], st["total"], st["cu"], st["seq"], st["pos"], st["slot"])
    return _plan_outputs(st)


def _own_append(st):
    _ctx().paged_q8_append(st["cfg"], st["kvh"], st["qkv"], st["case"]["seqs"], st["cu"], st["total"], st["max_q"], st["qn"],
                           st["kn"], None, st["table"], st["lens"], st["q"])
    return _append_outputs(st)


def _own_decode(st):
    _ctx().paged_q8_attn_decode(st["cfg"], st["kvh"], st["q"], st["case"]["seqs"], st["table"], st["lens"], st["max_len"],
                                st["out"])
    return {"out": st["out"]}


def _own_prompt(st):
    _ctx().paged_q8_attn_prompt(st["cfg"], st["kvh"], st["q"], st["case"]["seqs"], st["cu"], st["total"], st["max_q"],
                                st["table"], st["lens"], st["max_len"], st["out"], st["prefix"], st["docs"], st["max_len"])
    return {"out": st["out"]}


def _plan_outputs(st):
    return {x: st[x] for x in ("lens", "table", "free", "n_free", "cu")} | {x: st[x][:st["total"]] for x in ("seq", "pos", "slot")}


def _append_outputs(st):
    """The queries, the scales, and the cache as the values that its codes stand for."""
    c = st["case"]
    split = (2, st["pages"], c["kv"], c["page"] // c["block"], c["block"], c["hd"])
    torch.mul(st["codes"].view(split), st["scales"][..., None, None], out=st["values"].view(split))
    return {"q": st["q"], "scales": st["scales"], "values": st["values"]}


def _plain_plan(st):
    p, width = st["case"]["page"], st["width"]
    lens, keep, new = st["lens"].long(), st["keep"].long(), st["new"].long()
    have, stay, want = (lens + p - 1) // p, (keep + p - 1) // p, (keep + new + p - 1) // p
    j = torch.arange(width, device=DEV)
    gone = (j >= stay[:, None]) & (j < have[:, None])
    take = (j >= stay[:, None]) & (j < want[:, None])
    back = st["table"][gone].flip(0)          # the last sequence's last page first
    n = st["n_free"].long()
    st["free"].index_copy_(0, n + torch.arange(len(back), device=DEV), back)
    st["table"][gone] = -1
    taken = torch.arange(int(take.sum()), device=DEV)
    st["table"][take] = st["free"][n + len(back) - 1 - taken]
    st["n_free"] += len(back) - len(taken)
    st["lens"].copy_(keep + new)
    cu = torch.cumsum(new, 0)
    st["cu"][1:] = cu
    seq = torch.repeat_interleave(torch.arange(len(new), device=DEV), new, output_size=st["total"])
    pos = torch.arange(st["total"], device=DEV) - (cu - new)[seq] + keep[seq]
    st["seq"][:st["total"]] = seq
    st["pos"][:st["total"]] = pos
    st["slot"][:st["total"]] = st["table"].long()[seq, pos // p] * p + pos % p
    return _plan_outputs(st)


def _plain_append(st):
    c, hd, half, block = st["case"], st["case"]["hd"], st["case"]["hd"] // 2, st["case"]["block"]
    T, H, kv, per = st["total"], c["heads"], c["kv"], c["page"] // c["block"]
    x = st["qkv"].view(T, H + 2 * kv, hd)
    q, k, v = x[:, :H], x[:, H:H + kv], x[:, H + kv:]
    inv = lambda t: 1.0 / torch.sqrt((t * t).sum(-1, keepdim=True) / hd + EPS)  # noqa: E731
    q, k = q * inv(q) * st["qn"], k * inv(k) * st["kn"]
    v = v * inv(v) if c["v_norm"] else v
    cu, lens = st["cu"].long(), st["lens"].long()
    new = cu[1:] - cu[:-1]
    first = lens - new                                                  # the first new position of each sequence
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device=DEV), new, output_size=T)
    pos = torch.arange(T, device=DEV) - cu[seq] + first[seq]
    e = torch.arange(half, device=DEV).double() * 2.0 / hd               # angles of far positions need 64 bits
    ang = pos.double()[:, None] / torch.pow(torch.full_like(e, THETA), e)
    cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]

    def turn(t):
        a, b = (t[..., :half], t[..., half:]) if c["neox"] else (t[..., 0::2], t[..., 1::2])
        a, b = a * cos - b * sin, a * sin + b * cos
        return torch.cat([a, b], -1) if c["neox"] else torch.stack([a, b], -1).flatten(-2)

    kvs = torch.stack([turn(k), v])                                     # [2, T, kv, hd]
    codes = st["codes"].view(2, -1, kv, per, block, hd)
    # blocks by number: page * per + place in the page; what of the first block of each sequence stays
    number = lambda s, j: st["table"].long()[s, j // c["page"]] * per + j % c["page"] // block  # noqa: E731
    every = torch.arange(c["seqs"], device=DEV)
    fb = number(every, first.clamp(max=st["width"] * c["page"] - 1))
    old = first % block                                                 # positions that stay
    flat = st["scales"].transpose(2, 3).reshape(2, -1, kv)              # [2, block number, kv]: a copy
    old_scale = flat[:, fb]
    b = number(seq, pos)
    top = torch.zeros_like(flat).scatter_reduce_(1, b[None, :, None].expand(2, T, kv), kvs.abs().amax(-1), "amax")
    touched = torch.zeros(flat.shape[1], dtype=torch.bool, device=DEV).index_fill_(0, b, True)
    scale = top / 127.0
    stays = torch.zeros_like(flat).index_copy_(1, fb, torch.where((old > 0)[None, :, None], old_scale, torch.zeros_like(old_scale)))
    scale = torch.maximum(scale, stays)
    flat = torch.where(touched[None, :, None], scale, flat)
    st["scales"].copy_(flat.view(2, -1, per, kv).transpose(2, 3))
    # the codes that stay, on the grown scale
    keep_rows = codes[:, fb // per, :, fb % per]                        # [seqs, 2, kv, block, hd]
    now = flat[:, fb].transpose(0, 1)[..., None, None]
    was = old_scale.transpose(0, 1)[..., None, None]
    again = torch.round(keep_rows.float() * torch.where(now == 0, torch.zeros_like(now), was / now)).to(torch.int8)
    stay = torch.arange(block, device=DEV).view(1, 1, 1, block, 1) < old.view(-1, 1, 1, 1, 1)
    codes[:, fb // per, :, fb % per] = torch.where(stay & (now != was), again, keep_rows)
    s = flat[:, b][..., None]
    made = torch.round(kvs / torch.where(s == 0, torch.ones_like(s), s)).clamp(-127, 127).to(torch.int8)
    codes[:, b // per, :, b % per, pos % block] = made.transpose(0, 1)
    st["q"].copy_(turn(q).reshape(T, H * hd))
    return _append_outputs(st)


def _scores(st, s, dist):
    """Raw scores [..., heads, queries, keys] -> capped and biased; dist [..., 1, queries, keys]."""
    c = st["case"]
    s = s * st["scale"]
    if c["softcap"]:
        s = torch.tanh(s / c["softcap"]) * c["softcap"]
    if c["alibi"]:
        s = s - st["slopes"].view(-1, 1, 1) * dist.abs()
    return s


def _softmax(s, seen):
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _cached(st, n):
    """Values of the first n positions of every sequence: K and V as [seqs, kv, n, hd]."""
    c = st["case"]
    j = torch.arange(n, device=DEV)
    page = st["table"].long()[:, j // c["page"]]                        # [seqs, n]
    h = torch.arange(c["kv"], device=DEV).view(1, -1, 1)
    return (st["codes"][i][page[:, None], h, j % c["page"]] * st["scales"][i][page[:, None], h, j % c["page"] // c["block"]][..., None]
            for i in range(2))


def _plain_decode(st):
    c, n = st["case"], st["max_len"]
    S, H, kv, hd = c["seqs"], c["heads"], c["kv"], c["hd"]
    k, v = _cached(st, n)
    s = torch.matmul(st["q"].view(S, kv, H // kv, hd), k.transpose(2, 3)).view(S, H, 1, n)
    dist = (st["lens"].long()[:, None] - 1 - torch.arange(n, device=DEV)).view(S, 1, 1, n)
    seen = (dist >= 0) & ((dist < c["window"]) if c["window"] else (dist >= 0))
    p = _softmax(_scores(st, s, dist), seen).view(S, kv, H // kv, n)
    return {"out": torch.matmul(p, v).view(S, H, hd)}


def _plain_prompt(st):
    c, n, mq = st["case"], st["max_len"], st["max_q"]
    S, H, kv, hd = c["seqs"], c["heads"], c["kv"], c["hd"]
    k, v = _cached(st, n)
    cu = st["cu"].long()
    r = torch.arange(mq, device=DEV)
    new = (cu[1:] - cu[:-1])[:, None]
    real = r < new                                                      # [S, mq]
    at = torch.where(real, cu[:-1, None] + r, torch.zeros_like(cu[:-1, None]))
    q = st["q"][at].view(S, mq, kv, H // kv, hd).permute(0, 2, 3, 1, 4).reshape(S, kv, H // kv * mq, hd)
    s = torch.matmul(q, k.transpose(2, 3)).view(S, H, mq, n)
    i = (st["lens"].long()[:, None] - new + r)[:, None, :, None]        # positions of the queries
    j = torch.arange(n, device=DEV).view(1, 1, 1, n)
    seen = j < st["lens"].long().view(S, 1, 1, 1)
    if c["causal"]:
        ahead = j <= i
        if st["prefix"] is not None:
            ahead = ahead | (j < st["prefix"].long().view(S, 1, 1, 1))
        seen = seen & ahead
    if c["window"]:
        seen = seen & (i - j < c["window"])
    if st["docs"] is not None:
        d = st["docs"].long()
        mine = torch.gather(d, 1, i.view(S, mq).clamp(0, n - 1)).view(S, 1, mq, 1)
        seen = seen & (d.view(S, 1, 1, n) == mine)
    p = _softmax(_scores(st, s, i - j), seen).view(S, kv, H // kv * mq, n)
    out = torch.matmul(p, v).view(S, H, mq, hd).transpose(1, 2)
    return {"out": out[real]}


_OWN = {"plan": _own_plan, "append": _own_append, "decode": _own_decode, "prompt": _own_prompt}
_PLAIN = {"plan": _plain_plan, "append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt}


# ── what a pass cannot do without ────────────────────────────────────────────

def _pairs(case, new, lens):
    """Visible (query, key) pairs of a prompt, summed over the sequences, and the cached positions that any query sees."""
    pairs = keys = 0
    for a, n in zip(new, lens):
        i = np.arange(n - a, n, dtype=np.int64)
        lo, hi = np.zeros_like(i), np.full_like(i, n - 1)
        if case["causal"]:
            hi = np.maximum(i, min(case["prefix"], n) - 1)
        if case["window"]:
            lo = np.maximum(lo, i - case["window"] + 1)
        docs = _docs_of(case, n)
        if docs is not None:
            lo = np.maximum(lo, np.searchsorted(docs, docs[i], "left"))
            hi = np.minimum(hi, np.searchsorted(docs, docs[i], "right") - 1)
        pairs += int(np.maximum(0, hi - lo + 1).sum())
        keys += int(hi.max() - lo.min() + 1)
    return pairs, keys


def work(case):
    op, ceil = case["op"], lambda a, b: -(-a // b)
    if op == "plan":
        new, past = _new_past(case)
        keep, p = _keeps(case, past), case["page"]
        moved = sum(ceil(max(n, a), p) + ceil(a + b, p) - 2 * ceil(a, p) for n, a, b in zip(past, keep, new))
        return {"bytes": 12 * sum(new) + 8 * moved + 20 * case["seqs"], "flops": 0}
    token = case["kv"] * case["hd"]
    scales = 8 * case["kv"] / case["block"]                             # bytes of both scales per position
    if op == "append":
        # with the values of the whole pool that a pass here returns: a byte read and two written for each
        new, past = _new_past(case)
        row = case["heads"] * case["hd"]
        pool = 2 * token * case["page"] * sum(ceil(a + b, case["page"]) for a, b in zip(new, past))
        return {"bytes": sum(new) * (4 * (row + 2 * token) + 4 * row + 2 * token) + 3 * pool, "flops": sum(new) * 10 * (row + token) + pool}
    if op == "decode":
        lens = _spread(case["seqs"], case["lo"], case["hi"])
        seen = sum(min(n, case["window"]) if case["window"] else n for n in lens)
        return {"bytes": seen * (2 * token + scales) + 8 * case["seqs"] * case["heads"] * case["hd"] + 4 * seen / case["page"],
                "flops": 4 * seen * case["heads"] * case["hd"]}
    new, past = _new_past(case)
    pairs, keys = _pairs(case, new, [a + b for a, b in zip(new, past)])
    return {"bytes": 8 * sum(new) * case["heads"] * case["hd"] + keys * (2 * token + scales), "flops": 4 * pairs * case["heads"] * case["hd"]}


# ── the definitions in 64 bits ───────────────────────────────────────────────

def exact(case, seed):
    return None if case["op"] == "plan" else _EXACT[case["op"]](prepare(case, seed), case)


def _exact_append(st, c):
    hd, H, kv, B = c["hd"], c["heads"], c["kv"], c["block"]
    x = st["qkv"].double().reshape(st["total"], H + 2 * kv, hd)
    rms = (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    cu = np.concatenate([[0], np.cumsum(st["new"])])
    pos = torch.as_tensor(np.concatenate([np.arange(n - m, n) for m, n in zip(st["new"], st["lens_host"])]), device=DEV)
    i = torch.arange(0, hd, 2, device=DEV, dtype=torch.float64)
    z = torch.polar(torch.ones(st["total"], hd // 2, device=DEV, dtype=torch.float64), pos.double()[:, None] * THETA ** (-i / hd))
    pair = (torch.arange(hd // 2, device=DEV), torch.arange(hd // 2, device=DEV) + hd // 2) if c["neox"] else (i.long(), i.long() + 1)
    y = x[:, :H + kv] * rms[:, :H + kv] * torch.cat([st["qn"].double().expand(H, hd), st["kn"].double().expand(kv, hd)])
    w = torch.complex(y[..., pair[0]], y[..., pair[1]]) * z[:, None]
    y[..., pair[0]], y[..., pair[1]] = w.real, w.imag
    both = (y[:, H:], x[:, H + kv:] * (rms[:, H + kv:] if c["v_norm"] else 1.0))
    codes, scales = st["codes"].double(), st["scales"].double()
    values = codes * scales.repeat_interleave(B, 3)[..., None]
    table = st["table"].cpu().numpy()
    for s, (m, n) in enumerate(zip(st["new"], st["lens_host"])):
        lo = (n - m) // B                                               # blocks lo .. hi - 1 of the sequence are written
        hi = -(-n // B)
        old = n - m - lo * B
        at = torch.as_tensor(table[s, np.arange(lo, hi) * B // c["page"]], device=DEV).long()
        sub = torch.as_tensor(np.arange(lo, hi) * B % c["page"] // B, device=DEV)
        for t in range(2):
            fresh = torch.zeros(hi - lo, B, kv, hd, device=DEV, dtype=torch.float64)
            fresh.view(-1, kv, hd)[old:old + m] = both[t][cu[s]:cu[s] + m]
            size = fresh.abs().amax((1, 3)) / 127                       # [blocks, kv]
            was = scales[t][at[0], :, sub[0]].clone()
            if old:
                size[0] = torch.maximum(size[0], was)
            told = torch.where(size > 0, size, torch.ones_like(size))[:, None, :, None]
            made = torch.round(fresh / told).clamp(-127, 127) * size[:, None, :, None]
            view = values[t].view(st["pages"], kv, c["page"] // B, B, hd)
            if old:
                had = codes[t].view(st["pages"], kv, c["page"] // B, B, hd)[at[0], :, sub[0], :old]   # [kv, old, hd]
                grown = torch.round(had * (was / torch.where(size[0] > 0, size[0], torch.ones_like(was)))[:, None, None])
                made[0, :old] = (torch.where((size[0] == was)[:, None, None], had, grown) * size[0][:, None, None]).transpose(0, 1)
            scales[t][at, :, sub] = size
            # slots behind the last position keep their codes; they stand for them on the block's new scale
            rest = hi * B - n
            if rest:
                made[-1, B - rest:] = (codes[t].view(st["pages"], kv, c["page"] // B, B, hd)[at[-1], :, sub[-1], B - rest:]
                                       * size[-1][:, None, None]).transpose(0, 1)
            view[at, :, sub] = made.transpose(1, 2)
    return {"q": y[:, :H].reshape(st["total"], -1), "scales": scales, "values": values}


def _exact_rows(st, c, s, h, queries, i, n, keep):
    """Attention of queries [m, hd] at positions i [m] of head h of sequence s over its first n cached positions."""
    pages = st["table"][s, :-(-n // c["page"])].long()
    kh = h // (c["heads"] // c["kv"])
    K, V = ((st["codes"][t][pages, kh].double().reshape(-1, c["block"], c["hd"]) * st["scales"][t][pages, kh].double().reshape(-1, 1, 1))
            .reshape(-1, c["hd"])[:n] for t in range(2))
    t = queries.double() @ K.T / math.sqrt(c["hd"])
    t = c["softcap"] * torch.tanh(t / c["softcap"]) if c["softcap"] else t
    if c["alibi"]:
        t = t - 2.0 ** (-8.0 * (h + 1) / c["heads"]) * (i[:, None] - torch.arange(n, device=DEV)).abs()
    t = t.masked_fill(~keep, -math.inf)
    e = torch.exp(t - t.amax(1, keepdim=True).nan_to_num(neginf=0.0))
    return e / e.sum(1, keepdim=True).clamp(min=1e-300) @ V


def _exact_decode(st, c):
    out = torch.zeros_like(st["out"], dtype=torch.float64)
    for s, n in enumerate(st["lens"].tolist()):
        if n == 0:
            continue
        i = torch.tensor([n - 1], device=DEV)
        keep = torch.ones(1, n, dtype=torch.bool, device=DEV)
        if c["window"]:
            keep[0, :max(0, n - c["window"])] = False
        for h in range(c["heads"]):
            out[s, h:h + 1] = _exact_rows(st, c, s, h, st["q"][s, h:h + 1], i, n, keep)
    return {"out": out}


def _exact_prompt(st, c):
    out = torch.zeros_like(st["out"], dtype=torch.float64)
    first = 0
    for s, (m, n) in enumerate(zip(st["new"], st["lens_host"])):
        i = torch.arange(n - m, n, device=DEV)
        j = torch.arange(n, device=DEV)
        keep = torch.ones(m, n, dtype=torch.bool, device=DEV)
        if c["causal"]:
            keep &= (j[None] <= i[:, None]) | (j < min(c["prefix"], n))[None]
        if c["window"]:
            keep &= j[None] > i[:, None] - c["window"]
        if c["doc"]:
            d = torch.as_tensor(_docs_of(c, n), device=DEV)
            keep &= d[i][:, None] == d[None]
        for h in range(c["heads"]):
            out[first:first + m, h] = _exact_rows(st, c, s, h, st["q"][first:first + m, h], i, n, keep)
        first += m
    return {"out": out}


_EXACT = {"append": _exact_append, "decode": _exact_decode, "prompt": _exact_prompt}

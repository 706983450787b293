"""The batched-serving operators of this package, case by case: appending rotated keys and values to a paged cache,
attention of one new token per sequence and of whole prompts over that cache, eviction from it by accumulated
attention weight, and the rules applied to logits before a token is chosen.

`own` false: each operator in its plain form, elementary torch operations in 32 bits.  `own` true: the package's
entry points.  Head shapes, windows and vocabularies are those of the package's decode configurations (14/2 heads of
64, 32/4 of 128, 16/8 of 256 with a window of 1024; vocabularies of 151936 and 262144 tokens).
"""
import importlib
import math

import numpy as np
import torch

own = False

DEV = "cuda"
NO_MASK = 0xFFFFFFFF
THETA = 1e6
EPS = 1e-6


# ── cases ────────────────────────────────────────────────────────────────────

def listed():
    return [
        # one decode step of a batch of chats: 64 sequences append a token each to an f16 cache
        dict(name="append, 64 sequences", op="append", seqs=64, new_lo=1, new_hi=1, past_lo=100, past_hi=4000, heads=32,
             kv=4, hd=128, f16=True, page=16, v_norm=False, neox=True),
        # three prompts of uneven length with normalised values, 32-bit cache
        dict(name="append, prompts", op="append", seqs=3, new_lo=1001, new_hi=4001, past_lo=0, past_hi=700, heads=16,
             kv=8, hd=256, f16=False, page=32, v_norm=True, neox=False),
        # one chat on a sliding-window layer with capped scores, 32-bit cache: the call's latency is what counts
        dict(name="decode, one window", op="decode", seqs=1, lo=2345, hi=2345, heads=16, kv=8, hd=256, f16=False, page=32,
             softcap=50.0, window=1024, alibi=False, mass=False),
        # a batch of chats with histories of very different lengths
        dict(name="decode, 64 ragged", op="decode", seqs=64, lo=200, hi=8192, heads=32, kv=4, hd=128, f16=True, page=16,
             softcap=0.0, window=0, alibi=False, mass=False),
        # one long document whose cache collects attention weights for eviction
        dict(name="decode, one long", op="decode", seqs=1, lo=130001, hi=130001, heads=32, kv=4, hd=128, f16=True,
             page=64, softcap=0.0, window=0, alibi=False, mass=True),
        # a short follow-up question on a cached conversation
        dict(name="prompt, follow-up", op="prompt", seqs=1, new_lo=257, new_hi=257, past_lo=1243, past_hi=1243, heads=14,
             kv=2, hd=64, f16=True, page=16, causal=True, softcap=0.0, window=0, alibi=False, prefix=0, doc=0),
        # one long prompt from its first token
        dict(name="prompt, 8192", op="prompt", seqs=1, new_lo=8192, new_hi=8192, past_lo=0, past_hi=0, heads=32, kv=4,
             hd=128, f16=True, page=16, causal=True, softcap=0.0, window=0, alibi=False, prefix=0, doc=0),
        # packed documents, the first tokens seen in both directions, capped scores and a distance bias
        dict(name="prompt, documents", op="prompt", seqs=3, new_lo=1501, new_hi=2777, past_lo=0, past_hi=515, heads=16,
             kv=8, hd=256, f16=True, page=32, causal=True, softcap=50.0, window=1024, alibi=True, prefix=300, doc=900),
        # a few chats around their cache budget
        dict(name="evict, short", op="evict", seqs=8, lo=900, hi=1300, budget=1024, recent=128, kv=2, hd=64, f16=True,
             page=16),
        # long contexts cut to a quarter
        dict(name="evict, long", op="evict", seqs=16, lo=20000, hi=32768, budget=8192, recent=1024, kv=4, hd=128, f16=True,
             page=64),
        # the logits of one chat, with a grammar
        dict(name="logits, one row", op="logits", rows=1, vocab=151936, hist=512, bias=16),
        # the logits of a batch: long histories, long bias lists, grammars on most rows
        dict(name="logits, 64 rows", op="logits", rows=64, vocab=262144, hist=8192, bias=300),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def _shape(rng):
    heads, kv, hd = rng.choice([(14, 2, 64), (32, 4, 128), (16, 8, 256), (8, 8, 128), (16, 1, 128), (6, 2, 64)])
    return dict(heads=heads, kv=kv, hd=hd, f16=rng.random() < 0.75, page=rng.choice([1, 16, 24, 32, 64, 128]))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prompt", "prompt", "evict", "logits"])
    if op == "append":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, 8192 // seqs))
        past = _log(rng, 1, 4000)
        return dict(op=op, seqs=seqs, new_lo=max(1, hi // 3), new_hi=hi, past_lo=past // 4, past_hi=past, v_norm=rng.random() < 0.3,
                    neox=rng.random() < 0.7, **_shape(rng))
    if op == "decode":
        s = _shape(rng)
        per_token = s["kv"] * s["hd"] * (2 if s["f16"] else 4)
        seqs = _log(rng, 1, 128)
        hi = _log(rng, 1, min(131072, max(64, (1 << 28) // (per_token * seqs))))
        return dict(op=op, seqs=seqs, lo=rng.choice([0, 1, hi // 20, hi]), hi=hi, softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                    window=rng.choice([0, 0, 0, 1024, _log(rng, 1, 4096)]), alibi=rng.random() < 0.25,
                    mass=rng.random() < 0.4, **s)
    if op == "prompt":
        s = _shape(rng)
        seqs = _log(rng, 1, 8)
        hi = _log(rng, 1, 4096 // seqs)
        past = _log(rng, 1, 2048)
        return dict(op=op, seqs=seqs, new_lo=max(1, hi // 4), new_hi=hi, past_lo=past // 3, past_hi=past, causal=rng.random() < 0.85,
                    softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), window=rng.choice([0, 0, 1024, _log(rng, 1, 2048)]),
                    alibi=rng.random() < 0.25, prefix=rng.choice([0, 0, _log(rng, 1, 600)]),
                    doc=rng.choice([0, 0, _log(rng, 30, 1500)]), **s)
    if op == "evict":
        s = _shape(rng)
        s.pop("heads")
        seqs = _log(rng, 1, 32)
        hi = _log(rng, 2, 262144 // seqs // s["kv"] * 4)
        budget = _log(rng, 1, max(1, hi // 2))
        return dict(op=op, seqs=seqs, lo=rng.choice([0, 1, hi // 3, hi]), hi=hi, budget=budget, recent=rng.choice([0, budget // 8, budget // 2, budget]), **s)
    return dict(op=op, rows=_log(rng, 1, 64), vocab=rng.choice([32003, 151936, 262144, _log(rng, 100, 262144)]),
                hist=_log(rng, 1, 8192), bias=rng.choice([0, _log(rng, 1, 300)]))


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
    new = [max(1, v) for v in _spread(case["seqs"], case["new_lo"], case["new_hi"])]
    past = _spread(case["seqs"], case["past_lo"], case["past_hi"], 0.37)
    return new, past


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
    shape = (pages, case["page"], case["kv"], case["hd"])
    kind = torch.float16 if case["f16"] else torch.float32
    return torch.randn(shape, generator=g, device=DEV, dtype=kind), torch.randn(shape, generator=g, device=DEV, dtype=kind)


def _handle(st, case):
    """The descriptors of cache and attention layer that a program builds once."""
    p = _pkg()
    st["kvh"] = p.PagedKV(n_kv_heads=case["kv"], head_dim=case["hd"], kv_f16=int(case["f16"]), page_size=case["page"],
                          n_pages=st["pages"], max_pages=st["width"], k=st["k"].data_ptr(), v=st["v"].data_ptr())
    if case["op"] == "append":
        st["cfg"] = p.AttnCfg(n_heads=case["heads"], n_kv_heads=case["kv"], head_dim=case["hd"], rope_neox=int(case["neox"]),
                              rope_theta=THETA, eps=EPS, scale=1.0, kv_cap=1, window=0, v_norm=int(case["v_norm"]),
                              kv_f16=int(case["f16"]))
    elif case["op"] != "evict":
        st["cfg"] = p.PagedAttnCfg(n_heads=case["heads"], window=case["window"], causal=int(case.get("causal", True)),
                                   scale=st["scale"], softcap=case["softcap"],
                                   slopes=st["slopes"].data_ptr() if case["alibi"] else None)


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case, "op": case["op"]}
    if case["op"] == "logits":
        return _prepare_logits(case, g, st)
    if case["op"] in ("append", "prompt"):
        new, past = _new_past(case)
        lens = [a + b for a, b in zip(new, past)]
        cu = np.concatenate([[0], np.cumsum(new)])
        st.update(new=new, lens_host=lens, total=int(cu[-1]), max_q=max(new), cu=_i32(cu))
    else:
        lens = _spread(case["seqs"], case["lo"], case["hi"])
    caps = [n + 17 for n in lens]  # a program reserves room for the tokens to come
    dst = [-(-min(n, case["budget"]) // case["page"]) for n in lens] if case["op"] == "evict" else []
    table, pages, width = _tables(g, caps, case["page"])
    if case["op"] == "evict":  # the kept positions move to fresh pages at the pool's end
        st["first_dst"] = pages
        t = np.zeros((len(lens), max(1, max(dst))), dtype=np.int64)
        for s, n in enumerate(dst):
            t[s, :n] = np.arange(pages, pages + n)
            pages += n
        full = np.zeros((len(lens), width), dtype=np.int64)
        full[:, :t.shape[1]] = t
        st["dst"] = _i32(full)
    st.update(table=table, pages=pages, width=width, lens=_i32(lens), max_len=max(1, max(lens)))
    st["k"], st["v"] = _pool(g, pages, case)
    if case["op"] == "append":
        nq, nkv = case["heads"] * case["hd"], case["kv"] * case["hd"]
        st["qkv"] = torch.randn(st["total"], nq + 2 * nkv, generator=g, device=DEV) * 2.0
        st["qn"] = 1.0 + 0.2 * torch.randn(case["hd"], generator=g, device=DEV)
        st["kn"] = 1.0 + 0.2 * torch.randn(case["hd"], generator=g, device=DEV)
        st["seq"] = _i32(np.repeat(np.arange(case["seqs"]), new))
        st["pos"] = _i32(np.concatenate([np.arange(b, b + a) for a, b in zip(new, past)]))
        st["q"] = torch.empty(st["total"], nq, device=DEV)
    elif case["op"] == "evict":
        # accumulated weights fall off as a power of their rank; many positions never got any
        u = torch.rand(case["seqs"], case["kv"], st["max_len"], generator=g, device=DEV)
        st["mass"] = torch.where(u < 0.1, torch.zeros_like(u), 0.01 / (u + 1e-4) ** 1.5)
        cap = st["cap"] = min(st["max_len"], case["budget"])
        st["mass_out"] = torch.zeros(case["seqs"], case["kv"], cap, device=DEV)
        st["kept"] = torch.zeros(case["seqs"], case["kv"], case["budget"], dtype=torch.int32, device=DEV)
        st["lens_out"] = torch.zeros(case["seqs"], dtype=torch.int32, device=DEV)
    else:
        rows = case["seqs"] if case["op"] == "decode" else st["total"]
        st["scale"] = 1.0 / math.sqrt(case["hd"])
        # scores spread by about 1.5; some positions draw most heads, as the first tokens of a text do
        st["q"] = torch.randn(rows, case["heads"], case["hd"], generator=g, device=DEV) * 1.5
        st["k"].mul_(torch.where(torch.rand(pages, case["page"], 1, 1, generator=g, device=DEV) < 0.01, 2.0, 1.0).to(st["k"].dtype))
        st["out"] = torch.empty(rows, case["heads"], case["hd"], device=DEV)
        st["slopes"] = _i32(np.zeros(1)) if not case["alibi"] else torch.tensor(
            [2.0 ** (-8.0 * (i + 1) / case["heads"]) for i in range(case["heads"])], device=DEV)
        if case.get("mass"):
            st["mass"] = torch.rand(case["seqs"], case["kv"], st["max_len"], generator=g, device=DEV)
        if case["op"] == "prompt":
            st["prefix"] = _i32([min(case["prefix"], n) for n in lens]) if case["prefix"] else None
            docs = _docs_of(case, st["max_len"])
            st["docs"] = None if docs is None else _i32(np.tile(docs, (case["seqs"], 1)))
    if own:
        _handle(st, case)
    return st


def _logit_lists(case):
    """Lengths of each row's history and bias list, and which rows follow a grammar."""
    hist = _spread(case["rows"], case["hist"] // 3, case["hist"])
    bias = [min(n, case["vocab"]) for n in _spread(case["rows"], case["bias"] // 4, case["bias"], 0.61)]
    masked = [r % 4 != 3 for r in range(case["rows"])]
    return hist, bias, masked


def _prepare_logits(case, g, st):
    rows, vocab = case["rows"], case["vocab"]
    hist, bias, masked = _logit_lists(case)
    r = np.random.default_rng(int(torch.randint(1 << 31, (1,), generator=g, device=DEV)))
    ho, bo = np.concatenate([[0], np.cumsum(hist)]), np.concatenate([[0], np.cumsum(bias)])
    # words repeat as in text: a few very often, most seldom
    history = np.minimum((r.pareto(0.7, int(ho[-1])) * 20).astype(np.int64) * 7919 % vocab, vocab - 1)
    ids = np.concatenate([r.permutation(vocab)[:n] for n in bias]) if bo[-1] else np.zeros(0, np.int64)
    rules = np.zeros((rows, 8), dtype=np.uint32)
    f = rules.view(np.float32)
    f[:, 0] = r.uniform(0.9, 1.4, rows)
    f[:, 1] = r.uniform(0.0, 0.5, rows)
    f[:, 2] = r.uniform(-0.2, 0.6, rows)
    rules[:, 3], rules[:, 4], rules[:, 5], rules[:, 6] = ho[:-1], hist, bo[:-1], bias
    number = np.cumsum(masked) - 1
    rules[:, 7] = np.where(masked, number, NO_MASK)
    words = -(-vocab // 32)
    share = torch.tensor([(0.001, 0.5, 0.98)[m % 3] for m in range(max(1, sum(masked)))], device=DEV)
    m = torch.zeros(len(share), words, dtype=torch.int64, device=DEV)
    for b in range(32):
        m |= (torch.rand(len(share), words, generator=g, device=DEV) < share[:, None]).long() << b
    st.update(logits=torch.randn(rows, vocab, generator=g, device=DEV) * 4.0, history=_i32(history), ids=_i32(ids[:int(bo[-1])]),
              values=torch.randn(int(bo[-1]), generator=g, device=DEV) * 3.0, rules=torch.as_tensor(rules.view(np.int32), device=DEV),
              masks=torch.where(m >= 1 << 31, m - (1 << 32), m).to(torch.int32), out=torch.empty(rows, vocab, device=DEV))
    return st


# ── one pass ─────────────────────────────────────────────────────────────────

def run(st):
    return (_OWN if own else _PLAIN)[st["op"]](st)


def _own_append(st):
    _ctx().paged_append(st["cfg"], st["kvh"], st["qkv"], st["total"], st["qn"], st["kn"], st["seq"], st["pos"], None,
                        st["table"], st["case"]["seqs"], st["q"])
    return {"q": st["q"], "k": st["k"], "v": st["v"]}


def _own_decode(st):
    _ctx().paged_attn_decode(st["cfg"], st["kvh"], st["q"], st["case"]["seqs"], st["table"], st["lens"], st["max_len"],
                             st["out"], st.get("mass"), st["max_len"])
    return {"out": st["out"], "mass": st["mass"]} if st["case"]["mass"] else {"out": st["out"]}


def _own_prompt(st):
    _ctx().paged_attn_prompt(st["cfg"], st["kvh"], st["q"], st["case"]["seqs"], st["cu"], st["total"], st["max_q"], st["table"],
                             st["lens"], st["max_len"], st["out"], st["prefix"], st["docs"], st["max_len"])
    return {"out": st["out"]}


def _own_evict(st):
    c = st["case"]
    _ctx().kv_evict(st["kvh"], c["seqs"], st["table"], st["lens"], st["max_len"], st["mass"], st["max_len"], c["budget"],
                    c["recent"], st["dst"], st["lens_out"], st["mass_out"], st["cap"], st["kept"])
    return _evict_outputs(st)


def _own_logits(st):
    c = st["case"]
    _ctx().logits_process(st["logits"], c["vocab"], c["rows"], st["rules"], st["history"], st["ids"], st["values"], st["masks"], st["out"])
    return {"out": st["out"]}


def _evict_outputs(st):
    d = st["first_dst"]
    return {"k": st["k"][d:], "v": st["v"][d:], "mass": st["mass_out"], "kept": st["kept"], "lens": st["lens_out"]}


def _slots(table, j, page):
    """Pool slots of positions j (any shape [S, n]) of each sequence."""
    return torch.gather(table.long(), 1, j // page) * page + j % page


def _plain_append(st):
    c, hd, half = st["case"], st["case"]["hd"], st["case"]["hd"] // 2
    T, H, kv = st["total"], c["heads"], c["kv"]
    x = st["qkv"].view(T, H + 2 * kv, hd)
    q, k, v = x[:, :H], x[:, H:H + kv], x[:, H + kv:]
    inv = lambda t: 1.0 / torch.sqrt((t * t).sum(-1, keepdim=True) / hd + EPS)  # noqa: E731
    q, k = q * inv(q) * st["qn"], k * inv(k) * st["kn"]
    v = v * inv(v) if c["v_norm"] else v
    e = torch.arange(half, device=DEV).float() * 2.0 / hd
    freq = 1.0 / torch.pow(torch.full_like(e, THETA), e)
    ang = st["pos"].float()[:, None] * freq
    cos, sin = torch.cos(ang)[:, None], torch.sin(ang)[:, None]

    def turn(t):
        a, b = (t[..., :half], t[..., half:]) if c["neox"] else (t[..., 0::2], t[..., 1::2])
        a, b = a * cos - b * sin, a * sin + b * cos
        return torch.cat([a, b], -1) if c["neox"] else torch.stack([a, b], -1).flatten(-2)

    pos, seq = st["pos"].long(), st["seq"].long()
    slot = st["table"].long()[seq, pos // c["page"]] * c["page"] + pos % c["page"]
    st["k"].view(-1, kv, hd)[slot] = turn(k).to(st["k"].dtype)
    st["v"].view(-1, kv, hd)[slot] = v.to(st["v"].dtype)
    return {"q": turn(q).reshape(T, H * hd), "k": st["k"], "v": st["v"]}


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
    c = st["case"]
    j = torch.arange(n, device=DEV).expand(c["seqs"], n)
    slot = _slots(st["table"], j, c["page"])
    return (st[x].view(-1, c["kv"], c["hd"])[slot].float().transpose(1, 2) for x in "kv")


def _plain_decode(st):
    c, n = st["case"], st["max_len"]
    S, H, kv, hd = c["seqs"], c["heads"], c["kv"], c["hd"]
    k, v = _cached(st, n)
    s = torch.matmul(st["q"].view(S, kv, H // kv, hd), k.transpose(2, 3)).view(S, H, 1, n)
    dist = (st["lens"].long()[:, None] - 1 - torch.arange(n, device=DEV)).view(S, 1, 1, n)
    seen = (dist >= 0) & ((dist < c["window"]) if c["window"] else (dist >= 0))
    p = _softmax(_scores(st, s, dist), seen).view(S, kv, H // kv, n)
    out = torch.matmul(p, v).view(S, H, hd)
    if not c["mass"]:
        return {"out": out}
    st["mass"] += p.sum(2)
    return {"out": out, "mass": st["mass"]}


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


def _plain_evict(st):
    c, n = st["case"], st["max_len"]
    S, kv, hd, budget = c["seqs"], c["kv"], c["hd"], c["budget"]
    lens = st["lens"].long()[:, None, None]
    j = torch.arange(n, device=DEV).expand(S, kv, n)
    # the newest first, then by weight, the lowest position first among equals, then what is not there
    key = torch.where(j >= lens - c["recent"], torch.full_like(st["mass"], math.inf), st["mass"])
    key = torch.where(j < lens, key, torch.full_like(key, -math.inf))
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    best = torch.sort(torch.where(torch.arange(best.shape[-1], device=DEV) < lens, best, torch.full_like(best, n)), dim=-1).values
    m = best.shape[-1]
    there = torch.arange(m, device=DEV).expand(S, kv, m) < lens
    src = torch.where(there, best, torch.zeros_like(best))
    st["kept"][..., :m] = torch.where(there, best.int(), st["kept"][..., :m])
    st["mass_out"][..., :m] = torch.where(there, torch.gather(st["mass"], 2, src), st["mass_out"][..., :m])
    st["lens_out"].copy_(st["lens"].clamp(max=budget))
    h = torch.arange(kv, device=DEV).view(1, kv, 1).expand(S, kv, m)
    frm = torch.gather(st["table"].long()[:, None].expand(S, kv, -1), 2, src // c["page"]) * c["page"] + src % c["page"]
    i = torch.arange(m, device=DEV).expand(S, kv, m)
    to = torch.gather(st["dst"].long()[:, None].expand(S, kv, -1), 2, i // c["page"]) * c["page"] + i % c["page"]
    for x in (st["k"], st["v"]):
        flat = x.view(-1, kv, hd)
        flat[to[there], h[there]] = flat[frm[there], h[there]]
    return _evict_outputs(st)


def _plain_logits(st):
    c, x = st["case"], st["logits"]
    rows, vocab = c["rows"], c["vocab"]
    rules = st["rules"]
    f = rules.view(torch.float32)
    hl, bl = rules[:, 4].long(), rules[:, 6].long()
    row = torch.repeat_interleave(torch.arange(rows, device=DEV), hl)
    count = torch.zeros(rows, vocab, device=DEV).index_put_((row, st["history"].long()), torch.ones(len(row), device=DEV), accumulate=True)
    y = torch.where(x > 0, x / f[:, :1], x * f[:, :1]) - (count * f[:, 1:2] + f[:, 2:3])
    y = torch.where(count > 0, y, x)
    if len(st["ids"]):
        add = torch.zeros_like(x).index_put_((torch.repeat_interleave(torch.arange(rows, device=DEV), bl), st["ids"].long()), st["values"])
        y = y + add
    t = torch.arange(vocab, device=DEV)
    which = rules[:, 7]
    ok = (st["masks"][which.clamp(min=0).long()][:, t // 32] >> (t % 32).int()) & 1
    return {"out": torch.where((which[:, None] < 0) | (ok == 1), y, torch.full_like(y, -math.inf))}


_OWN = {"append": _own_append, "decode": _own_decode, "prompt": _own_prompt, "evict": _own_evict, "logits": _own_logits}
_PLAIN = {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt, "evict": _plain_evict, "logits": _plain_logits}


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
    op = case["op"]
    if op == "logits":
        hist, bias, masked = _logit_lists(case)
        cells = case["rows"] * case["vocab"]
        return {"bytes": 8 * cells + sum(masked) * case["vocab"] / 8 + 4 * sum(hist) + 8 * sum(bias) + 32 * case["rows"], "flops": 4 * cells}
    size = 2 if case["f16"] else 4
    token = case["kv"] * case["hd"]
    if op == "append":
        new, _ = _new_past(case)
        row = case["heads"] * case["hd"]
        return {"bytes": sum(new) * (4 * (row + 2 * token) + 4 * row + 2 * size * token + 12), "flops": sum(new) * 10 * (row + token)}
    if op == "decode":
        lens = _spread(case["seqs"], case["lo"], case["hi"])
        seen = sum(min(n, case["window"]) if case["window"] else n for n in lens)
        b = seen * token * size * 2 + 8 * case["seqs"] * case["heads"] * case["hd"] + 4 * seen / case["page"]
        return {"bytes": b + (8 * seen * case["kv"] if case["mass"] else 0), "flops": 4 * seen * case["heads"] * case["hd"]}
    if op == "prompt":
        new, past = _new_past(case)
        pairs, keys = _pairs(case, new, [a + b for a, b in zip(new, past)])
        return {"bytes": 8 * sum(new) * case["heads"] * case["hd"] + 2 * keys * token * size, "flops": 4 * pairs * case["heads"] * case["hd"]}
    lens = _spread(case["seqs"], case["lo"], case["hi"])
    kept = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": 4 * case["kv"] * sum(lens) + kept * (4 * token * size + 8 * case["kv"]), "flops": 0}


# ── the definitions in 64 bits ───────────────────────────────────────────────

def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed), case)


def _exact_append(st, c):
    hd, H, kv = c["hd"], c["heads"], c["kv"]
    k, v = st["k"].double(), st["v"].double()
    x = st["qkv"].double().reshape(st["total"], H + 2 * kv, hd)
    rms = (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    i = torch.arange(0, hd, 2, device=DEV, dtype=torch.float64)
    z = torch.polar(torch.ones(st["total"], hd // 2, device=DEV, dtype=torch.float64), st["pos"].double()[:, None] * THETA ** (-i / hd))
    pair = (torch.arange(hd // 2, device=DEV), torch.arange(hd // 2, device=DEV) + hd // 2) if c["neox"] else (i.long(), i.long() + 1)

    def turned(t):
        w = torch.complex(t[..., pair[0]], t[..., pair[1]]) * z[:, None]
        o = torch.empty_like(t)
        o[..., pair[0]], o[..., pair[1]] = w.real, w.imag
        return o

    y = turned(x[:, :H + kv] * rms[:, :H + kv] * torch.cat([st["qn"].double().expand(H, hd), st["kn"].double().expand(kv, hd)]))
    at = st["table"].cpu().numpy()[st["seq"].cpu().numpy(), st["pos"].cpu().numpy() // c["page"]]
    at, inside = torch.as_tensor(at, device=DEV).long(), st["pos"].long() % c["page"]
    k[at, inside] = y[:, H:]
    v[at, inside] = x[:, H + kv:] * (rms[:, H + kv:] if c["v_norm"] else 1.0)
    return {"q": y[:, :H].reshape(st["total"], -1), "k": k, "v": v}


def _exact_rows(st, c, s, h, queries, i, n, keep):
    """Attention of queries [m, hd] at positions i [m] of head h of sequence s over its first n cached positions."""
    pages = st["table"][s, :-(-n // c["page"])].long()
    kh = h // (c["heads"] // c["kv"])
    K, V = (st[x][pages, :, kh].double().reshape(-1, c["hd"])[:n] for x in "kv")
    t = queries.double() @ K.T / math.sqrt(c["hd"])
    t = c["softcap"] * torch.tanh(t / c["softcap"]) if c["softcap"] else t
    if c["alibi"]:
        t = t - 2.0 ** (-8.0 * (h + 1) / c["heads"]) * (i[:, None] - torch.arange(n, device=DEV)).abs()
    t = t.masked_fill(~keep, -math.inf)
    e = torch.exp(t - t.amax(1, keepdim=True).nan_to_num(neginf=0.0))
    p = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    return p, p @ V


def _exact_decode(st, c):
    out = torch.zeros_like(st["out"], dtype=torch.float64)
    mass = st["mass"].double() if c["mass"] else None
    for s, n in enumerate(st["lens"].tolist()):
        if n == 0:
            continue
        i = torch.tensor([n - 1], device=DEV)
        keep = torch.ones(1, n, dtype=torch.bool, device=DEV)
        if c["window"]:
            keep[0, :max(0, n - c["window"])] = False
        for h in range(c["heads"]):
            p, out[s, h:h + 1] = _exact_rows(st, c, s, h, st["q"][s, h:h + 1], i, n, keep)
            if mass is not None:
                mass[s, h // (c["heads"] // c["kv"]), :n] += p[0]
    return {"out": out} if mass is None else {"out": out, "mass": mass}


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
            out[first:first + m, h] = _exact_rows(st, c, s, h, st["q"][first:first + m, h], i, n, keep)[1]
        first += m
    return {"out": out}


def _exact_evict(st, c):
    K, V, M = st["k"].double(), st["v"].double(), st["mass_out"].double()
    mass = st["mass"].cpu().numpy()
    table, dst, kept, lens = (st[x].cpu().numpy() for x in ("table", "dst", "kept", "lens"))
    for s, n in enumerate(lens.tolist()):
        m = min(n, c["budget"])
        for h in range(c["kv"]):
            old = max(0, n - c["recent"]) if n > m else n
            # what is not among the newest: heaviest first, then lowest position
            order = np.lexsort((np.arange(old), -mass[s, h, :old].astype(np.float64)))[:m - (n - old)]
            keep = np.concatenate([np.sort(order), np.arange(old, n)]).astype(np.int64)
            kept[s, h, :m] = keep
            M[s, h, :m] = torch.as_tensor(mass[s, h, keep], device=DEV).double()
            a, b = (torch.as_tensor(t[s, x // c["page"]].astype(np.int64) * c["page"] + x % c["page"], device=DEV)
                    for t, x in ((table, keep), (dst, np.arange(m))))
            for x in (K, V):
                x.view(-1, c["kv"], c["hd"])[b, h] = x.view(-1, c["kv"], c["hd"])[a, h]
    d = st["first_dst"]
    return {"k": K[d:], "v": V[d:], "mass": M, "kept": kept, "lens": np.minimum(lens, c["budget"])}


def _exact_logits(st, c):
    rules = st["rules"].cpu().numpy()
    f, u = rules.view(np.float32).astype(np.float64), rules.view(np.uint32)
    x = st["logits"].cpu().numpy().astype(np.float64)
    history, ids, values = st["history"].cpu().numpy(), st["ids"].cpu().numpy(), st["values"].cpu().numpy().astype(np.float64)
    masks = st["masks"].cpu().numpy().view(np.uint32)
    for r in range(c["rows"]):
        a, n, b, m = (int(u[r, k]) for k in (3, 4, 5, 6))
        tok, times = np.unique(history[a:a + n], return_counts=True)
        y = x[r, tok]
        x[r, tok] = np.where(y > 0, y / f[r, 0], y * f[r, 0]) - f[r, 1] * times - f[r, 2]
        x[r, ids[b:b + m]] += values[b:b + m]
        if u[r, 7] != NO_MASK:
            bits = np.unpackbits(masks[u[r, 7]].view(np.uint8), bitorder="little")[:c["vocab"]]
            x[r, bits == 0] = -math.inf
    return {"out": x}


_EXACT = {"append": _exact_append, "decode": _exact_decode, "prompt": _exact_prompt, "evict": _exact_evict, "logits": _exact_logits}

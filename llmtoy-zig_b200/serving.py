"""Greedy decoding of many sequences over one paged cache.

    dec = BatchDecoder(ctx, upload_decoder(ctx, model, kv_f16=True), max_seqs=8, max_len=4096)
    streams = dec.generate([[1, 2, 3], [7, 8]], n_gen=32)

The prompts of a batch run together: one pass over all their tokens
(lt_paged_append, lt_paged_attn_prompt), then one token per sequence and step
(lt_paged_attn_decode), the logits under each request's rules
(lt_logits_process).  With a budget, the cache of a sequence that outgrows it is
cut to its heaviest and newest positions (lt_kv_evict), whose weights the decode
steps accumulate.  The models are those of decoder.ModelSpec's LLAMA family with
stacked Q/K/V rows (Qwen2, Qwen3, Qwen3-MoE shapes); every other op is the one
the single-sequence decoder uses, on several rows.
"""
from __future__ import annotations

from contextlib import contextmanager
from dataclasses import dataclass, field

from . import AttnCfg, Context, LogitRule, NO_MASK, PagedAttnCfg, PagedKV
from .decoder import LLAMA, ModelSpec


@dataclass
class Request:
    """A prompt and what it asks of its logits."""
    prompt: list
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    bias: dict = field(default_factory=dict)   # token id -> added to its logit
    allowed: list | None = None                # token ids that may be chosen (a grammar's state); None: all


class PagePool:
    """Pages of one cache, handed out and taken back by number."""

    def __init__(self, n_pages: int):
        self.free = list(range(n_pages - 1, -1, -1))

    def take(self, n: int) -> list[int]:
        if n > len(self.free):
            raise MemoryError(f"{n} cache pages wanted, {len(self.free)} free")
        return [self.free.pop() for _ in range(n)]

    def give(self, pages: list[int]) -> None:
        self.free.extend(reversed(pages))


class BatchDecoder:
    """max_seqs sequences of up to max_len cached positions each; budget > 0: at most that many stay cached
    after a step, the newest `recent` among them."""

    def __init__(self, ctx: Context, spec: ModelSpec, max_seqs: int, max_len: int, page_size: int = 16, n_pages: int = 0,
                 budget: int = 0, recent: int = 0):
        import torch
        if spec.family != LLAMA or any(L.wqkv is None for L in spec.layers):
            raise ValueError("BatchDecoder takes LLAMA-family models with stacked Q/K/V rows")
        if budget and not 0 <= recent < budget <= max_len:
            raise ValueError("0 <= recent < budget <= max_len")
        self.ctx, self.spec, self.max_seqs, self.page = ctx, spec, max_seqs, page_size
        self.budget, self.recent, self.max_len = budget, recent, max_len
        s = self.spec
        self.width = -(-max_len // page_size)
        self.n_pages = n_pages or max_seqs * self.width
        self.pool = PagePool(self.n_pages)
        self.pages = []  # of each sequence
        kind = torch.float16 if s.kv_f16 else torch.float32
        shape = (self.n_pages, page_size, s.n_kv_heads, s.head_dim)
        torch.cuda.synchronize()
        self.emb = torch.empty(s.vocab, s.d_model, device="cuda")
        ctx.dequant(s.token_emb, 0, s.vocab, self.emb)
        self.cfg = AttnCfg(s.n_heads, s.n_kv_heads, s.head_dim, int(s.rope_neox), s.rope_theta, s.eps, s.head_dim ** -0.5, 1)
        self.attn = PagedAttnCfg(n_heads=s.n_heads, causal=1, scale=s.head_dim ** -0.5)
        self.caches, self.mass, self.biases = [], [], []
        for L in s.layers:
            k, v = torch.zeros(shape, dtype=kind, device="cuda"), torch.zeros(shape, dtype=kind, device="cuda")
            kv = PagedKV(n_kv_heads=s.n_kv_heads, head_dim=s.head_dim, kv_f16=int(s.kv_f16), page_size=page_size,
                         n_pages=self.n_pages, max_pages=self.width, k=k.data_ptr(), v=v.data_ptr())
            self.caches.append((kv, k, v))
            self.mass.append(torch.zeros(max_seqs, s.n_kv_heads, max_len, device="cuda") if budget else None)
            b = None if L.qkv_bias is None else L.qkv_bias.contiguous()  # read 16 bytes at a time
            self.biases.append(b if b is None or b.data_ptr() % 16 == 0 else b.clone())
        torch.cuda.synchronize()

    @contextmanager
    def _between(self):
        """What runs in here allocates with torch and launches on the context's stream only.  torch hands a block out
        again in the order of its own stream, so all work, whosever, ends before and after; in between no torch kernel
        runs while the context's stream has work, and blocks change hands in the order of that stream."""
        import torch
        torch.cuda.synchronize()
        try:
            yield
        finally:
            torch.cuda.synchronize()

    def _dev(self, values, dtype="uint32"):
        """A host list as a device array (torch tensor of its bits)."""
        import numpy as np
        import torch
        a = np.ascontiguousarray(np.asarray(values).astype(dtype))
        t = torch.empty(max(1, a.size), dtype=torch.float32 if dtype == "float32" else torch.int32, device="cuda")
        if a.size:
            self.ctx.copy_to_device(t, a)
        return t

    def _layers(self, x, ntok: int, seq, pos, slot, attend) -> None:
        """x[ntok][d_model] <- the decoder layers; attend(layer, q, out) is the batch's attention."""
        import torch
        ctx, s = self.ctx, self.spec
        nq, nkv = s.n_heads * s.head_dim, s.n_kv_heads * s.head_dim
        xn, qkv = torch.empty_like(x), torch.empty(ntok, nq + 2 * nkv, device="cuda")
        q, att = torch.empty(ntok, nq, device="cuda"), torch.empty(ntok, nq, device="cuda")
        bias = zeros = None
        for i, L in enumerate(s.layers):
            ctx.rmsnorm(x, L.attn_norm, s.eps, s.d_model, ntok, xn)
            if self.biases[i] is None:
                ctx.qmatvec(L.wqkv, xn, qkv, ntok)
            else:
                if bias is None:
                    bias, zeros = torch.empty_like(qkv), self._dev([0] * ntok)
                ctx.gather_rows(self.biases[i], nq + 2 * nkv, zeros, ntok, bias)  # its one row for every token
                ctx.qmatvec_add(L.wqkv, xn, bias, qkv, ntok)
            ctx.paged_append(self.cfg, self.caches[i][0], qkv, ntok, L.q_norm, L.k_norm, seq, pos, slot, self.table,
                             self.n_seq, q)
            attend(i, q, att)
            ctx.qmatvec_add(L.wo, att, x, x, ntok)
            if L.router is None:
                ctx.ffn_block(L.ffn_gate, L.ffn_up, L.ffn_down, s.act, L.ffn_norm, s.eps, x, ntok, x)
            else:
                ctx.moe_block(L.router, L.exp_gate, L.exp_up, L.exp_down, s.act, s.norm_topk, None, L.ffn_norm, s.eps, x,
                              ntok, s.n_used, x)

    def _choose(self, x, rows) -> list[int]:
        """The next token of every sequence from rows `rows` of x."""
        import torch
        ctx, s, n = self.ctx, self.spec, self.n_seq
        last, xn = torch.empty(n, s.d_model, device="cuda"), torch.empty(n, s.d_model, device="cuda")
        self.logits, ids = torch.empty(n, s.vocab, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
        ctx.gather_rows(x, s.d_model, self._dev(rows), n, last)
        ctx.rmsnorm(last, s.out_norm, s.eps, s.d_model, n, xn)
        ctx.qmatvec(s.lm_head, xn, self.logits, n)
        rules, history, bias_ids, bias_values, masks = self._rules()
        ctx.logits_process(self.logits, s.vocab, n, rules, history, bias_ids, bias_values, masks, self.logits)
        ctx.argmax(self.logits, s.vocab, n, ids)
        return ctx.copy_to_host(ids, 4 * n, "uint32").tolist()

    def _rules(self):
        import numpy as np
        rules, history, ids, values, masks = (LogitRule * self.n_seq)(), [], [], [], []
        for r, q in enumerate(self.requests):
            mask = NO_MASK
            if q.allowed is not None:
                mask = len(masks)
                words = np.zeros((self.spec.vocab + 31) // 32, np.uint32)
                a = np.asarray([t for t in q.allowed if t < self.spec.vocab], np.int64)
                np.bitwise_or.at(words, a // 32, (np.uint32(1) << (a % 32).astype(np.uint32)))
                masks.append(words)
            rules[r] = LogitRule(q.repetition, q.frequency, q.presence, len(history), len(self.tokens[r]), len(ids),
                                 len(q.bias), mask)
            history += self.tokens[r]
            ids += q.bias.keys()
            values += q.bias.values()
        return (self._dev(np.frombuffer(rules, np.uint32)), self._dev(history), self._dev(ids), self._dev(values, "float32"),
                self._dev(np.concatenate(masks)) if masks else None)

    def _checked(self, requests: list) -> list:
        """The requests, or ValueError.  Prompt ids index the embedding on the device, which takes them as they are.
        Ids past the vocabulary in bias and allowed name no token and are skipped."""
        requests = [q if isinstance(q, Request) else Request(list(q)) for q in requests]
        new = [len(q.prompt) for q in requests]
        if not 0 < len(new) <= self.max_seqs or not 0 < min(new) <= max(new) < self.max_len:
            raise ValueError("1 .. max_seqs prompts of 1 .. max_len - 1 tokens")
        vocab = self.spec.vocab
        for r, q in enumerate(requests):
            bad = [t for t in q.prompt if not 0 <= t < vocab]
            if bad:
                raise ValueError(f"request {r}: prompt token {bad[0]} of a vocabulary of {vocab}")
            if q.allowed is not None and (any(t < 0 for t in q.allowed) or not any(t < vocab for t in q.allowed)):
                raise ValueError(f"request {r}: allowed tokens are negative or leave nothing of the vocabulary")
        return requests

    def start(self, requests: list) -> list[int]:
        """Run the prompts; the first token of each sequence.  The batch before gives its pages back; a batch that is
        refused (ValueError, MemoryError) leaves it as it was."""
        requests = self._checked(requests)
        new = [len(q.prompt) for q in requests]
        need = [-(-n // self.page) for n in new]
        there = len(self.pool.free) + sum(len(p) for p in self.pages)
        if sum(need) > there:
            raise MemoryError(f"{sum(need)} cache pages wanted, {there} free")
        self.close()
        self.requests = requests
        self.n_seq, self.tokens = len(requests), [list(q.prompt) for q in self.requests]
        for m in self.mass:
            if m is not None:
                m.zero_()
        self.pages = [self.pool.take(n) for n in need]
        self.lens, self.pos = list(new), list(new)  # cached positions; the next token's place in the text
        with self._between():
            return self._take(self._prompts(new))

    def _prompts(self, new: list[int]) -> list[int]:
        import torch
        self._tables()
        cu = [sum(new[:i]) for i in range(self.n_seq + 1)]
        seq = self._dev([r for r, n in enumerate(new) for _ in range(n)])
        pos = self._dev([j for n in new for j in range(n)])
        dcu, total, most = self._dev(cu), cu[-1], max(new)
        x = torch.empty(total, self.spec.d_model, device="cuda")
        self.ctx.gather_rows(self.emb, self.spec.d_model, self._dev([t for s in self.tokens for t in s]), total, x)
        self._layers(x, total, seq, pos, None, lambda i, q, out: self.ctx.paged_attn_prompt(
            self.attn, self.caches[i][0], q, self.n_seq, dcu, total, most, self.table, self.dlens, most, out))
        return self._choose(x, [c - 1 for c in cu[1:]])

    def step(self) -> list[int]:
        """One more token of every sequence."""
        if not self.pages:
            raise ValueError("no batch is running: start one first")
        for r in range(self.n_seq):
            if self.lens[r] >= self.max_len:
                raise ValueError(f"sequence {r} is at max_len")
            if self.lens[r] % self.page == 0 and self.lens[r] // self.page == len(self.pages[r]):
                self.pages[r] += self.pool.take(1)
        with self._between():
            ids = self._next()
            if self.budget and max(self.lens) > self.budget:
                self._evict()
        return self._take(ids)

    def _next(self) -> list[int]:
        import torch
        n = self.n_seq
        seq, pos, slot = self._dev(range(n)), self._dev(self.pos), self._dev(self.lens)
        self.lens = [v + 1 for v in self.lens]
        self.pos = [v + 1 for v in self.pos]
        self._tables()
        x = torch.empty(n, self.spec.d_model, device="cuda")
        self.ctx.gather_rows(self.emb, self.spec.d_model, self._dev([t[-1] for t in self.tokens]), n, x)
        self._layers(x, n, seq, pos, slot, lambda i, q, out: self.ctx.paged_attn_decode(
            self.attn, self.caches[i][0], q, n, self.table, self.dlens, max(self.lens), out, self.mass[i], self.max_len))
        return self._choose(x, range(n))

    def _evict(self) -> None:
        import torch
        out = torch.empty(self.n_seq, dtype=torch.int32, device="cuda")
        for (kv, _, _), m in zip(self.caches, self.mass):
            self.ctx.kv_evict(kv, self.n_seq, self.table, self.dlens, max(self.lens), m, self.max_len, self.budget, self.recent,
                              None, out, m, self.max_len)
        self.ctx.sync()  # nothing is under way on the context's stream while torch clears these
        for m in self.mass:  # slots that the coming tokens take start from nothing
            m[:, :, self.budget:] = 0
        torch.cuda.synchronize()
        self.lens = [min(v, self.budget) for v in self.lens]
        for r, v in enumerate(self.lens):
            keep = -(-v // self.page)
            self.pool.give(self.pages[r][keep:])
            self.pages[r] = self.pages[r][:keep]

    def _tables(self) -> None:
        self.table = self._dev([p for pages in self.pages for p in pages + [NO_MASK] * (self.width - len(pages))])
        self.dlens = self._dev(self.lens)

    def _take(self, ids: list[int]) -> list[int]:
        for t, i in zip(self.tokens, ids):
            t.append(i)
        return ids

    def close(self) -> None:
        """Give the batch's pages back."""
        for pages in self.pages:
            self.pool.give(pages)
        self.pages = []

    def generate(self, requests: list, n_gen: int) -> list[list[int]]:
        """n_gen new token ids per request."""
        if n_gen < 1:
            raise ValueError("n_gen: at least one token")
        try:
            out = [[t] for t in self.start(requests)]
            for _ in range(n_gen - 1):
                for o, t in zip(out, self.step()):
                    o.append(t)
        finally:
            self.close()
        return out

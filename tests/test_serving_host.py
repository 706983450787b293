"""What serving.BatchDecoder decides on the host: which requests it takes, and whose pages are
whose.  No device is used: a refused request is
refused before anything is launched."""
from __future__ import annotations

import importlib
from contextlib import nullcontext
from types import SimpleNamespace

import pytest

VOCAB = 100


def serving():
    return importlib.import_module("llmtoy-zig_b200.serving")


def decoder(max_seqs=3, max_len=16, n_pages=6, page=4):
    """A BatchDecoder without its device arrays."""
    s = serving()
    d = s.BatchDecoder.__new__(s.BatchDecoder)
    d.ctx, d.spec = None, SimpleNamespace(vocab=VOCAB)
    d.max_seqs, d.max_len, d.page, d.n_pages = max_seqs, max_len, page, n_pages
    d.budget, d.recent, d.mass, d.width = 0, 0, [], -(-max_len // page)
    d.pool, d.pages = s.PagePool(n_pages), []
    d._between = nullcontext
    d._prompts = lambda new: [1] * len(new)

    def one_more():
        d.lens = [n + 1 for n in d.lens]
        return [1] * d.n_seq
    d._next = one_more
    return d


@pytest.mark.parametrize("request_kw", [
    dict(prompt=[0, VOCAB]), dict(prompt=[-1]), dict(prompt=[1 << 40]), dict(prompt=[]), dict(prompt=[1] * 16),
    dict(prompt=[1], allowed=[]), dict(prompt=[1], allowed=[VOCAB]), dict(prompt=[1], allowed=[5, -1])])
def test_requests_out_of_range_are_refused(request_kw):
    d, s = decoder(), serving()
    with pytest.raises(ValueError):
        d.start([s.Request([3]), s.Request(**request_kw)])
    assert len(d.pool.free) == d.n_pages


def test_number_of_requests():
    d = decoder()
    for n in (0, 4):
        with pytest.raises(ValueError):
            d.start([[1]] * n)
    assert [q.prompt for q in d._checked([[1], (0, VOCAB - 1)])] == [[1], [0, VOCAB - 1]]
    ok = serving().Request([1], bias={0: 1.0, VOCAB: 2.0}, allowed=[VOCAB - 1, VOCAB + 40])
    assert d._checked([ok]) == [ok]


def test_ids_past_the_vocabulary_allow_nothing():
    import numpy as np
    d, s = decoder(), serving()
    d._dev = lambda values, dtype="uint32": np.asarray(values)
    d.n_seq, d.tokens = 1, [[1]]
    d.requests = d._checked([s.Request([1], allowed=[3, VOCAB - 1, VOCAB, VOCAB + 40])])
    bits = np.unpackbits(d._rules()[4].astype(np.uint32).view(np.uint8), bitorder="little")
    assert np.flatnonzero(bits).tolist() == [3, VOCAB - 1]


# ── pages ────────────────────────────────────────────────────────────────────

def held(d):
    pages = [p for s in d.pages for p in s]
    assert sorted(pages + d.pool.free) == list(range(d.n_pages))  # none lost, none twice
    return len(pages)


def test_refused_batch_leaves_the_pool_as_it_was():
    d = decoder(n_pages=6, page=4)
    for _ in range(3):
        with pytest.raises(MemoryError):
            d.start([[1] * 9, [1] * 9, [1] * 3])  # 3 + 3 + 1 pages
        assert held(d) == 0
        with pytest.raises(MemoryError):
            d.generate([[1] * 9, [1] * 9, [1] * 3], 2)
        assert held(d) == 0
    d.start([[1] * 9, [1] * 9])
    assert held(d) == 6


def test_start_replaces_the_batch():
    d = decoder(n_pages=6, page=4)
    d.start([[1] * 9, [1] * 9])
    d.start([[1] * 12, [1] * 5, [1]])  # as many pages as the batch before gives back
    assert held(d) == 6
    pages, tokens = [list(p) for p in d.pages], [list(t) for t in d.tokens]
    for bad in ([[1] * 15, [1] * 9], [[VOCAB]], [[1]] * 4):  # refused: the running batch goes on
        with pytest.raises((MemoryError, ValueError)):
            d.start(bad)
        assert (d.pages, d.tokens, d.n_seq) == (pages, tokens, 3) and held(d) == 6
    d.close()
    assert held(d) == 0
    d.close()
    assert held(d) == 0


@pytest.mark.parametrize("what", ["pool", "max_len", "device"])
def test_generate_gives_the_pages_back_when_it_fails(what):
    d = decoder(n_pages=4, page=4, max_len=16)
    if what == "device":
        def broken():
            raise RuntimeError("launch failed")
        d._next = broken
    with pytest.raises({"pool": MemoryError, "max_len": ValueError, "device": RuntimeError}[what]):
        d.generate([[1] * 7, [1] * 7] if what == "pool" else [[1] * 14], 8)
    assert held(d) == 0
    assert len(d.generate([[1] * 7], 1)[0]) == 1 and held(d) == 0


def test_step_without_a_batch_is_refused():
    """Its page table would be empty."""
    d = decoder()
    with pytest.raises(ValueError):
        d.step()
    d.start([[1, 2]])
    d.step()
    d.close()
    with pytest.raises(ValueError):
        d.step()


def test_number_of_generated_tokens():
    d = decoder(max_len=32, n_pages=8)
    for n in (1, 2, 7):
        assert [len(t) for t in d.generate([[1], [2, 3]], n)] == [n, n]
    for n in (0, -1):
        with pytest.raises(ValueError):
            d.generate([[1]], n)

"""What serving.BatchDecoder decides on the host: which requests it takes.  No device is used: a refused request is
refused before anything is launched."""
from __future__ import annotations

import importlib
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
    d.pool = s.PagePool(n_pages)
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

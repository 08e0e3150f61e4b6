"""Which lengths a BlockCache may be taken back to: what the host knows of the ring of bf16 rows, against a model of the ring
(no GPU needed)."""
import random

import pytest
import torch

from w8a8 import cache


def made():
    """A BlockCache without its memory: nothing is launched here."""
    c = cache.BlockCache.__new__(cache.BlockCache)
    c.KV, c.capacity, c.D, c.dtype = 1, 4096, 128, torch.int8
    c.data = torch.zeros(16, dtype=torch.uint8)
    c._ring, c._made = [None, None, c.data._version, True], c.data
    return c


class Model:
    """The ring's contents and the rows that the cache is meant to hold."""

    def __init__(self):
        self.ring, self.rows, self.next = {}, [], 0

    def append(self, n, m):
        del self.rows[n:]
        first, last = n // 64, (n + m - 1) // 64
        for at in range(n, n + m):
            self.rows.append(self.next)
            if at // 64 >= last - 1:
                self.ring[at // 64 % 2, at % 64] = self.next
            self.next += 1
        return first, last

    def holds(self, n):
        return all(self.ring.get((n // 64 % 2, r)) == self.rows[n // 64 * 64 + r] for r in range(n % 64))


def test_known_lengths(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    rng = random.Random(1)
    lost = kept = 0
    for _ in range(40):
        c, model = made(), Model()
        for step in range(60):
            n = len(model.rows)
            if step and rng.random() < 0.5:
                n = rng.choice([rng.randint(0, n), max(0, n - rng.randint(0, 150)), n // 64 * 64])
            ok = model.holds(n)
            assert (c._lost(n) is None) == ok
            lost, kept = lost + (not ok), kept + ok
            if not ok:
                n = n // 64 * 64
                assert c._lost(n) is None
            m = rng.choice([1, rng.randint(1, 20), rng.randint(1, 300)])
            if n + m > 4000:
                continue
            model.append(n, m)
            c._appended(n, m)
            assert c._lost(n + m) is None
            for x in range(max(0, n + m - 70), n + m + 1):
                assert (c._lost(x) is None) == model.holds(x), (n, m, x)
    assert lost > 100 and kept > 100


def test_refused(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    c = made()
    c._appended(0, 600)
    c._appended(128, 10)
    k = torch.zeros(1, 10, 128, dtype=torch.bfloat16)
    for f, args in ((cache.append, (c, k, k, 100)), (cache.append, (c, k, k, 127)), (cache.read, (c, 0, 100)), (cache.read, (c, 99, 100))):
        with pytest.raises(ValueError, match="block 1"):
            f(*args)
    cache.append(c, k[:, :0], k[:, :0], 100)  # nothing is put there, nothing read
    for n in (0, 64, 128, 129, 138):
        assert c._lost(n) is None
    c._appended(64, 20)
    assert c._lost(84) is None and c._lost(70) is None


def test_unknown_lengths(monkeypatch):
    """Where the host does not know what the memory holds, nothing is refused."""
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])

    def went_back():
        c = made()
        c._appended(0, 600)
        c._appended(128, 10)
        assert c._lost(100) is not None
        return c
    c = went_back()
    c.data.copy_(torch.ones(16, dtype=torch.uint8))   # another cache's contents
    assert c._lost(100) is None
    c._appended(100, 5)                               # .. and known again from here on
    assert c._lost(103) is None
    c._appended(100, 600)
    assert c._lost(103) is not None and c._lost(699) is None
    c = went_back()
    c.data = torch.zeros(16, dtype=torch.uint8)       # other memory
    assert c._lost(100) is None
    c._appended(0, 600)
    assert c._lost(100) is None
    c = went_back()
    c._appended(torch.zeros(1, dtype=torch.int32), 5)  # a length in device memory
    assert c._lost(100) is None
    c._appended(0, 600)
    assert c._lost(100) is None
    c = went_back()
    capturing[0] = True                               # a captured append comes again with every replay
    c._appended(10, 5)
    capturing[0] = False
    assert c._lost(100) is None
    c._appended(0, 600)
    assert c._lost(100) is None
    assert went_back()._lost(torch.zeros(1, dtype=torch.int32)) is None

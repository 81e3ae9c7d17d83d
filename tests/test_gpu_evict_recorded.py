"""Evictions of more than 8192 rows in recordings: replays with new weights, with other calls between
them, and the refusal of one that finds no scratch."""
import numpy as np
import pytest

import long_cache_reference as ref
from test_gpu_evict import weights
from test_gpu_scratch import fresh

pytestmark = pytest.mark.gpu


class Eviction:
    def __init__(self, g4, sets, n, keep, first, recent, place):
        self.g4, self.args, self.place = g4, (sets, n, keep, first, recent), place
        self.w, self.rows = g4.Buffer(sets * n * 4), g4.Buffer(sets * keep * 4)
        self.kept = self.w if place else g4.Buffer(sets * n * 4)

    def fill(self, w):
        self.now = w
        self.w.upload(w)
        self.rows.upload(np.full(self.rows.nbytes // 4, -1, np.int32))

    def __call__(self):
        self.g4.cache_evict(self.w, *self.args, self.rows, self.kept)

    def check(self):
        sets, n, keep, first, recent = self.args
        rows = self.rows.download(np.int32).reshape(sets, keep)
        kept = self.kept.download(np.uint32).reshape(sets, n)
        for s in range(sets):
            r, k = ref.evict(self.now[s], keep, first, recent)
            np.testing.assert_array_equal(rows[s], r)
            np.testing.assert_array_equal(kept[s], k.view(np.uint32))


@pytest.mark.parametrize("place", [False, True])
@pytest.mark.parametrize("sets,n,keep,first,recent", [
    (1, 8193, 5000, 4, 100), (3, 20000, 6000, 4, 128), (1, 131072, 32768, 4, 512), (2, 30000, 0, 0, 0)])
def test_replays_with_new_weights(g4, sets, n, keep, first, recent, place):
    rng = np.random.default_rng([sets, n])
    e = Eviction(g4, sets, n, keep, first, recent, place)
    e.fill(weights(rng, sets, n))
    e()
    with g4.Encoder() as enc:
        e()
    for turn in range(5):
        e.fill(weights(rng, sets, n) if turn % 2 else rng.integers(0, 40, (sets, n)).astype(np.float32))
        enc.cmdbuf.submit()
        e.check()
        if turn > 1:  # eager calls of other sizes between the replays
            other = Eviction(g4, 1 + turn % 2, 9000 + 20000 * turn, 3000, 1, 2, not place)
            other.fill(weights(rng, 1 + turn % 2, 9000 + 20000 * turn))
            other()
            other.check()
        if turn == 3:
            g4.sync()


def test_two_recordings_share_scratch(g4):
    rng = np.random.default_rng(7)
    calls = [Eviction(g4, 1, 50000, 20000, 4, 64, False), Eviction(g4, 4, 12000, 3000, 0, 300, True)]
    recs = []
    for e in calls:
        e.fill(weights(rng, e.args[0], e.args[1]))
        e()
        with g4.Encoder() as enc:
            e()
        recs.append(enc.cmdbuf)
    for turn in range(4):
        for e in calls:
            e.fill(weights(rng, e.args[0], e.args[1]))
        for rec in recs if turn % 2 else recs[::-1]:
            rec.submit()
        for e in calls:
            e.check()


def test_a_recording_without_an_earlier_call_is_refused():
    fresh("""
w, rows = g4.Buffer(20000 * 4), g4.Buffer(20000 * 4)
def refused(n):
    with g4.Encoder():
        try:
            g4.cache_evict(w, 1, n, n // 2, 4, 8, rows, w)
        except g4.G4Error as e:
            return e.code == g4.G4_E_STATE
    return False
assert refused(20000)
g4.cache_evict(w, 1, 9000, 100, 4, 8, rows, w)
assert refused(20000)
x = np.arange(20000, dtype=np.float32)
w.upload(x)
g4.cache_evict(w, 1, 20000, 10000, 4, 8, rows, w)
with g4.Encoder() as enc:
    g4.cache_evict(w, 1, 20000, 10000, 4, 8, rows, w)
for _ in range(3):
    w.upload(x)
    enc.cmdbuf.submit()
    assert (rows.download(np.int32, 10000) == np.concatenate([np.arange(4), np.arange(10004, 20000)])).all()
""")

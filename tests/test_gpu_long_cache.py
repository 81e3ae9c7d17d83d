"""The operators of long caches together: a chat whose caches are trimmed as it goes, over FP32 rows
and over rows of 4 bits, eager, recorded and through Node.

Tolerances as in test_gpu_kv4.py and test_gpu_attention_weights.py: 2e-5 of max |v| for outputs, 2e-5
of a key's weight per call."""
import json
import os
import shutil
import subprocess
import sys

import numpy as np
import pytest

import long_cache_reference as ref

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOL, HEADS = 2e-5, 8


class Chat:
    """One layer's cache: FP32 rows or 4 bits, its weights, and the same on the host."""

    def __init__(self, g4, hd, cap, quantised):
        self.g4, self.hd, self.cap, self.quantised, self.len = g4, hd, cap, quantised, 0
        if quantised:
            self.cache = g4.Kv4Cache(cap, hd)
            bufs, widths = self.cache.planes()
        else:
            self.k, self.v = g4.Buffer(cap * hd * 4), g4.Buffer(cap * hd * 4)
            bufs, widths = [self.k, self.v], [hd, hd]
        self.planes = g4.CachePlanes(bufs, bufs, widths)
        self.w, self.rows = g4.Buffer(cap * 4), g4.Buffer(cap * 4)
        self.kh, self.vh, self.wh = np.zeros((cap, hd)), np.zeros((cap, hd)), np.zeros(cap)

    def step(self, q, k, v):
        """New rows appended and attended over; y on the device."""
        g4, n = self.g4, len(k)
        qb, kb, vb = (g4.Buffer.from_array(a) for a in (q, k, v))
        y = g4.Buffer(q.nbytes)
        at, end = self.len, self.len + n
        if self.quantised:
            self.cache.append(kb, vb, n, at)
            self.cache.attention(qb, n, HEADS, end, at, False, 0, y, self.w, self.w)
            self.kh[at:end], self.vh[at:end] = (ref.unpack(*ref.pack(a)) for a in (k, v))
        else:
            for dst, src in ((self.k, kb), (self.v, vb)):
                g4.check(g4.lib().g4_copy(dst.ptr, at * self.hd * 4, src.ptr, 0, n * self.hd * 4))
            g4.attention(qb, self.k, self.v, n, HEADS, self.hd, end, at, False, 0, y)
            g4.attention_weights(qb, self.k, n, HEADS, self.hd, end, at, False, 0, self.w, self.w)
            self.kh[at:end], self.vh[at:end] = k, v
        self.len = end
        p = ref.weights(q, self.kh, end, at)
        want = p @ self.vh[:end]
        self.wh[:end] += p.sum((0, 1))
        assert np.abs(y.download(np.float32).reshape(q.shape) - want).max() <= TOL * np.abs(self.vh).max()

    def trim(self, keep, first, recent):
        """The picks are those of the device's own weights, which are near the host's."""
        n = self.len
        w = self.w.download(np.float32)
        assert (np.abs(w[:n] - self.wh[:n]) <= 2 * TOL * self.wh[:n]).all() and (w[n:] == 0).all()
        self.g4.cache_evict(self.w, 1, n, keep, first, recent, self.rows, self.w)
        self.planes.rows(self.rows, keep, 0, n)
        rows, kept = ref.evict(w[:n], keep, first, recent)
        np.testing.assert_array_equal(self.rows.download(np.int32, keep), rows)
        np.testing.assert_array_equal(self.w.download(np.float32, n), kept)
        for a in (self.kh, self.vh):
            a[:keep] = a[rows]
        self.wh[:keep], self.wh[keep:] = self.wh[rows], 0
        self.len = keep


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("quantised", [True, False])
def test_a_chat_whose_cache_is_trimmed(g4, hd, quantised):
    rng = np.random.default_rng([hd, quantised])
    chat = Chat(g4, hd, 260, quantised)
    at = 1.5 / hd ** 0.25

    def rows(n):
        return ((rng.standard_normal((n, HEADS, hd)) * at).astype(np.float32),
                (rng.standard_normal((n, hd)) * at).astype(np.float32), rng.standard_normal((n, hd)).astype(np.float32))

    chat.step(*rows(200))  # a prompt
    for turn in range(3):
        for _ in range(5):
            chat.step(*rows(1))
        chat.step(*rows(11))
        chat.trim(150 + turn, 4, 20)
    chat.step(*rows(1))


def test_recorded_with_new_inputs(g4):
    rng = np.random.default_rng(5)
    hd, n, keep = 256, 700, 300
    c = g4.Kv4Cache(n, hd)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    q, k, v, kf = (g4.Buffer(4 * m) for m in (3 * HEADS * hd, 3 * hd, 3 * hd, n * hd))
    y, w, w2, rows, kept, back = (g4.Buffer(4 * m) for m in (3 * HEADS * hd, n, n, 2 * keep, 2 * n, 3 * hd))
    both = g4.Buffer(2 * n * 4)

    def step():
        c.append(k, v, 3, n - 3)
        c.read(n - 3, 3, back, None)
        c.attention(q, 3, HEADS, n, n - 3, False, 0, y, w)
        g4.attention_weights(q, kf, 3, HEADS, hd, n, n - 3, True, 512, w2)
        for i, x in enumerate((w, w2)):
            g4.check(g4.lib().g4_copy(both.ptr, i * n * 4, x.ptr, 0, n * 4))
        g4.cache_evict(both, 2, n, keep, 4, 32, rows, kept)

    def fill():
        x = f(n, hd)
        kf.upload(x)
        c.append(kf, g4.Buffer.from_array(f(n, hd)), n, 0)
        for b, s in ((q, (3, HEADS, hd)), (k, (3, hd)), (v, (3, hd))):
            b.upload(0.2 * f(*s))

    outs = (y, w, w2, rows, kept, back)
    fill()
    step()
    with g4.Encoder() as enc:
        step()
    for turn in range(4):
        fill()
        step()
        want = [b.download(np.uint32) for b in outs]
        for b in outs:
            b.upload(np.zeros(b.nbytes // 4, np.float32))
        # other calls between the replays, of larger and smaller sizes
        other = g4.Kv4Cache(5000, 512)
        x = g4.Buffer.from_array(f(40, HEADS, 512))
        other.attention(x, 40, HEADS, 100 + 1200 * turn, 50, False, 0, g4.Buffer(x.nbytes), g4.Buffer(20000))
        enc.cmdbuf.submit()
        for b, a in zip(outs, want):
            np.testing.assert_array_equal(b.download(np.uint32), a)


def test_two_recordings_and_eager_calls_share_scratch(g4):
    rng = np.random.default_rng(6)
    calls = []
    for hd, n, qrows in ((256, 900, 2), (512, 3000, 1), (64, 400, 50)):
        c = g4.Kv4Cache(n, hd)
        x = [g4.Buffer.from_array(rng.standard_normal((n, hd)).astype(np.float32)) for _ in range(2)]
        c.append(x[0], x[1], n, 0)
        q = g4.Buffer.from_array((0.2 * rng.standard_normal((qrows, HEADS, hd))).astype(np.float32))
        y, w, w2 = g4.Buffer(q.nbytes), g4.Buffer(4 * n), g4.Buffer(4 * n)

        def call(c=c, q=q, qrows=qrows, n=n, y=y, w=w, w2=w2, x=x, hd=hd):
            c.attention(q, qrows, HEADS, n, n - qrows, False, 0, y, w)
            g4.attention_weights(q, x[0], qrows, HEADS, hd, n, n - qrows, False, 0, w2)

        call()
        calls.append((call, (y, w, w2), [b.download(np.uint32) for b in (y, w, w2)]))
    recs = []
    for call, _, _ in calls[:2]:
        with g4.Encoder() as enc:
            call()
        recs.append(enc.cmdbuf)
    big = g4.Kv4Cache(20000, 512)
    bq, by = (g4.Buffer(100 * HEADS * 512 * 4) for _ in range(2))
    for _ in range(3):
        for (_, bufs, _), rec in zip(calls, recs):
            for b in bufs:
                b.upload(np.zeros(b.nbytes // 4, np.float32))
            rec.submit()
            big.attention(bq, 100, HEADS, 20000, 19900, False, 0, by, g4.Buffer(80000))
        calls[2][0]()
        for _, bufs, want in calls:
            for b, a in zip(bufs, want):
                np.testing.assert_array_equal(b.download(np.uint32), a)


def test_calls_are_repeatable(g4):
    rng = np.random.default_rng(8)
    for hd, n, qrows in ((512, 9000, 1), (256, 1500, 60)):
        c = g4.Kv4Cache(n, hd)
        x = g4.Buffer.from_array(rng.standard_normal((n, hd)).astype(np.float32))
        c.append(x, x, n, 0)
        q = g4.Buffer.from_array((0.2 * rng.standard_normal((qrows, HEADS, hd))).astype(np.float32))
        seen = []
        for _ in range(5):
            y, w, w2 = g4.Buffer(q.nbytes), g4.Buffer(4 * n), g4.Buffer(4 * n)
            c.attention(q, qrows, HEADS, n, n - qrows, False, 0, y, w)
            g4.attention_weights(q, x, qrows, HEADS, hd, n, n - qrows, False, 0, w2)
            seen.append([b.download(np.uint32) for b in (y, w, w2)])
        for s in seen[1:]:
            for a, b in zip(s, seen[0]):
                np.testing.assert_array_equal(a, b)


def test_a_recording_without_an_earlier_call_is_refused():
    # in a process of its own, where nothing has made scratch
    code = """
import sys
sys.path.insert(0, %r)
import numpy as np
import g4hip as g4
g4.init(0)
c = g4.Kv4Cache(9000, 256)
q, y, w, k = g4.Buffer(40 * 8 * 256 * 4), g4.Buffer(40 * 8 * 256 * 4), g4.Buffer(300000 * 4), g4.Buffer(9000 * 256 * 4)
rows = g4.Buffer(300000 * 4)
calls = [lambda: c.attention(q, 40, 8, 9000, 8960, False, 0, y, w),
         lambda: g4.attention_weights(q, k, 40, 8, 256, 9000, 8960, False, 0, w)]
free = [lambda: c.append(k, k, 5, 7), lambda: c.read(3, 4, y, q), lambda: g4.cache_evict(w, 3, 1000, 900, 4, 8, rows, w)]
for call in calls:
    with g4.Encoder() as enc:
        try:
            call()
            raise SystemExit("recorded")
        except g4.G4Error as e:
            assert e.code == g4.G4_E_STATE, e
with g4.Encoder() as enc:
    for call in free:
        call()
enc.cmdbuf.submit()
for call in calls:
    call()
with g4.Encoder() as enc:
    for call in calls + free:
        call()
enc.cmdbuf.submit()
g4.sync()
""" % os.path.join(ROOT, "gemma4-js_amd")
    p = subprocess.run([sys.executable, "-c", code], stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                       text=True, timeout=100)
    assert p.returncode == 0, p.stdout[-2000:]


@pytest.mark.skipif(shutil.which("node") is None, reason="no node")
def test_node_surface(g4, tmp_path):
    rng = np.random.default_rng(60)
    m = dict(len=300, hd=128, rows=3, heads=HEADS, keep=200)
    at = 1.5 / 128 ** 0.25
    q = (rng.standard_normal((3, HEADS, 128)) * at).astype(np.float32)
    k = (rng.standard_normal((300, 128)) * at).astype(np.float32)
    v = rng.standard_normal((300, 128)).astype(np.float32)
    for name, a in (("q", q), ("k", k), ("v", v)):
        a.tofile(tmp_path / (name + ".bin"))
    (tmp_path / "meta.json").write_text(json.dumps(m))
    p = subprocess.run(["node", os.path.join(ROOT, "tests", "js", "long_cache.js"), str(tmp_path)],
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert p.returncode == 0, p.stdout
    read = lambda n, t: np.fromfile(tmp_path / (n + ".out"), t)  # noqa: E731
    kk, vv = ref.unpack(*ref.pack(k)), ref.unpack(*ref.pack(v))
    p4 = ref.weights(q, kk, 300, 297)
    assert np.abs(read("y", np.float32).reshape(q.shape) - p4 @ vv).max() <= TOL * np.abs(v).max()
    want = p4.sum((0, 1)) + ref.weights(q, k, 300, 297).sum((0, 1))
    w = read("weights", np.float32)
    assert (np.abs(w - want) <= 2 * TOL * want).all()
    rows, kept = ref.evict(w, 200, 2, 10)
    np.testing.assert_array_equal(read("rows", np.int32), rows)
    np.testing.assert_array_equal(read("kept", np.float32), kept)
    np.testing.assert_array_equal(read("kback", np.float32).reshape(200, 128), kk[rows])
    np.testing.assert_array_equal(read("vback", np.float32).reshape(200, 128), vv[rows])
    assert "g4_cache_evict" in json.loads((tmp_path / "out.json").read_text())["refused"]

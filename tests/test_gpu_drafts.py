"""The drafted-token operators together: one check step of a draft tree, eager, recorded and
through Node, and the same state reached token by token."""
import json
import os
import shutil
import subprocess
import sys

import numpy as np
import pytest

import draft_reference as ref
import synthetic as syn

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

HEADS, VOCAB, HIDDEN = 4, 3001, 256


class Step:
    """Two layers' caches (head dims 64 and 256, one windowed) and a tree of drafted tokens.
    The hidden state of a node is what its attention leaves, cut to HIDDEN values."""

    def __init__(self, g4, seed=5, nodes=13, prefix=150):
        rng = np.random.default_rng(seed)
        self.g4, self.rng, self.nodes, self.prefix = g4, rng, nodes, prefix
        self.cap = prefix + nodes + 7
        self.dims = [(64, 32), (256, 0)]  # head dim, window
        self.k = [rng.standard_normal((self.cap, hd)).astype(np.float32) / hd ** 0.25 for hd, _ in self.dims]
        self.v = [rng.standard_normal((self.cap, hd)).astype(np.float32) for hd, _ in self.dims]
        self.q = [(2 * rng.standard_normal((nodes, HEADS, hd)) / hd ** 0.25).astype(np.float32)
                  for hd, _ in self.dims]
        self.E = syn.bf16_rne(rng.standard_normal((VOCAB, HIDDEN)).astype(np.float32))
        self.parents = np.array([rng.integers(max(-1, i - 4), i) if i else -1 for i in range(nodes)], np.int32)
        self.u = rng.random(nodes).astype(np.float32)
        b = g4.Buffer.from_array
        self.kb, self.vb, self.qb = ([b(a) for a in arrays] for arrays in (self.k, self.v, self.q))
        self.Eb, self.pb, self.ub = b(self.E), b(self.parents), b(self.u)
        self.yb = [g4.Buffer(a.nbytes) for a in self.q]
        self.logits = g4.Buffer(nodes * VOCAB * 4)
        self.tokens, self.probs = g4.Buffer(nodes * 4), g4.Buffer(nodes * 4)
        self.path = b(np.zeros(nodes, np.int32))
        planes = [p for kv in zip(self.kb, self.vb) for p in kv]
        self.planes = g4.CachePlanes(planes, planes, [hd for hd, _ in self.dims for _ in range(2)])

    def check(self):
        """Attention of both layers, the head on the second one's output, the picks."""
        g4 = self.g4
        for i, (hd, window) in enumerate(self.dims):
            g4.attention_tree(self.qb[i], self.kb[i], self.vb[i], self.nodes, HEADS, hd, self.prefix,
                              self.pb, window > 0, window, self.yb[i])
        # rows of HEADS * 256 values: the head takes the first 256 of each, one call per row
        # would, so the states are the first heads
        g4.bf16_head_rows(self.yb[1], self.nodes * HEADS, self.Eb, VOCAB, HIDDEN, self.wide, VOCAB,
                          1.0, 30.0)
        g4.sample(self.wide, self.nodes, VOCAB, self.ub, self.tokens, self.probs,
                  stride=HEADS * VOCAB, temperature=0.8, top_k=200, top_p=0.95)

    @property
    def wide(self):
        if not hasattr(self, "_wide"):
            self._wide = self.g4.Buffer(self.nodes * HEADS * VOCAB * 4)
        return self._wide

    def keep(self, n):
        self.planes.rows(self.path, n, self.prefix, self.prefix + self.nodes)

    def results(self):
        y = [b.download(np.float32) for b in self.yb]
        return y + [self.tokens.download(np.int32), self.probs.download(np.float32)]


def walk(parents, drafted, picked):
    """Indices of the accepted nodes: from the first node on, a child that holds the token
    picked at its parent (the lowest index of several)."""
    path = [0]
    while True:
        nxt = [j for j, p in enumerate(parents) if p == path[-1] and drafted[j] == picked[path[-1]]]
        if not nxt:
            return path
        path.append(nxt[0])


def test_a_check_step_equals_its_definition(g4):
    s = Step(g4)
    s.check()
    y0, y1, tokens, probs = s.results()
    n = s.prefix + s.nodes
    for y, i in ((y0, 0), (y1, 1)):
        want = ref.attention_tree(s.q[i], s.k[i][:n], s.v[i][:n], s.prefix, s.parents.tolist(), s.dims[i][1])
        assert np.abs(y.reshape(want.shape) - want).max() <= 2e-5 * np.abs(s.v[i]).max()
    logits = s.wide.download(np.float32).reshape(s.nodes, HEADS, VOCAB)[:, 0]
    x = y1.reshape(s.nodes, HEADS, 256)[:, 0].astype(np.float64)
    e = syn.bf16_to_f32(s.E).astype(np.float64)
    want = 30 * np.tanh(x @ e.T / 30)
    assert np.abs(logits - want).max() <= 2.0 ** -24 * 24 * (np.abs(x) @ np.abs(e).T).max() + 2e-5
    for r in range(s.nodes):
        t, p = ref.sample(logits[r], s.u[r], temperature=0.8, top_k=200, top_p=0.95)
        assert tokens[r] == t and abs(probs[r] - p) <= 1e-6 * p


def test_accepted_rows_continue_as_a_chain(g4):
    """After the accepted rows were kept, attention over the cache is what a chain of the same
    tokens gives (to rounding: the keys are summed in another order)."""
    s = Step(g4, seed=8)
    s.check()
    tokens = s.results()[2]
    # a draft that some path of the tree agrees with
    drafted = np.full(s.nodes, -1)
    at = 0
    while True:
        children = [j for j in range(s.nodes) if s.parents[j] == at]
        if not children:
            break
        drafted[children[-1]] = tokens[at]
        at = children[-1]
    path = walk(s.parents.tolist(), drafted, tokens)
    assert len(path) > 2 and path == ref.path_of(s.parents.tolist(), path[-1])
    before = [b.download(np.float32).reshape(s.cap, -1) for kv in zip(s.kb, s.vb) for b in kv]
    s.path.upload((np.array(path) + s.prefix).astype(np.int32))
    s.keep(len(path))
    n = s.prefix + len(path)
    for old, buf in zip(before, [b for kv in zip(s.kb, s.vb) for b in kv]):
        want = old.copy()
        want[s.prefix:n] = old[s.prefix + np.array(path)]
        np.testing.assert_array_equal(buf.download(np.float32).reshape(old.shape), want)
    for i, (hd, window) in enumerate(s.dims):
        q = np.ascontiguousarray(s.q[i][path])
        y = g4.Buffer(q.nbytes)
        g4.attention(g4.Buffer.from_array(q), s.kb[i], s.vb[i], len(path), HEADS, hd, n, s.prefix,
                     window > 0, window, y)
        tree = s.yb[i].download(np.float32).reshape(s.q[i].shape)[path]
        assert np.abs(y.download(np.float32).reshape(q.shape) - tree).max() <= 4e-5 * np.abs(s.v[i]).max()


def test_a_recorded_step_replays_with_new_inputs(g4):
    s = Step(g4, seed=21)
    s.check()  # the sizes' scratch
    s.keep(4)
    with g4.Encoder() as enc:
        s.check()
        s.keep(4)
    rng = np.random.default_rng(1)
    kv = [b for pair in zip(s.kb, s.vb) for b in pair]
    for turn in range(4):
        s.parents = np.array([rng.integers(-1, i) if i else -1 for i in range(s.nodes)], np.int32)
        for b, a in ((s.pb, s.parents), (s.ub, rng.random(s.nodes).astype(np.float32)),
                     (s.path, (s.prefix + np.sort(rng.choice(s.nodes, s.nodes, False))).astype(np.int32)),
                     (s.qb[turn % 2], rng.standard_normal(s.q[turn % 2].shape).astype(np.float32))):
            b.upload(a)
        start = [b.download(np.float32) for b in kv]
        s.check()
        s.keep(4)
        eager = s.results() + [b.download(np.float32) for b in kv]
        for b, a in zip(kv, start):
            b.upload(a)
        # other work of the same operators between the replays
        other = Step(g4, seed=30 + turn, nodes=3 + 5 * turn, prefix=400)
        other.check()
        other.keep(2)
        for b in s.yb + [s.tokens, s.probs, s.wide]:
            b.upload(np.zeros(b.nbytes // 4, np.float32))
        enc.cmdbuf.submit()
        for got, want in zip(s.results() + [b.download(np.float32) for b in kv], eager):
            np.testing.assert_array_equal(got, want)


def test_two_recordings_and_eager_calls_share_scratch(g4):
    a, b = Step(g4, seed=40, nodes=20, prefix=900), Step(g4, seed=41, nodes=7, prefix=60)
    for s in (a, b):
        s.check()
    want = [s.results() for s in (a, b)]
    recs = []
    for s in (a, b):
        with g4.Encoder() as enc:
            s.check()
        recs.append(enc.cmdbuf)
    big = Step(g4, seed=42, nodes=64, prefix=3000)  # the scratch grows past the recordings'
    big.check()
    for _ in range(3):
        for s, rec in zip((a, b), recs):
            for buf in s.yb + [s.tokens, s.probs]:
                buf.upload(np.zeros(buf.nbytes // 4, np.float32))
            rec.submit()
            big.check()
        for s, w in zip((a, b), want):
            for got, x in zip(s.results(), w):
                np.testing.assert_array_equal(got, x)


def test_a_recording_without_an_earlier_call_is_refused():
    # in a process of its own, where nothing has made scratch
    code = """
import sys
sys.path.insert(0, %r)
import numpy as np
import g4hip as g4
g4.init(0)
nodes, hd, prefix, vocab, k = 8, 256, 4000, 70000, 64
q, y, kv = g4.Buffer(nodes * 8 * hd * 4), g4.Buffer(nodes * 8 * hd * 4), g4.Buffer((prefix + nodes) * hd * 4)
parents = g4.Buffer.from_array(np.arange(-1, nodes - 1, dtype=np.int32))
x, E, z = g4.Buffer(nodes * k * 4), g4.Buffer(vocab * k * 2), g4.Buffer(nodes * vocab * 4)
u, tok, pr = g4.Buffer(4 * nodes), g4.Buffer(4 * nodes), g4.Buffer(4 * nodes)
path = g4.Buffer.from_array(np.arange(100, 200, dtype=np.int32))
calls = [lambda: g4.attention_tree(q, kv, kv, nodes, 8, hd, prefix, parents, False, 0, y),
         lambda: g4.bf16_head_rows(x, nodes, E, vocab, k, z, vocab, 1.0, 30.0),
         lambda: g4.sample(z, nodes, vocab, u, tok, pr, vocab, top_k=4),
         lambda: g4.CachePlanes([kv], [kv], [hd]).rows(path, 100, 90, prefix)]
for call in calls:
    with g4.Encoder() as enc:
        try:
            call()
            raise SystemExit("recorded")
        except g4.G4Error as e:
            assert e.code == g4.G4_E_STATE, e
for call in calls:
    call()
with g4.Encoder() as enc:
    for call in calls:
        call()
enc.cmdbuf.submit()
g4.sync()
""" % os.path.join(ROOT, "gemma4-js_amd")
    p = subprocess.run([sys.executable, "-c", code], stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                       text=True, timeout=100)
    assert p.returncode == 0, p.stdout[-2000:]


def test_calls_are_repeatable(g4):
    s = Step(g4, seed=50, nodes=33, prefix=2000)
    s.check()
    want = s.results()
    for _ in range(5):
        s.check()
        for got, x in zip(s.results(), want):
            np.testing.assert_array_equal(got, x)


@pytest.mark.skipif(shutil.which("node") is None, reason="no node")
def test_node_surface(g4, tmp_path):
    s = Step(g4, seed=60)
    s.check()
    y0, _, tokens, probs = s.results()
    for name, a in (("q", s.q[0]), ("k", s.k[0]), ("v", s.v[0]), ("parents", s.parents), ("u", s.u),
                    ("E", s.E), ("x", s.yb[1].download(np.float32)),
                    ("rows", np.array([3, 1, 170, 5], np.int32))):
        a.tofile(tmp_path / (name + ".bin"))
    meta = dict(nodes=s.nodes, heads=HEADS, hd=64, prefix=s.prefix, window=32, cap=s.cap, vocab=VOCAB,
                hidden=HIDDEN)
    (tmp_path / "meta.json").write_text(json.dumps(meta))
    p = subprocess.run(["node", os.path.join(ROOT, "tests", "js", "drafts.js"), str(tmp_path)],
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert p.returncode == 0, p.stdout
    out = json.loads((tmp_path / "out.json").read_text())
    read = lambda n, t: np.fromfile(tmp_path / n, t)  # noqa: E731
    np.testing.assert_array_equal(read("y.out", np.float32), y0)
    np.testing.assert_array_equal(read("tokens.out", np.int32), tokens)
    np.testing.assert_array_equal(read("probs.out", np.float32), probs)
    want = s.k[0].copy()
    want[10:14] = np.where((np.array([3, 1, 170, 5]) < s.cap)[:, None], s.k[0][[3, 1, 0, 5]], np.nan)
    if s.cap > 170:
        want[12] = s.k[0][170]
    np.testing.assert_array_equal(read("k.out", np.float32).reshape(want.shape), want)
    assert "top_p" in out["refused"]

"""What the operators of long caches hold in scratch while a cache grows.  Scratch only grows, so each
case runs in a process of its own."""
import pytest

from test_gpu_scratch import fresh

pytestmark = pytest.mark.gpu

HEAD = """
hip = ctypes.CDLL("libamdhip64.so")
def free():
    g4.sync()
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    assert hip.hipMemGetInfo(ctypes.byref(a), ctypes.byref(b)) == 0
    return a.value
def attend(c, q, y, w, rows, hd, keys, window=0):
    c.attention(q, rows, 8, keys, keys - rows, window > 0, window, y, w, w)
def weigh(k, q, w, rows, hd, keys, window=0):
    g4.attention_weights(q, k, rows, 8, hd, keys, keys - rows, window > 0, window, w, w)
"""


@pytest.mark.parametrize("op", ["attend", "weigh"])
def test_one_token_holds_its_own_rows(op):
    # 8 rows of 131072 scores, 4.2 MB, and for the attention 512 splits of 8 rows of 512, 8.4 MB
    out = fresh(HEAD + """
op, keys, hd = %r, 131072, 512
c, k = g4.Kv4Cache(keys, hd), g4.Buffer(keys * hd * 4)
q, y, w = g4.Buffer(8 * hd * 4), g4.Buffer(8 * hd * 4), g4.Buffer(keys * 4)
call = (lambda n: attend(c, q, y, w, 1, hd, n)) if op == "attend" else (lambda n: weigh(k, q, w, 1, hd, n))
call(64)
before = free()
call(keys)
print(before - free())
""" % op)
    assert int(out) < ((16 << 20) if op == "attend" else (8 << 20)), out


@pytest.mark.parametrize("op", ["attend", "weigh"])
@pytest.mark.parametrize("rows", [1, 64])
def test_a_growing_cache_does_not_leave_blocks_behind(op, rows):
    # need grows with every call: it is met by few, larger blocks, not by one of each size
    out = fresh(HEAD + """
op, rows, hd, first, calls, step = %r, %d, 64, 20000, 300, 64
keys = first + calls * step
c, k = g4.Kv4Cache(keys, hd), g4.Buffer(keys * hd * 4)
q, y, w = g4.Buffer(rows * 8 * hd * 4), g4.Buffer(rows * 8 * hd * 4), g4.Buffer(keys * 4)
call = (lambda n: attend(c, q, y, w, rows, hd, n)) if op == "attend" else (lambda n: weigh(k, q, w, rows, hd, n))
call(64)
before = free()
for i in range(calls):
    call(first + i * step)
print(before - free())
""" % (op, rows))
    # the scores of the last call, or of a chunk of the calls with more (and, of 32 rows each, their
    # sums): blocks of 1.5 times the size of the one before add up to less than 4.5 times that, and
    # HIP hands out 2 MB at a time
    scores = min(rows * 8 * 39200 * 4, 256 << 20)
    assert int(out) < 5 * scores + (32 << 20), (int(out) / scores, out)


def test_recorded_at_a_size_that_a_larger_call_left():
    # scratch is larger than the call needs by then: recordings of smaller calls, and of that one
    fresh(HEAD + """
hd, keys = 64, 30000
rng = np.random.default_rng(1)
x = g4.Buffer.from_array(rng.standard_normal((keys, hd)).astype(np.float32))
c = g4.Kv4Cache(keys, hd)
c.append(x, x, keys, 0)
q = g4.Buffer.from_array(rng.standard_normal((8, hd)).astype(np.float32))
y, w, w2 = g4.Buffer(8 * hd * 4), g4.Buffer(keys * 4), g4.Buffer(keys * 4)
def call(n):
    c.attention(q, 1, 8, n, n - 1, False, 0, y, w)
    g4.attention_weights(q, x, 1, 8, hd, n, n - 1, False, 0, w2)
for n in range(29000, 30001, 100):
    call(n)
recs = []
for n in (400, 29950, 30000):
    call(n)
    want = [b.download(np.uint32) for b in (y, w, w2)]
    with g4.Encoder() as enc:
        call(n)
    recs.append((n, want, enc.cmdbuf))
for turn in range(3):
    for n, want, rec in recs:
        rec.submit()
        for b, a in zip((y, w, w2), want):
            got = b.download(np.uint32)
            assert np.array_equal(got[:n] if b is not y else got, a[:n] if b is not y else a), (turn, n)
        call(29000 + 17 * turn)
""")

"""Sizes at which a drafted-token operator once took many times what its neighbours take.  Both
times are measured here, in turn, so a bound is a ratio, with room for a busy machine."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def us(g4, *calls):
    """Microseconds per call: of each the least of a few runs, taken in turn."""
    best = [float("inf")] * len(calls)
    for call in calls:
        call()
    for _ in range(7):
        for i, call in enumerate(calls):
            start, stop = g4.Event(), g4.Event()
            start.record()
            for _ in range(10):
                call()
            stop.record()
            g4.sync()
            best[i] = min(best[i], start.elapsed_ms(stop) * 100)
    print("us per call:", *("%.1f" % b for b in best), flush=True)
    return best


@pytest.mark.parametrize("n,rows", [(512, 8192), (2048, 4096)])
def test_head_of_many_groups_of_states(g4, n, rows):
    # 8 and 32 groups of 64 states, which together fill the GPU: at most half the time of a call
    # for each (with a block for every 16 rows and group 7.1 and 24 calls' time, now 1.8 and 4.3)
    k = 1536
    x, E, out = g4.Buffer(n * k * 4), g4.Buffer(rows * k * 2), g4.Buffer(n * rows * 4)
    g4.fill_random(E, rows * k, g4.RAND_BF16_NORMAL, 5, 0.03)
    x.upload(np.random.default_rng(n).standard_normal((n, k)).astype(np.float32))
    one, all_ = us(g4, lambda: g4.bf16_head_rows(x, 64, E, rows, k, out),
                   lambda: g4.bf16_head_rows(x, n, E, rows, k, out))
    assert all_ < n // 64 / 2 * one


@pytest.mark.parametrize("rows", [1, 64])
@pytest.mark.parametrize("cuts", [dict(top_p=0.75), dict(top_k=131072), dict(top_k=131072, top_p=0.9)])
def test_sampling_of_flat_rows(g4, rows, cuts):
    # at temperature 1.5 the cuts of rows of unit spread lie among some 20000 tokens each, more
    # than are listed: the row's block reads it again for every step of the search
    vocab = 262144
    rng = np.random.default_rng(rows)
    flat, peaked = (g4.Buffer.from_array((rng.standard_normal((rows, vocab)) * sigma).astype(np.float32))
                    for sigma in (1.0, 4.0))
    u = g4.Buffer.from_array(rng.random(rows).astype(np.float32))
    tok, pr = g4.Buffer(rows * 4), g4.Buffer(rows * 4)
    one, many = us(g4, lambda: g4.sample(peaked, rows, vocab, u, tok, pr, temperature=1.5, top_p=0.75),
                   lambda: g4.sample(flat, rows, vocab, u, tok, pr, temperature=1.5, **cuts))
    assert many < 14 * one

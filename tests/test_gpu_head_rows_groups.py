"""g4_bf16_head_rows for more than 64 states over tables of few rows, on both sides of the border
between the kernel that splits K and the one that keeps the states in groups."""
import numpy as np
import pytest

from test_gpu_head_rows import case, check, run

pytestmark = pytest.mark.gpu


# 16-row blocks times 64-state groups: up to 768 (at 256 CUs) for the first kernel
@pytest.mark.parametrize("n,rows,k", [
    (128, 6144, 256), (128, 6145, 256), (193, 3060, 1528), (193, 3088, 1528), (700, 1300, 264),
    (513, 1000, 1536), (3000, 257, 72), (3000, 255, 72), (12300, 64, 8), (12288, 64, 8), (16000, 3, 40)])
def test_groups_over_few_rows(g4, n, rows, k):
    print("head rows", n, rows, k, flush=True)
    x, E = case(np.random.default_rng([n, rows, k]), n, rows, k)
    check(run(g4, x, E), x, E)

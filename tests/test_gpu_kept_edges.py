"""cc_attend_weigh where its scores are all alike, larger than f32 tells apart, or no numbers, and its form for many columns
(query rows times heads of a kv head: more than 64) on what test_gpu_kept.py asks of few: against the same plain
implementation in 64 bits."""
import numpy as np
import pytest

from test_gpu_kept import Kept, check_weigh, ctx, filled  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------- scores that are alike ---

@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("past", [0, 100])
@pytest.mark.parametrize("size", [0.0, 1e-38, 1e-30])
@pytest.mark.parametrize("n", [1, 20, 40])
def test_weigh_queries_of_nothing_over_keys_of_nothing(ctx, D, past, size, n):
    """Zero or tiny queries over zero keys (a warm-up's, padded rows'): every row gets as much as the others, and the rows
    behind a query get nothing."""
    rng = np.random.default_rng(D + past)
    T = past + n
    c = Kept(rng, 1, D, D, T // 64 + 1, 1, T // 64 + 1)
    c.append_at([(0, 0, T)], np.zeros((T, D), np.float32), rng.standard_normal((T, D)).astype(np.float32))
    c.weight[:] = 0.5
    q = (size * rng.standard_normal((n, 2 * D))).astype(np.float32)
    check_weigh(ctx, c, [(0, past, n)], 2, q=q, fade=0.5)


@pytest.mark.parametrize("n", [20, 40])
def test_weigh_a_padded_batchs_last_page(ctx, n):
    """Rows of zeros behind a prompt's own fill its last page: q, k and v."""
    rng = np.random.default_rng(7)
    c = filled(rng, 2, 128, 128, [64])
    c.table = np.concatenate([c.table, np.array([[(c.table[0, 0] + 1) % len(c.k)]], np.int32)], 1)
    c.append_at([(0, 64, n)], *np.zeros((2, n, 256), np.float32))
    q = rng.standard_normal((n + 20, 4 * 128)).astype(np.float32)
    q[20:] = 0
    check_weigh(ctx, c, [(0, 44, n + 20)], 4, q=q)


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("n", [1, 40])
def test_weigh_large_queries_across_large_keys(ctx, D, n):
    """Queries and keys whose products would pass f32's range, in channels that do not meet: scores of zero."""
    rng = np.random.default_rng(D)
    c = filled(rng, 1, D, 2, [70 + n])
    k, v = np.zeros((70 + n, D), np.float32), rng.standard_normal((70 + n, D)).astype(np.float32)
    k[:, 7] = 1e7
    c.append_at([(0, 0, 70 + n)], k, v)
    q = np.zeros((n, 2 * D), np.float32)
    q[:, [5, D + 5]] = 1e38
    check_weigh(ctx, c, [(0, 70, n)], 2, q=q)

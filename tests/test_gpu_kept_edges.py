"""cc_attend_weigh where its scores are all alike, larger than f32 tells apart, or no numbers, and its form for many columns
(query rows times heads of a kv head: more than 64) on what test_gpu_kept.py asks of few: against the same plain
implementation in 64 bits."""
import numpy as np
import pytest

import test_gpu_kept as base
from test_gpu_kept import Kept, check_weigh, ctx, dev, filled, same_bits, scale_index  # noqa: F401
from test_gpu_operators import code_index, quantise

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


# ------------------------------------------------- scores that f32 rounds to whole numbers ---

def one_hot_values(c, pages, T):
    """v of row t: 1 in channel t % D. So an output's channel is the probability of the rows t % D."""
    v = np.zeros((T, c.nkv, c.D), np.float32)
    v[np.arange(T), :, np.arange(T) % c.D] = 1
    code, scale = quantise(v)
    for t in range(T):
        page = pages[t // 64]
        for h in range(c.nkv):
            c.v[page, h, code_index(1, c.D)[t % 64]] = (code[t, h] + 128).astype(np.uint8)
            c.v.view(np.float32)[page, h, 16 * c.D + scale_index(1, c.D)[t % 64]] = scale[t, h]


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("size", [300.0, 3e3, 2e5, 1e6, 3e7, 1e10, 1e15])
@pytest.mark.parametrize("n", [1, 8, 40, 300])
def test_weigh_adds_up_what_attention_gives(ctx, n, size, mixed):
    """However large the scores: what a row's weight gains is what the outputs took of it, also where rows of small and of
    large scores stand beside each other (`mixed`). An output's p is a sum of pairs, 2^-20 of the largest value (1), so n * 2 of
    them are off by no more than n * 2^-19; a weight's p is formed from the same score, once the fused and once the rounded
    product where the scores of a column pass 2^10 within the call: 2^-14 of it. l's two roundings and the sums of n * 2 terms
    are below another 2^-14."""
    rng = np.random.default_rng(int(np.log10(size)) + n)
    nkv, D, past, heads = 2, 128, 130, 4
    T = past + n
    c = filled(rng, nkv, D, D, [T])
    one_hot_values(c, c.table[0], T)
    q = (size * rng.standard_normal((n, heads * D))).astype(np.float32)
    if mixed:
        q *= np.repeat(2.0 ** rng.integers(-9, 5, (n, heads)), D, 1).astype(np.float32)
    cache, marks = c.device()
    out = ctx.attend_weigh(cache, [(0, past, n)], dev(q), marks=marks, fade=0.0).numpy().reshape(n, nkv, 2, D)
    got = c.m[0].numpy()[c.table[0]].transpose(1, 0, 2).reshape(nkv, -1)[:, :T].astype(np.float64)
    took = out.astype(np.float64).sum((0, 2))
    gained = np.zeros((nkv, D))
    for t in range(T):
        gained[:, t % D] += got[:, t]
    off = np.abs(gained - took)
    assert (off <= gained * 2.0 ** -13 + n * 2.0 ** -19).all(), (off.max(), gained[np.unravel_index(off.argmax(), off.shape)])
    assert (np.abs(got.sum(1) - 2 * n) <= 2 * n * 2.0 ** -13).all(), got.sum(1)
    assert (got <= 2 * n * (1 + 2.0 ** -13)).all()


@pytest.mark.parametrize("size", [1e-30, 1e-4, 300.0, 1e6, 1e12])
def test_weigh_scores_of_any_magnitude_in_many_columns(ctx, size):
    base.test_weigh_scores_of_any_magnitude(ctx, 40, size)


@pytest.mark.parametrize("D,first,n", [(64, 64, 1), (256, 64, 1), (64, 64, 40), (256, 64, 12), (256, 32, 80)])
def test_weigh_a_score_one_step_of_f32_above(ctx, D, first, n):
    """Scores of 1.44 * 2^27, whole multiples of 16 in f32: an odd one in the first rows, the next in those behind, which then
    take all but 2^-16 of the attention or less. (f32 has nothing between the two: the first plus 8 is rounded to the second.)"""
    # q . k / sqrt(D) is 2^27 + 16 c, with codes 64 and c in channels of different groups; the score's 24 bits are those of
    # log2(e) * (1 + c * 2^-23)
    log2e = np.float32(1.4426950408889634)
    bits = [int((log2e * np.float32(1 + c * 2.0 ** -23)).view(np.uint32)) for c in range(12)]
    c0, c1 = next((a, b) for a in range(12) for b in range(12) if bits[a] % 2 and bits[b] == bits[a] + 1)
    rng = np.random.default_rng(D + n)
    past = 128
    c = filled(rng, 1, D, 2, [past + n])
    k = np.zeros((past + n, D), np.float32)
    cache_pages = c.table[0]
    for t in range(past):      # codes as they are, scales of 1
        page, at = cache_pages[t // 64], t % 64
        c.k[page, 0, code_index(0, D)[at]] = 128
        c.k[page, 0, code_index(0, D)[at, 4]] = 128 + 64
        c.k[page, 0, code_index(0, D)[at, 36]] = 128 + (c0 if t < first else c1)
        c.k.view(np.float32)[page, 0, 16 * D + scale_index(0, D)[at]] = 1.0
    for t in range(past, past + n):
        page, at = cache_pages[t // 64], t % 64
        c.k[page, 0, code_index(0, D)[at]] = 128
        c.k.view(np.float32)[page, 0, 16 * D + scale_index(0, D)[at]] = 1.0
    root = {64: 8, 256: 16}[D]
    q = np.zeros((n, D), np.float32)
    q[:, 4] = root * 2.0 ** 21            # times 64 / root: 2^27
    q[:, 36] = root * 2.0 ** 4            # times c / root: c * 2^4, a step of 2^27 in f32 for each c
    cache, marks = c.device()
    out = ctx.attend_weigh(cache, [(0, past, n)], dev(q), marks=marks, fade=0.0).numpy()
    values = np.concatenate([c.exact_rows(1, p, 0) for p in cache_pages])
    want = values[first:past].mean(0)
    # p of the first rows: 2^-16 of the others', 1/3 .. 1 times as many; f16 pairs and f32 sums of 128 rows: 2^-16 more
    lim = np.abs(values[:past]).max() * 2.0 ** -14
    assert np.isfinite(out).all()
    assert (np.abs(out - want) <= lim).all()
    got = c.m[0].numpy()[cache_pages, 0].reshape(-1)
    assert (np.abs(got[first:past] - n / (past - first)) <= n / (past - first) * 2.0 ** -14).all()
    assert (got[:first] <= n * 2.0 ** -14 / first).all() and not got[past:past + n].any()


# ------------------------------------------------------------ what is no number ---

@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("past,n", [(70, 2), (60, 8), (70, 30), (70, 40), (1500, 8), (1500, 40)])
def test_weigh_a_query_that_is_no_number_counts_for_what_it_sees(ctx, D, past, n):
    """A NaN in the first row's query: the weights of the rows that it sees, of its kv head, are NaN, those of the rows behind it
    are the others' sums."""
    rng = np.random.default_rng(D + n)
    c = filled(rng, 2, D, D, [past + n], rope_rows=2000)
    q = rng.standard_normal((n, 4 * D)).astype(np.float32)
    q[0, D + 5] = np.nan                       # head 1, of kv head 0
    cache, marks = c.device()
    out = ctx.attend_weigh(cache, [(0, past, n)], dev(q), marks=marks, fade=0.0).numpy().reshape(n, 4, D)
    q[0, D + 5] = 0
    want, bound, weight, wbound = c.weigh([(0, past, n)], q, 4, fade=0.0)
    bad = np.zeros((n, 4), bool)
    bad[0, 1] = True
    assert np.isnan(out[bad]).all()
    assert (np.abs(out - want.reshape(out.shape))[~bad] <= np.broadcast_to(bound[:, None, None], out.shape)[~bad]).all()
    got, weight, wbound = (a[c.table[0]].transpose(1, 0, 2).reshape(2, -1)[:, :past + n] for a in (c.m[0].numpy(), weight, wbound))
    assert np.isnan(got[0, :past + 1]).all()
    got[0, :past + 1] = weight[0, :past + 1]
    assert (np.abs(got - weight) <= wbound).all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_weigh_a_key_that_is_no_number_among_many_columns(ctx, D):
    """A NaN scale of the last row's key: the row that sees it is NaN, and with it every weight; the others are as without it."""
    rng = np.random.default_rng(D)
    n = 40
    c = filled(rng, 1, D, D, [70 + n])
    at = c.table[0, (69 + n) // 64], 0, 16 * D + scale_index(0, D)[(69 + n) % 64, 1]
    q = rng.standard_normal((n, 2 * D)).astype(np.float32)
    want, bound, weight, wbound = c.weigh([(0, 70, n)], q, 2)
    c.k.view(np.float32)[at] = np.nan
    cache, marks = c.device()
    out = ctx.attend_weigh(cache, [(0, 70, n)], dev(q), marks=marks).numpy()
    assert np.isnan(out[-1]).all()
    assert (np.abs(out - want)[:-1] <= bound[:-1, None]).all()
    assert np.isnan(c.m[0].numpy()[c.table[0], 0].reshape(-1)[:70 + n]).all()


# ------------------------------------- what test_gpu_kept.py asks of up to 64 columns ---

@pytest.mark.parametrize("D", [64, 128, 256])
def test_weigh_what_many_columns_do_not_see(ctx, D):
    base.test_weigh_what_rows_do_not_see(ctx, D, 40)


def test_weigh_a_nan_query_among_many_columns(ctx):
    base.test_weigh_keys_and_queries_that_are_no_numbers(ctx, 40)


@pytest.mark.parametrize("observe", [1000, 7])
def test_weigh_many_columns_past_4_gib(ctx, observe):
    """80 rows of two heads over blocks past 2^31 and 2^32 bytes of the pools, as over a small cache's."""
    from chattorrent_amd.ccdecode import DeviceArray, KVCache, Marks
    rng = np.random.default_rng(18)
    nkv, D, n = 8, 256, 30000
    small = Kept(rng, nkv, D, D, 6, 1, 6)
    small.table[0] = np.arange(6)
    near, near_marks = small.device()
    pools = [DeviceArray((n, nkv, small.k.shape[2]), np.uint8) for _ in range(2)]
    marks = [DeviceArray((n, nkv, 64), t) for t in (np.float32, np.int32)]
    table = np.array([[29999, 3, 14800, 29400, 14650, 29250]], np.int32)
    far = KVCache(*pools, dev(table), small.d[3], D)
    k, v = (dev(rng.standard_normal((380, nkv * D)).astype(np.float32)) for _ in range(2))
    q = dev(rng.standard_normal((80, 2 * nkv * D)).astype(np.float32))
    got = []
    for cache, m in ((near, near_marks), (far, Marks(*marks))):
        ctx.kv_append_at(cache, [(0, 0, 380)], k, v, marks=m)
        got.append(ctx.attend_weigh(cache, [(0, 300, 80)], q, marks=m, observe=observe).numpy())
    assert np.isfinite(got[0]).all() and same_bits(*got)
    assert same_bits(marks[0].numpy()[table[0]].reshape(6, -1)[:5], small.m[0].numpy().reshape(6, -1)[:5])

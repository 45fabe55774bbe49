"""The operators on device buffers (cc_kv_append, cc_kv_bounds, cc_attend_pages,
cc_logits_adjust, cc_sample) against plain implementations in numpy, in 64 bits,
through the C ABI, at the sizes and masks where they can go wrong; their use on
streams, in captured graphs and on a context's own cache; and a run of them
together."""
import ctypes as C
import math
import os
import subprocess
import sys

import numpy as np
import pytest

from chattorrent_amd import configs

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U32 = 2.0 ** -24      # half a step of f32, relative to the value


@pytest.fixture(scope="module")
def ctx(gpu):
    from chattorrent_amd.ccdecode import Context
    c = Context(configs.with_layers(configs.SMOLLM2, 1), n_max=256, t_max=8, slots=2)
    yield c
    c.close()


def dev(a):
    from chattorrent_amd.ccdecode import DeviceArray
    return DeviceArray.of(a)


# ------------------------------------------------------------- plain: cache ---

def code_index(which, D):
    t, d = np.arange(64)[:, None], np.arange(D)[None]
    if which == 0:
        return t * D + (D // 4) * ((d % 32) // 8) + 8 * (d // 32) + d % 8
    u = 16 * ((t % 16) // 4) + 4 * (t // 16) + t % 4
    return ((u // 16) * D + d) * 16 + u % 16


def scale_index(which, D):
    t, g = np.arange(64)[:, None], np.arange(D // 32)[None]
    if which == 0:
        return t * (D // 32) + g
    u = 16 * ((t % 16) // 4) + 4 * (t // 16) + t % 4
    return ((u // 16) * (D // 32) + g) * 16 + u % 16


def bound_index(D):
    w, d = np.arange(2)[:, None], np.arange(D)[None]
    return (2 * w + (d % 32) // 16) * (D // 2) + 16 * (d // 32) + d % 16


def quantise(x):
    """store_kv's steps in f32: whole codes and scales of x [..., D]."""
    g = x.astype(np.float32).reshape(*x.shape[:-1], -1, 32)
    scale = np.abs(g).max(-1) / np.float32(127)
    inv = np.where(scale > 0, np.float32(1) / np.where(scale > 0, scale, 1), 0).astype(np.float32)
    return np.clip(np.rint(g * inv[..., None]), -127, 127).reshape(x.shape), scale


def bounds_of(x):
    """Codes [2, D] and scales [D/32] of the keys x f32 [64, D]."""
    mx, mn = x.max(0), x.min(0)
    B = np.maximum(np.abs(mx), np.abs(mn)).reshape(-1, 32).max(-1) / np.float32(127)
    s = np.repeat(B, 32)
    with np.errstate(divide="ignore", invalid="ignore"):
        hi = np.where(s > 0, np.clip(np.ceil(mx / s), -127, 127), 0)
        lo = np.where(s > 0, np.clip(np.floor(mn / s), -127, 127), 0)
    return np.stack([hi, lo]), B


def rotate32(x, cs):
    """RoPE in f32 steps: x [..., D], cs [..., rot/2, 2]."""
    h = cs.shape[-2]
    a, o, c, s = x[..., :h], x[..., h:2 * h], cs[..., 0], cs[..., 1]
    return np.concatenate([a * c - o * s, o * c + a * s, x[..., 2 * h:]], -1).astype(np.float32)


class Plain:
    """A paged cache on the host, in the documented layout, and its operators in plain steps."""

    def __init__(self, rng, nkv, D, rot, n_pages, slots, max_pages, fill=0x5A):
        self.nkv, self.D, self.rot, self.ng = nkv, D, rot, D // 32
        self.k = np.full((n_pages, nkv, 64 * D + 256 * self.ng), fill, np.uint8)
        self.v = self.k.copy()
        for pool in (self.k, self.v):      # stale scales are NaN
            pool.view(np.float32)[:, :, 16 * D:] = np.nan
        self.bounds = np.full((n_pages, nkv * (2 * D + D // 8)), fill, np.uint8)
        order = rng.permutation(n_pages)
        self.table = np.zeros((slots, max_pages), np.int32)
        n = min(n_pages, slots * max_pages)
        self.table.reshape(-1)[:n] = order[:n]
        inv = 10000.0 ** (-2.0 * np.arange(rot // 2) / rot)
        ang = np.arange(max_pages * 64)[:, None] * inv
        self.rope = np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)

    def device(self, bounds=True):
        from chattorrent_amd.ccdecode import KVCache
        self.d = [dev(a) for a in (self.k, self.v, self.table, self.rope, self.bounds)]
        return KVCache(self.d[0], self.d[1], self.d[2], self.d[3], self.D, bounds=self.d[4] if bounds else None)

    def append(self, jobs, k, v):
        row = 0
        for slot, past, n in jobs:
            for i in range(n):
                p = past + i
                page, t = self.table[slot, p // 64], p % 64
                kr = rotate32(k[row].reshape(self.nkv, self.D), self.rope[p][None])
                for which, pool, x in ((0, self.k, kr), (1, self.v, v[row].reshape(self.nkv, self.D))):
                    code, scale = quantise(x)
                    for h in range(self.nkv):
                        pool[page, h, code_index(which, self.D)[t]] = (code[h] + 128).astype(np.uint8)
                        pool.view(np.float32)[page, h, 16 * self.D + scale_index(which, self.D)[t]] = scale[h]
                row += 1
            for p in range(past // 64, (past + n) // 64):
                self.make_bounds(self.table[slot, p])

    def rows(self, which, page, h):
        """The 64 rows of a block as f32 products of code and scale."""
        pool = (self.k, self.v)[which]
        code = pool[page, h, code_index(which, self.D)].astype(np.float32) - 128
        scale = pool.view(np.float32)[page, h, 16 * self.D + scale_index(which, self.D)]
        return code * np.repeat(scale, 32, -1)

    def make_bounds(self, page):
        D = self.D
        for h in range(self.nkv):
            code, B = bounds_of(self.rows(0, page, h))
            self.bounds[page, h * 2 * D + bound_index(D)] = code.astype(np.int8).view(np.uint8)
            self.bounds.view(np.float32)[page, self.nkv * D // 2 + h * self.ng:][:self.ng] = B

    def scores(self, slot, h, q, pages):
        """Scores of a kv head's rotated queries q f32 [G, D] for pages, rounded to f32."""
        D = self.D
        code, T = quantise(q)
        out = []
        for p in pages:
            page = self.table[slot, p]
            b = self.bounds[page, h * 2 * D + bound_index(D)].view(np.int8).astype(np.float64)
            B = self.bounds.view(np.float32)[page, self.nkv * D // 2 + h * self.ng:][:self.ng].astype(np.float64)
            best = np.maximum(code * b[0], code * b[1]).reshape(len(q), -1, 32).sum(-1)
            out.append(np.float32((best * T.astype(np.float64) * B).sum(-1)).max())
        return np.array(out, np.float32)

    def kept(self, slot, pos, h, q, budget, sink, recent):
        seen = pos // 64 + 1
        if seen <= budget:
            return list(range(seen))
        mid = np.arange(sink, seen - recent)
        best = np.argsort(-self.scores(slot, h, q, mid), kind="stable")[:budget - sink - recent]
        return list(range(sink)) + sorted(mid[best].tolist()) + list(range(seen - recent, seen))

    def attend(self, jobs, q, heads, budget, sink, recent):
        """(output in 64 bits, the size of the sums behind it: the largest |v| read, the largest |q|.|k| behind a score)."""
        G, D = heads // self.nkv, self.D
        out, vmax, smax = np.zeros(q.shape), np.zeros(q.shape[0]), np.zeros(q.shape[0])
        row = 0
        for slot, past, n in jobs:
            for i in range(n):
                pos = past + i
                cs = self.rope[pos].astype(np.float64)
                for h in range(self.nkv):
                    qr = q[row].reshape(heads, D)[h * G:(h + 1) * G]
                    pages = self.kept(slot, pos, h, rotate32(qr, self.rope[pos][None]), budget, sink, recent)
                    x = qr.astype(np.float64)
                    r = self.rot // 2
                    a, o = x[:, :r], x[:, r:2 * r]
                    x = np.concatenate([a * cs[:, 0] - o * cs[:, 1], o * cs[:, 0] + a * cs[:, 1], x[:, 2 * r:]], -1)
                    tok = np.concatenate([np.arange(64) + 64 * p for p in pages])
                    ok = tok <= pos
                    kk, vv = (np.concatenate([self.exact_rows(w, self.table[slot, p], h) for p in pages])[ok]
                              for w in (0, 1))
                    s = x @ kk.T / math.sqrt(D)
                    w = np.exp(s - s.max(-1, keepdims=True))
                    out[row].reshape(heads, D)[h * G:(h + 1) * G] = w @ vv / w.sum(-1, keepdims=True)
                    vmax[row] = max(vmax[row], np.abs(vv).max())
                    smax[row] = max(smax[row], (np.abs(x) @ np.abs(kk).T).max() / math.sqrt(D))
                row += 1
        return out, vmax, smax

    def exact_rows(self, which, page, h):
        pool = (self.k, self.v)[which]
        code = pool[page, h, code_index(which, self.D)].astype(np.float64) - 128
        scale = pool.view(np.float32)[page, h, 16 * self.D + scale_index(which, self.D)].astype(np.float64)
        return code * np.repeat(scale, 32, -1)


def attend_bound(D, vmax, smax):
    """How far a value of the output may be off. A score is a sum of D products whose f16 pair carries the query to 2^-22 of
    its value (2^-24 absolute below 2^-3: the same of a query of order 1), rotated with three f32 roundings, and whose groups
    meet in f32 (D/32 + 2 roundings); scaled, shifted by the maximum (two roundings of a value of up to smax*1.45 + 8) and
    raised by a v_exp within two steps. All are relative to the sum of magnitudes behind the score, smax, so a weight is off
    by e = smax * (2^-22 + (3 + D/32 + 6) * 2^-24) + 8 * 2^-23 relative, weights are averages of values up to vmax, the
    numerator and the sum each carry e, the P.V pair 2^-22 and the joins a dozen more roundings."""
    e = smax * (2.0 ** -22 + (9 + D / 32) * U32) + 8 * 2 * U32
    return 2 * vmax * (e + 2.0 ** -22 + 32 * U32)


def same_bits(a, b):
    return np.array_equal(np.ascontiguousarray(a).view(np.uint8), np.ascontiguousarray(b).view(np.uint8))


# ------------------------------------------------------------------- append ---

@pytest.mark.parametrize("nkv,D,rot,jobs", [
    (3, 64, 64, [(0, 0, 1)]),                                    # a first token
    (1, 128, 128, [(0, 63, 1), (1, 64, 1), (2, 127, 2)]),        # pages completed and begun
    (8, 128, 128, [(2, 0, 64), (0, 5, 130), (1, 191, 1)]),       # whole pages, and ends inside them
    (2, 256, 64, [(1, 60, 9), (0, 0, 200)]),                     # partial rotation, heads of 256
    (5, 64, 6, [(0, 1, 70), (3, 100, 28)]),                      # RoPE halves that are not whole groups of 8 channels
    (3, 128, 2, [(0, 30, 40)]),
])
@pytest.mark.parametrize("pad", [0, 4, 5])
def test_append_bits(ctx, nkv, D, rot, jobs, pad):
    """Codes, scales and key bounds are the plain f32 steps' bits, in a cache of which nothing else changes (stale rows, other
    pages, other pages' bounds); rows at any stride, aligned to 16 bytes or not."""
    rng = np.random.default_rng(len(jobs) * 1000 + D + rot + pad)
    ref = Plain(rng, nkv, D, rot, 24, 4, 5)
    # every earlier row holds something finite
    before = [(s, 0, p) for s, p, _ in jobs if p]
    if before:
        n = sum(b[2] for b in before)
        ref.append(before, rng.standard_normal((n, nkv * D)).astype(np.float32),
                   rng.standard_normal((n, nkv * D)).astype(np.float32))
    cache = ref.device()
    n = sum(j[2] for j in jobs)
    k = rng.standard_normal((n, nkv * D + pad)).astype(np.float32) * 3
    v = rng.standard_normal((n, nkv * D + pad)).astype(np.float32)
    k[n // 2, :32] = 0.0          # a group without any magnitude
    v[n // 2, 32:64] = 1e-42      # subnormal
    dk, dv = Strided(k, nkv * D), Strided(v, nkv * D)
    ctx.kv_append(cache, jobs, dk, dv)
    got = [a.numpy() for a in (ref.d[0], ref.d[1], ref.d[4])]
    ref.append(jobs, k[:, :nkv * D], v[:, :nkv * D])
    for name, a, b in zip(("k", "v", "bounds"), got, (ref.k, ref.v, ref.bounds)):
        assert same_bits(a, b), (name, np.argwhere(a != b)[:5])


class Strided:
    """f32 rows of `width` values, `width + pad` floats apart, on the device (rows after the first start unaligned where pad
    is odd)."""

    def __init__(self, a, width):
        self.whole = dev(a)
        self.shape, self.dtype, self.ld = (a.shape[0], width), a.dtype, a.shape[1]

    def data_ptr(self):
        return self.whole.data_ptr()

    def stride(self, d):
        return self.ld if d in (0, -2) else 1


def test_append_many_jobs_in_one_call(ctx):
    """More jobs than a launch holds; a job with no page of its own in between."""
    rng = np.random.default_rng(3)
    ref = Plain(rng, 1, 64, 32, 300, 300, 1)
    jobs = [(s, int(rng.integers(0, 40)), int(rng.integers(1, 24))) for s in range(300)]
    n = sum(j[2] for j in jobs)
    ref.table[17, 0] = 300        # outside the cache: its rows are not stored
    cache = ref.device()
    k, v = (rng.standard_normal((n, 64)).astype(np.float32) for _ in range(2))
    ctx.kv_append(cache, jobs, dev(k), dev(v))
    got = [a.numpy() for a in (ref.d[0], ref.d[1])]
    at = sum(j[2] for j in jobs[:17])
    keep = np.r_[0:at, at + jobs[17][2]:n]
    ref.append(jobs[:17] + jobs[18:], k[keep], v[keep])
    assert same_bits(got[0], ref.k) and same_bits(got[1], ref.v)


def test_bounds_of_stored_pages_equal_the_appends(ctx):
    """cc_kv_bounds over rows stored before gives the bounds that appending gave; pages that the rows cut are left alone."""
    rng = np.random.default_rng(5)
    ref = Plain(rng, 2, 128, 128, 8, 2, 4)
    ref.append([(0, 0, 250), (1, 0, 70)], *(rng.standard_normal((320, 256)).astype(np.float32) for _ in range(2)))
    want = ref.bounds.copy()
    ref.bounds[:] = 0x11
    cache = ref.device()
    ctx.kv_bounds(cache, [(0, 1, 249), (1, 0, 64)])
    got = ref.d[4].numpy()
    assert same_bits(got[ref.table[1, 0]], want[ref.table[1, 0]])
    for p in (1, 2):
        assert same_bits(got[ref.table[0, p]], want[ref.table[0, p]])
    for p in (0, 3):              # begun before the rows, or not full
        assert (got[ref.table[0, p]] == 0x11).all()


def test_append_stores_what_the_pass_stores(gpu):
    """On a context's own cache, the rows appended through cc_cache_of are cc_op_store_kv's, as cc_read_kv reads them."""
    from chattorrent_amd.ccdecode import Context, KVCache
    d = configs.with_layers(configs.SMOLLM2, 1)
    c = Context(d, n_max=256, t_max=80, slots=2)
    try:
        rng = np.random.default_rng(8)
        w = d["n_kv_heads"] * d["head_dim"]
        k, v = (rng.standard_normal((75, w)).astype(np.float32) for _ in range(2))
        for slot in (0, 1):
            c.fill_random_kv(slot, 100, 1, slot + 1)
        c.op_store_kv(0, 0, 0, k, 20)
        c.op_store_kv(0, 1, 0, v, 20)
        c.kv_append(KVCache.of_context(c, 0), [(1, 20, 75)], dev(k), dev(v))
        for which in (0, 1):
            for h in range(d["n_kv_heads"]):
                assert same_bits(c.read_kv(0, which, 0, h, 20, 95), c.read_kv(0, which, 1, h, 20, 95))
    finally:
        c.close()


# ------------------------------------------------------------------- attend ---

def filled(rng, nkv, D, rot, lengths, spare=0, topics=True):
    pages = [-(-n // 64) for n in lengths]
    ref = Plain(rng, nkv, D, rot, sum(pages) + spare, len(lengths), max(pages))
    at = 0
    order = rng.permutation(len(ref.k))
    for s, n in enumerate(pages):
        ref.table[s] = 0
        ref.table[s, :n] = order[at:at + n]
        at += n
    jobs = [(s, 0, n) for s, n in enumerate(lengths)]
    T = sum(lengths)
    k = rng.standard_normal((T, nkv * D)).astype(np.float32)
    if topics:
        k += np.repeat(rng.standard_normal((-(-T // 50), nkv * D)), 50, 0)[:T].astype(np.float32)
    ref.append(jobs, k, rng.standard_normal((T, nkv * D)).astype(np.float32))
    return ref


@pytest.mark.parametrize("heads,nkv,D,rot,jobs,budget,sink,recent", [
    (9, 3, 64, 64, [(0, 0, 1)], 1, 0, 1),                                # one token, its own
    (5, 1, 128, 128, [(0, 63, 1), (1, 64, 1), (2, 700, 1)], 4, 1, 2),    # page ends; scored and not in one call
    (40, 8, 128, 128, [(0, 1300, 1), (1, 640, 1)], 8, 1, 2),
    (12, 2, 256, 64, [(0, 900, 8), (1, 30, 3)], 6, 1, 2),                # verify rows over a page's end
    (21, 1, 64, 32, [(0, 500, 2)], 3, 0, 1),                             # a group of 21 heads: two tiles
    (48, 1, 128, 128, [(0, 400, 1)], 5, 2, 1),                           # three tiles
    (4, 4, 64, 64, [(0, 1500, 1)], 3, 1, 2),                             # nothing but sink and recent
    (6, 2, 128, 128, [(0, 1000, 1), (0, 1000, 1), (0, 999, 1)], 5, 0, 3),   # a slot more than once
    (8, 2, 128, 6, [(0, 2047, 70)], 40, 1, 2),                           # many rows, no scores needed
    (3, 3, 64, 64, [(0, 5000, 1)], 64, 1, 2),                            # many splits of few rows
])
def test_attend_against_64_bits(ctx, heads, nkv, D, rot, jobs, budget, sink, recent):
    rng = np.random.default_rng(heads * 7 + D + budget)
    lengths = [max([p + n for s, p, n in jobs if s == slot]) for slot in range(1 + max(j[0] for j in jobs))]
    ref = filled(rng, nkv, D, rot, lengths, spare=2)
    cache = ref.device()
    T = sum(j[2] for j in jobs)
    q = rng.standard_normal((T, heads * D)).astype(np.float32)
    want, vmax, smax = ref.attend(jobs, q, heads, budget, sink, recent)
    got = ctx.attend_pages(cache, jobs, dev(q), budget, sink=sink, recent=recent).numpy()
    off = np.abs(got - want).max(1)
    assert (off <= attend_bound(D, vmax, smax)).all(), (off, attend_bound(D, vmax, smax))


def test_attend_at_strides_beside_other_rows(ctx):
    """q and out as columns of wider rows, at odd strides: the columns beside stay as they were."""
    rng = np.random.default_rng(21)
    ref = filled(rng, 2, 64, 64, [400, 90])
    cache = ref.device()
    jobs = [(0, 399, 1), (1, 88, 2)]
    q = rng.standard_normal((3, 4 * 64 + 7)).astype(np.float32)
    out = np.full((3, 4 * 64 + 3), 5.0, np.float32)
    dq, do = Strided(q, 256), Strided(out, 256)
    ctx.attend_pages(cache, jobs, dq, 3, sink=1, recent=1, out=do)
    got = do.whole.numpy()
    want, vmax, smax = ref.attend(jobs, q[:, :256], 4, 3, 1, 1)
    assert (np.abs(got[:, :256] - want).max(1) <= attend_bound(64, vmax, smax)).all()
    assert (got[:, 256:] == 5.0).all()


def test_attend_equal_scores_keep_the_lower_pages(ctx):
    """Pages of the same keys score the same: the first of them are kept. Values tell the pages apart."""
    rng = np.random.default_rng(22)
    ref = filled(rng, 1, 64, 2, [64 * 12])
    for p in range(12):      # the same key block and bounds, another value in every page
        ref.k[ref.table[0, p]] = ref.k[ref.table[0, 0]]
        ref.bounds[ref.table[0, p]] = ref.bounds[ref.table[0, 0]]
        blk = np.zeros((64, 64))
        blk[:] = p + 1
        code, scale = quantise(blk)
        ref.v[ref.table[0, p], 0, code_index(1, 64)] = (code + 128).astype(np.uint8)
        ref.v.view(np.float32)[ref.table[0, p], 0, 16 * 64 + scale_index(1, 64)] = scale
    cache = ref.device()
    q = rng.standard_normal((1, 64)).astype(np.float32)
    got = ctx.attend_pages(cache, [(0, 64 * 12 - 1, 1)], dev(q), 5, sink=0, recent=1).numpy()
    assert np.allclose(got, (1 + 2 + 3 + 4 + 12) / 5, rtol=1e-5)   # equal weights: the pages' mean, in bounds of f32 sums


def test_attend_is_dense_attention_within_the_budget(gpu):
    """On a context's own cache, with a budget that covers the context: cc_op_attend's output, within both sides' bounds; and
    over fewer pages after cc_kv_bounds."""
    from chattorrent_amd.ccdecode import Context, DeviceArray, KVCache
    d = configs.with_layers(configs.SMOLLM2, 1)
    c = Context(d, n_max=1024, t_max=8, slots=1)
    try:
        c.fill_random_kv(0, 900, 3, 1)
        rng = np.random.default_rng(9)
        q = rng.standard_normal((4, d["n_heads"] * d["head_dim"])).astype(np.float32)
        want = c.op_attend(0, 0, q, 890)
        cache = KVCache.of_context(c, 0)
        got = c.attend_pages(cache, [(0, 890, 4)], dev(q), 16).numpy()
        assert np.abs(got - want).max() <= 2e-5 * np.abs(want).max() * 2
        bytes_ = int(c.lib.cc_bounds_bytes(C.byref(cache.c)))
        bounds = DeviceArray((cache.c.n_pages, bytes_), np.uint8)
        cache = KVCache.of_context(c, 0, bounds=bounds)
        c.kv_bounds(cache, [(0, 0, 894)])
        few = c.attend_pages(cache, [(0, 890, 4)], dev(q), 5).numpy()
        all_ = c.attend_pages(cache, [(0, 890, 4)], dev(q), 14).numpy()
        assert np.abs(all_ - want).max() <= 2e-5 * np.abs(want).max() * 2
        assert np.isfinite(few).all() and np.abs(few - want).max() > 1e-3
    finally:
        c.close()


def test_attend_extreme_scores_and_values(ctx):
    """Queries that put all weight on one token, values with scales past the shifted P.V split, and a page index outside the
    cache, whose tokens are masked."""
    rng = np.random.default_rng(23)
    for scale_q, scale_v in ((400.0, 1.0), (1.0, 3e5), (60.0, 1e-30)):
        ref = filled(rng, 2, 128, 128, [300])
        ref.v.view(np.float32)[:, :, 16 * 128:] *= scale_v
        cache = ref.device()
        q = (rng.standard_normal((1, 4 * 128)) * scale_q).astype(np.float32)
        want, vmax, smax = ref.attend([(0, 299, 1)], q, 4, 3, 1, 1)
        got = ctx.attend_pages(cache, [(0, 299, 1)], dev(q), 3, sink=1, recent=1).numpy()
        assert (np.abs(got - want).max(1) <= attend_bound(128, vmax, smax)).all(), (scale_q, scale_v)
    ref = filled(rng, 1, 64, 64, [250])
    masked = ref.table[0, 1]
    ref.table[0, 1] = 1 << 30
    cache = ref.device()
    q = rng.standard_normal((1, 128)).astype(np.float32)
    got = ctx.attend_pages(cache, [(0, 249, 1)], dev(q), 8).numpy()
    kept = [0, 2, 3]
    ref.table[0, 1] = masked
    ref.kept = lambda *a: kept
    want, vmax, smax = ref.attend([(0, 249, 1)], q, 2, 8, 0, 1)
    assert (np.abs(got - want).max(1) <= attend_bound(64, vmax, smax)).all()
    ref.table[0, :] = -1          # no page at all: zero
    cache = ref.device()
    assert not ctx.attend_pages(cache, [(0, 249, 1)], dev(q), 8).numpy().any()


def of_random_pages(rng, nkv, D, pages, kinds=None):
    """A chat of whole pages of random codes and scales; kinds: only that many different pages of keys."""
    ref = Plain(rng, nkv, D, D, pages, 1, pages)
    for pool in (ref.k, ref.v):
        pool[..., :64 * D] = rng.integers(1, 256, pool[..., :64 * D].shape)
        pool.view(np.float32)[..., 16 * D:] = np.abs(rng.standard_normal((pages, nkv, 2 * D))) * 0.01 + 0.002
    at = np.arange(pages)
    if kinds:
        at = ref.table[0, np.arange(pages) % kinds]
        ref.k[ref.table[0]] = ref.k[at]
    for i in range(pages):
        if kinds and i >= kinds:
            ref.bounds[ref.table[0, i]] = ref.bounds[at[i]]
        else:
            ref.make_bounds(ref.table[0, i])
    return ref


@pytest.mark.parametrize("pages,budget,sink,recent,kinds,nkv,D", [
    (259, 20, 1, 2, None, 2, 64), (260, 20, 1, 2, None, 1, 128),      # 256 and 257 pages to choose from
    (1027, 64, 1, 2, None, 1, 64), (1028, 64, 1, 2, 5, 1, 64),        # 1024, and 1025 of which many score the same
    (700, 650, 1, 2, None, 1, 64), (2600, 900, 3, 5, None, 1, 64),    # long lists, over many workgroups
    (400, 40, 39, 1, None, 1, 64), (300, 30, 0, 1, 2, 1, 64)])
def test_attend_over_many_pages(ctx, pages, budget, sink, recent, kinds, nkv, D):
    rng = np.random.default_rng(pages)
    ref = of_random_pages(rng, nkv, D, pages, kinds)
    cache = ref.device()
    jobs = [(0, 64 * pages - 30, 2), (0, 64 * (pages // 2), 1)]
    q = rng.standard_normal((3, 3 * nkv * D)).astype(np.float32)
    want, vmax, smax = ref.attend(jobs, q, 3 * nkv, budget, sink, recent)
    got = ctx.attend_pages(cache, jobs, dev(q), budget, sink=sink, recent=recent).numpy()
    # beside attend_bound: a lane adds 16 weights a page of up to 64 pages one after another, and as many products
    off, bound = np.abs(got - want).max(1), attend_bound(D, vmax, smax) + 2 * vmax * 16 * 64 * U32
    assert (off <= bound).all(), (off, bound)


@pytest.mark.parametrize("D,size", [(64, 1e6), (64, 1e-9), (128, 3e30), (256, 1e-30), (128, 65504.0)])
def test_attend_queries_of_any_magnitude(ctx, D, size):
    """Queries past f16's range and below it, against keys whose scales bring the scores back to order 1."""
    rng = np.random.default_rng(25)
    ref = of_random_pages(rng, 1, D, 9)
    ref.k.view(np.float32)[..., 16 * D:] /= np.float32(size)
    cache = ref.device()
    q = (rng.standard_normal((2, 4 * D)) * size).astype(np.float32)
    jobs = [(0, 500, 2)]
    want, vmax, smax = ref.attend(jobs, q, 4, 9, 0, 1)
    assert 0.1 < smax.min() and smax.max() < 1e3
    got = ctx.attend_pages(cache, jobs, dev(q), 9).numpy()
    assert (np.abs(got - want).max(1) <= attend_bound(D, vmax, smax)).all()


@pytest.mark.parametrize("D,nkv,budget", [(64, 2, 12), (128, 1, 12), (128, 2, 5), (256, 1, 12)])
def test_attend_values_whose_groups_differ_in_size(ctx, D, nkv, budget):
    """V's 32-channel groups of magnitudes 2^-40 to 2^40 beside each other in a page, the same from page to page or changing
    by 2^20: every channel to the bound of its own group's values."""
    rng = np.random.default_rng(D + budget)
    jobs = [(0, 64 * 12 - 20, 3)]
    for wander in (0, 10):
        ref = of_random_pages(rng, nkv, D, 12)
        scale = ref.v.view(np.float32)[..., 16 * D:]      # [pages, kv heads, 64 tokens' scales by group]
        for h in range(nkv):
            for g, e in enumerate(rng.permutation(np.linspace(-40, 40, D // 32)).round()):
                at = scale_index(1, D)[:, g]
                scale[:, h, at] *= 2.0 ** (e + rng.integers(-wander, wander + 1, (12, 1)))
        cache = ref.device()
        q = rng.standard_normal((3, 3 * nkv * D)).astype(np.float32)
        want, _, smax = ref.attend(jobs, q, 3 * nkv, budget, 1, 2)
        got = ctx.attend_pages(cache, jobs, dev(q), budget).numpy()
        for h in range(nkv):
            vmax = np.max([np.abs(ref.exact_rows(1, page, h)).max(0) for page in ref.table[0]], 0).reshape(-1, 32).max(-1)
            off = np.abs(got - want).reshape(3, nkv, 3, D // 32, 32)[:, h].max((1, 3))
            assert (off <= attend_bound(D, vmax[None], smax[:, None])).all(), (wander, h, off / vmax)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attend_a_page_outside_the_cache_changes_no_other_pages_bits(ctx, D):
    """A page that is none adds nothing, wherever it stands: each of four waves walks two pages, the absent one before or after.
    The tokens of most weight have no values, so that what is left hangs on the last bits of small weights."""
    rng = np.random.default_rng(D)
    ref = of_random_pages(rng, 4, D, 8)
    pages = ref.table[0].copy()
    there = pages[::2]
    ref.table = np.array([[p for a in there for p in (-1, a)], [p for a in there for p in (a, -1)]], np.int32)
    q = (rng.standard_normal((1, 4 * D)) * 5).astype(np.float32)
    at = np.arange(64)[:, None]
    for h in range(4):
        x = rotate32(q[0].reshape(4, D)[h][None], ref.rope[511][None])[0]
        for page in there:
            score = ref.rows(0, page, h) @ x
            heavy = at[score > np.median(score), 0]
            ref.v[page, h, code_index(1, D)[heavy]] = 128
    cache = ref.device(bounds=False)
    rows = dev(np.repeat(q, 128, 0))      # a launch of 128 rows and 4 kv heads: one workgroup each
    got = [ctx.attend_pages(cache, [(slot, 511, 1)] * 128, rows, 8).numpy() for slot in (0, 1)]
    assert same_bits(got[0], got[1]) and got[0].any()


def test_attend_queries_that_are_no_numbers(ctx):
    """A head whose query holds NaN or infinity gives NaN; the other heads and rows what they give without it."""
    rng = np.random.default_rng(26)
    ref = of_random_pages(rng, 2, 64, 40)
    cache = ref.device()
    q = rng.standard_normal((3, 4 * 64)).astype(np.float32)
    jobs = [(0, 2400, 3)]
    for budget in (40, 8):
        clean = ctx.attend_pages(cache, jobs, dev(q), budget).numpy().reshape(3, 4, 64)
        bad = q.reshape(3, 4, 64).copy()
        bad[0, 2:, 7] = np.nan
        bad[2, :2, 30] = np.inf
        got = ctx.attend_pages(cache, jobs, dev(bad.reshape(3, -1)), budget).numpy().reshape(3, 4, 64)
        assert np.isnan(got[0, 2:]).all() and np.isnan(got[2, :2]).all()
        for rows in (np.s_[0, :2], np.s_[1], np.s_[2, 2:]):
            assert same_bits(got[rows], clean[rows])


def test_attend_more_rows_than_a_launch_takes(ctx):
    """8300 rows of one job: each row's bits are those of calls of fewer."""
    rng = np.random.default_rng(27)
    ref = of_random_pages(rng, 1, 64, 130)
    cache = ref.device()
    q = rng.standard_normal((8300, 64)).astype(np.float32)
    whole = ctx.attend_pages(cache, [(0, 17, 8300)], dev(q), 4).numpy()
    for i in range(0, 8300, 1660):
        part = ctx.attend_pages(cache, [(0, 17 + i, 1660)], dev(q[i:i + 1660]), 4).numpy()
        assert same_bits(whole[i:i + 1660], part), i


def test_a_cache_of_more_than_4_gib(ctx):
    """Pages whose bytes lie past 2^31 and 2^32: appended to, scored and read as those of a small cache."""
    from chattorrent_amd.ccdecode import DeviceArray, KVCache
    rng = np.random.default_rng(28)
    nkv, D, n = 8, 256, 30000
    small = Plain(rng, nkv, D, D, 6, 1, 6)
    small.table[0] = np.arange(6)
    near = small.device()
    block = 64 * D + 8 * D
    assert 14563 * nkv * block < 2 ** 31 < 14650 * nkv * block < 29127 * nkv * block < 2 ** 32 < 29250 * nkv * block
    pools = [DeviceArray((n, nkv, block), "uint8") for _ in range(2)]
    far_table = np.array([[29999, 3, 14800, 29400, 14650, 29250]], np.int32)
    far = KVCache(pools[0], pools[1], dev(far_table), small.d[3], D,
                  bounds=DeviceArray((n, nkv * (2 * D + D // 8)), "uint8"))
    k, v = (dev(rng.standard_normal((380, nkv * D)).astype(np.float32)) for _ in range(2))
    q = dev(rng.standard_normal((2, 2 * nkv * D)).astype(np.float32))
    for budget in (6, 3):
        got = []
        for cache in (near, far):
            ctx.kv_append(cache, [(0, 0, 380)], k, v)
            got.append(ctx.attend_pages(cache, [(0, 378, 2)], q, budget).numpy())
        assert same_bits(*got)


def test_attend_twice_gives_the_same_bits(ctx):
    """Split workgroups are joined in split order, whichever ends last."""
    rng = np.random.default_rng(24)
    ref = filled(rng, 2, 128, 128, [4000, 3000])
    cache = ref.device()
    q = dev(rng.standard_normal((2, 10 * 128)).astype(np.float32))
    jobs = [(0, 3999, 1), (1, 2999, 1)]
    first = ctx.attend_pages(cache, jobs, q, 24).numpy()
    for _ in range(5):
        assert same_bits(first, ctx.attend_pages(cache, jobs, q, 24).numpy())


# ------------------------------------------------------------ adjust, sample ---

class Ask:
    """A call's wishes on the host: rows' parameters, histories, biases, masks."""

    def __init__(self, rng, rows, V, history=0, counts=False, biases=0, masks=0, **per_row):
        self.rows, self.V, self.a = rows, V, {}
        for name, value in per_row.items():
            t = np.int32 if name == "top_k" else np.float64 if name == "u" else np.float32
            self.a[name] = np.broadcast_to(np.asarray(value, t), (rows,)).copy()

        def ragged(most):
            n = rng.integers(0, most + 1, rows)
            n[0] = most
            return np.concatenate([[0], np.cumsum(n)]).astype(np.int32), int(n.sum())

        if history:
            self.a["pen_at"], n = ragged(history)
            ids = (V * rng.random(n) ** 4).astype(np.int32)
            ids[rng.random(n) < 0.05] = V + 3        # outside: passed over
            ids[rng.random(n) < 0.05] = -1
            self.a["pen_ids"] = ids
            if counts:
                self.a["pen_counts"] = rng.integers(-1, 4, n).astype(np.int32)
        if biases:
            self.a["bias_at"], n = ragged(biases)
            self.a["bias_ids"] = (V * rng.random(n) ** 2).astype(np.int32)
            b = (rng.standard_normal(n) * 4).astype(np.float32)
            b[rng.random(n) < 0.15] = -np.inf
            self.a["bias"] = b
        if masks:
            words = -(-V // 32) + 1
            bits = rng.random((masks, words * 32)) < np.geomspace(0.01, 0.99, masks)[:, None]
            self.a["mask"] = np.packbits(bits, axis=1, bitorder="little").view(np.uint32).copy()
            self.a["mask_of"] = rng.integers(-1, masks + 1, rows).astype(np.int32)    # masks: out of range, every token
        self.cap = 1.5

    def device(self):
        from chattorrent_amd.ccdecode import Sampling
        return Sampling(self.rows, self.V, freq_cap=self.cap, **{n: dev(a) for n, a in self.a.items()})

    def adjust(self, x):
        """In 64 bits, entry by entry."""
        out = x.astype(np.float64)
        get = self.a.get
        for r in range(self.rows):
            if "pen_at" in self.a:
                lo, hi = self.a["pen_at"][r:r + 2]
                count = {}
                for i in range(lo, hi):
                    t = int(self.a["pen_ids"][i])
                    c = int(self.a["pen_counts"][i]) if "pen_counts" in self.a else 1
                    if 0 <= t < self.V and c > 0:
                        count[t] = count.get(t, 0) + c
                rep = float(self.a["rep"][r]) if "rep" in self.a else 1.0
                freq, pres = (float(self.a[n][r]) if n in self.a else 0.0 for n in ("freq", "pres"))
                for t, c in count.items():
                    v = out[r, t]
                    v = v / rep if v > 0 else v * rep
                    out[r, t] = v - (pres + min(freq * c, self.cap))
            if "bias_at" in self.a:
                lo, hi = self.a["bias_at"][r:r + 2]
                last = {int(self.a["bias_ids"][i]): float(self.a["bias"][i]) for i in range(lo, hi)}
                for t, b in last.items():
                    out[r, t] += b
            if get("mask") is not None:
                m = int(self.a["mask_of"][r])
                if 0 <= m < len(self.a["mask"]):
                    bits = np.unpackbits(self.a["mask"][m].view(np.uint8), bitorder="little")[:self.V]
                    out[r, bits == 0] = -np.inf
        return out

    def sample(self, x):
        """(token, probability, how far u's place in the running sum is from the next border, relative) of each row."""
        adj = self.adjust(x)
        out = []
        for r in range(self.rows):
            with np.errstate(over="ignore"):
                v = adj[r].astype(np.float32)
            v = np.where(np.isnan(v), -np.inf, v).astype(np.float32)
            if not (v > -np.inf).any():
                out.append((-1, 0.0, 1.0))
                continue
            temp = float(self.a["temp"][r]) if "temp" in self.a else 0.0
            if temp <= 0:
                out.append((int(np.argmax(v)), 1.0, 1.0))
                continue
            big = np.finfo(np.float32).max
            with np.errstate(over="ignore"):
                s = np.where(np.isfinite(v), np.clip((v.astype(np.float64) / temp), -big, big), v).astype(np.float32)
            m = s.max()
            with np.errstate(invalid="ignore"):
                w = np.where(s == m, 1.0, np.exp(s.astype(np.float64) - float(m)))
            live = s > -np.inf
            cut = -np.inf
            k = int(self.a["top_k"][r]) if "top_k" in self.a else 0
            if 0 < k < self.V:
                cut = np.sort(s)[::-1][k - 1]
            p = float(self.a["top_p"][r]) if "top_p" in self.a else 1.0
            near = 1.0
            if p < 1:
                on = np.where(live & (s >= cut))[0]
                order = on[np.argsort(-s[on], kind="stable")]
                mass = np.cumsum(w[order])
                want = p * mass[-1]
                i = int(np.argmax(mass >= want)) if want > 0 else 0
                near = np.abs(mass - want).min() / mass[-1]
                cut = max(cut, s[order[i]])
            keep = live & (s >= cut)
            if "min_p" in self.a:
                keep &= w >= min(float(self.a["min_p"][r]), 1.0)
            w = np.where(keep, w, 0.0)
            run = np.cumsum(w)
            at = float(self.a["u"][r]) * run[-1]
            t = int(np.argmax(run > at)) if (run > at).any() else int(np.nonzero(w)[0][-1])
            border = np.abs(run[w > 0] - at).min() / run[-1]
            out.append((t, w[t] / run[-1], min(near, border)))
        return out


def check_sample(ctx, ask, x, ld=None):
    """Tokens equal wherever u (and top-p) is not within a 1e-9 of a border: sums of up to 2^18 weights held to 2^-43 are off
    by 2^-25 of the largest weight at the very most, 2^-34 as roundings add up, and exp in 64 bits agrees to a few 2^-53."""
    d = dev(x) if ld is None else Strided(np.concatenate([x, np.full((len(x), ld - x.shape[1]), 9e9, np.float32)], 1), x.shape[1])
    ids, probs = (a.numpy() for a in ctx.sample(d, ask.device()))
    for r, (t, p, near) in enumerate(ask.sample(x)):
        if near > 1e-9:
            assert ids[r] == t, (r, ids[r], t, near)
            assert abs(probs[r] - p) <= (U32 + 1e-9) * max(p, 1e-300) * 1.01 + 1e-45, (r, probs[r], p)
    return ids


@pytest.mark.parametrize("rows,V,pad", [(1, 1, 0), (2, 31, 1), (3, 4095, 0), (2, 4096, 4), (5, 4097, 3), (4, 49152, 0),
                                        (33, 20011, 5)])
def test_adjust_against_64_bits(ctx, rows, V, pad):
    """Every logit rounded once, untouched ones bit for bit; ids twice in a list, outside the vocabulary, counts of nothing,
    masks out of range; any row stride, in place as well."""
    rng = np.random.default_rng(rows * V + pad)
    x = (rng.standard_normal((rows, V + pad)) * 3).astype(np.float32)
    x[0, 0] = np.nan
    x[-1, V // 2] = np.inf
    x[-1, V // 3] = np.finfo(np.float32).min
    for kw in (dict(), dict(history=50, rep=1.3, freq=0.4, pres=0.25), dict(history=5000, counts=True, freq=0.1),
               dict(biases=60), dict(masks=3), dict(history=300, rep=1.1, pres=0.5, biases=40, masks=2)):
        ask = Ask(rng, rows, V, **kw)
        want = ask.adjust(x[:, :V])
        dx = Strided(x, V)
        got = ctx.adjust_logits(dx, ask.device()).numpy()
        with np.errstate(over="ignore", invalid="ignore"):
            r32 = want.astype(np.float32)
        untouched = np.array_equal(got, r32, equal_nan=True)
        assert untouched, (kw.keys(), np.argwhere(~((got == r32) | (np.isnan(got) & np.isnan(r32))))[:4])
        ctx.adjust_logits(dx, ask.device(), out=dx)
        again = dx.whole.numpy()
        assert np.array_equal(again[:, :V], got, equal_nan=True)
        assert same_bits(again[:, V:], x[:, V:])


@pytest.mark.parametrize("rows,V", [(1, 1), (3, 33), (7, 4096), (2, 4097), (5, 49152), (40, 30001), (600, 9000)])
@pytest.mark.parametrize("kw", [
    dict(), dict(temp=0.7), dict(temp=1.0, top_k=40), dict(temp=1.3, top_p=0.9), dict(temp=0.9, min_p=0.05),
    dict(temp=1.0, top_k=300, top_p=0.7, min_p=0.001), dict(temp=2.0, top_k=1, top_p=0.5), dict(temp=1.0, top_k=7000, top_p=0.99),
], ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()) or "greedy")
def test_sample_against_64_bits(ctx, rows, V, kw):
    rng = np.random.default_rng(rows + V + len(kw))
    x = (rng.standard_normal((rows, V)) * 2.5).astype(np.float32)
    u = rng.random(rows)
    u[0] = 0.0
    check_sample(ctx, Ask(rng, rows, V, u=u, **kw), x)
    check_sample(ctx, Ask(rng, rows, V, u=u, history=200, rep=1.2, freq=0.3, pres=0.1, biases=20, masks=2, **kw), x, ld=V + 3)


def test_sample_rows_that_ask_for_different_things(ctx):
    """Greedy, unrestricted and cut rows in one call; parameters that mean 'off'; u at its ends and outside."""
    rng = np.random.default_rng(31)
    rows, V = 12, 12345
    x = (rng.standard_normal((rows, V)) * 3).astype(np.float32)
    ask = Ask(rng, rows, V, u=[0, 0.5, 0.999999999, 0.3, 0.3, 0.3, 1.0, 0.2, 0.9, 0.1, 0.6, 0.7],
              temp=[0, 1, 1, -1, 1, 1, 0.5, 1, 1, 1, 1, 1], top_k=[5, 0, -3, 5, V, V + 9, 3, 1, 50, 0, 0, 2],
              top_p=[0.1, 1, 2, 0.5, 0.3, 1, 1, 0, 0.9, -1, 0.999, 1], min_p=[0, 0, 0, 0.1, 0, 0, 2, 0, 0.3, 0, 1e-9, 0])
    check_sample(ctx, ask, x)


@pytest.mark.parametrize("V,temp", [(33, 1.0), (4096, 0.6), (12345, 1.0), (151936, 1.8)])
def test_sample_rows_do_not_hang_on_their_neighbours(ctx, V, temp):
    """Each row's token and probability, bit for bit, in a call by itself and beside rows that ask for other cuts; u at the
    borders between tokens, where the last bit of a sum tells."""
    rng = np.random.default_rng(V)
    rows = 96
    x = np.repeat((rng.standard_normal((1, V)) * 2.5).astype(np.float32), rows, 0)
    s = (x[0].astype(np.float64) / np.float64(np.float32(temp))).astype(np.float32).astype(np.float64)
    run = np.cumsum(np.exp(s - s.max()))
    likely = np.searchsorted(run, rng.random(rows) * run[-1])
    u = np.minimum(run[np.minimum(likely, V - 1)] / run[-1], np.nextafter(1.0, 0.0))
    dx = dev(x)

    def draw(pick, u, **kw):
        ids, probs = (a.numpy() for a in ctx.sample(dx, Ask(rng, rows, V, u=u, temp=temp, **kw).device()))
        return ids[pick], probs[pick].view(np.uint32)

    odd = np.arange(rows) % 2 == 1
    off = dict(top_k=np.where(odd, 40, 0), top_p=np.where(odd, 0.9, 1.0), min_p=np.where(odd, 0.01, 0.0))
    for name, alone in (("plain", {}), ("top_k", dict(top_k=np.full(rows, 50))), ("top_p", dict(top_p=np.full(rows, 0.95))),
                        ("min_p", dict(min_p=np.full(rows, 0.001)))):
        want = draw(~odd, u, **alone)
        for others in ({"top_k": off["top_k"]}, {"top_p": off["top_p"]}, {"min_p": off["min_p"]}, off):
            kw = dict(others)
            for n, v in alone.items():      # what the even rows ask for, beside what the odd ones do
                kw[n] = np.where(odd, kw.get(n, v), v)
            got = draw(~odd, u, **kw)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), (name, sorted(others))


def test_sample_ties_infinities_and_empty_rows(ctx):
    """Equal values are kept or cut together; +inf takes everything; the type's lowest value is a value; NaN is none; a row
    that the mask leaves nothing of gives -1 and 0."""
    rng = np.random.default_rng(32)
    V = 9000
    x = np.round(rng.standard_normal((8, V)) * 2).astype(np.float32)       # a dozen distinct values
    x[1, :] = 1.0                                                          # all equal
    x[2, 100] = x[2, 8000] = np.inf
    x[3, :] = np.finfo(np.float32).min
    x[4, :] = np.nan
    x[5, :] = -np.inf
    x[5, 77] = -1e30
    x[6, ::2] = np.nan
    u = rng.random(8)
    for kw in (dict(), dict(temp=0.5), dict(temp=0.5, top_k=10), dict(temp=0.8, top_p=0.4), dict(temp=1.0, top_k=4000, top_p=0.8)):
        ids = check_sample(ctx, Ask(rng, 8, V, u=u, **kw), x)
        assert ids[2] in (100, 8000) and ids[4] == -1 and ids[5] == 77
    ask = Ask(rng, 8, V, u=u, temp=1.0, top_k=5, masks=1)
    ask.a["mask"][:] = 0
    ask.a["mask_of"][:] = 0
    ids = check_sample(ctx, ask, x)
    assert (ids == -1).all()


@pytest.mark.parametrize("spread", [0.0, 1e-4, 0.02])
def test_sample_among_nearly_equal_logits(ctx, spread):
    """More values share the cut's bin than are gathered: the row is drawn in passes, to the same token."""
    rng = np.random.default_rng(33)
    rows, V = 2, 50000
    x = (rng.standard_normal((rows, V)) * spread).astype(np.float32)
    x[:, 17] = -40.0 if spread else 0.0      # one far value keeps the bins wide
    for kw in (dict(top_p=0.6), dict(top_k=20000), dict(top_k=30000, top_p=0.5, min_p=0.1)):
        check_sample(ctx, Ask(rng, rows, V, u=rng.random(rows), temp=1.0, **kw), x)


@pytest.mark.parametrize("V", [9001, 49152, 151936])
@pytest.mark.parametrize("kw", [
    dict(top_k=700), dict(top_k=1000), dict(top_k=3000), dict(top_k=7000), dict(top_k=3000, min_p=0.05), dict(top_k=2000, min_p=1e-4)],
    ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()))
def test_sample_with_a_large_top_k_alone(ctx, V, kw):
    """More values above the cut's bin than are gathered whole, and no top-p: the weights before the bin are summed by the
    workgroups themselves. The draw over the whole range of u, so that a chunk's weight that is off shows in the token."""
    rng = np.random.default_rng(V + len(kw))
    rows = 16
    x = (rng.standard_normal((rows, V)) * 2.5).astype(np.float32)
    for temp in (1.0, 1.7):
        check_sample(ctx, Ask(rng, rows, V, u=(np.arange(rows) + rng.random(rows)) / rows, temp=temp, **kw), x)


def test_sample_with_the_cut_in_the_last_bin(ctx):
    """Flat rows under a few higher values: the k-th largest lies in the last bin, and the weights before it count."""
    rng = np.random.default_rng(38)
    rows, V = 8, 20011
    x = np.full((rows, V), -np.inf, np.float32)
    for r in range(rows):
        at = rng.choice(V, 3000, replace=False)
        x[r, at] = rng.standard_normal(3000) * 1e-4
        x[r, at[:200]] = rng.uniform(1.5, 2.0, 200)
    for kw in (dict(top_k=900), dict(top_k=2500), dict(top_k=2500, min_p=0.01), dict(top_k=V - 1)):
        check_sample(ctx, Ask(rng, rows, V, u=(np.arange(rows) + rng.random(rows)) / rows, temp=1.0, **kw), x)


@pytest.mark.parametrize("top", [0.0, 1e-30, -1e-40, 1e-8, 2.0 ** 26, -3.4028234663852886e38])
def test_sample_with_min_p_at_its_end(ctx, top):
    """min-p at and next to 1, where next to zero a great many f32 values share the largest weight, and where a step of f32 at the
    largest value is longer than the whole range of weights."""
    rng = np.random.default_rng(35)
    V = 3000
    x = np.full((4, V), np.float32(top))
    x[:, ::3] = np.nextafter(np.float32(top), np.float32(-np.inf))
    x[:, 1::3] = -np.inf if top < -1e38 else np.float32(top - 2 * max(1.0, abs(top)))
    x[2:, 5] = x[2:, 8] = 0.0 if -1e-39 < top < 0 else top
    for p in (1.0, 0.999999, 0.5):
        for kw in (dict(), dict(top_k=40), dict(top_p=0.9)):
            check_sample(ctx, Ask(rng, 4, V, u=rng.random(4), temp=1.0, min_p=p, **kw), x)


def test_sample_at_infinite_temperature_and_parameters_that_are_no_numbers(ctx):
    """All allowed tokens alike at temperature infinity, barred ones never; a top-p or min-p of NaN cuts nothing, a temperature
    of NaN is greedy."""
    rng = np.random.default_rng(37)
    V = 9000
    x = (rng.standard_normal((6, V)) * 3).astype(np.float32)
    x[:, ::2] = -np.inf
    u = rng.random(6)
    for kw in (dict(), dict(top_k=5), dict(top_p=0.5), dict(min_p=0.5)):
        for temp in (np.inf, np.finfo(np.float32).max):
            ids = check_sample(ctx, Ask(rng, 6, V, u=u, temp=temp, masks=1, **kw), x)
            assert (ids % 2 == 1).all()
    plain = ctx.sample(dev(x), Ask(rng, 6, V, u=u, temp=1.0).device())
    for kw in (dict(top_p=np.nan), dict(min_p=np.nan), dict(top_p=np.nan, min_p=np.nan, top_k=-5)):
        got = ctx.sample(dev(x), Ask(rng, 6, V, u=u, temp=1.0, **kw).device())
        assert np.array_equal(got[0].numpy(), plain[0].numpy())
    assert np.array_equal(ctx.sample(dev(x), Ask(rng, 6, V, u=u, temp=np.nan, top_k=5).device())[0].numpy(), x.argmax(1))


def test_the_largest_vocabulary_and_long_lists(ctx):
    """2^20 logits a row, odd ones beside; more than 2^16 entries in a row's lists, many of one token."""
    rng = np.random.default_rng(36)
    V = 1 << 20
    x = (rng.standard_normal((2, V)) * 2).astype(np.float32)
    for kw in (dict(), dict(temp=1.0), dict(temp=0.8, top_k=1000, top_p=0.95)):
        check_sample(ctx, Ask(rng, 2, V, u=rng.random(2), history=70000, rep=1.1, freq=0.01, pres=0.3, biases=100, masks=1, **kw), x)
    V = 9001
    x = (rng.standard_normal((2, V)) * 2).astype(np.float32)
    for kw in (dict(history=70000, rep=1.1, freq=0.01, biases=70000), dict(history=70000, counts=True, freq=0.01, biases=9)):
        ask = Ask(rng, 2, V, **kw)
        got = ctx.adjust_logits(dev(x), ask.device()).numpy()
        with np.errstate(over="ignore", invalid="ignore"):
            assert np.array_equal(got, ask.adjust(x).astype(np.float32), equal_nan=True)


def test_list_offsets_outside_the_lists(ctx):
    """Rows whose offsets lie before or past the lists, next to the ends of 32 bits, or run backwards: the entries within count."""
    rng = np.random.default_rng(39)
    V, top, low = 9001, 2**31 - 1, -2**31
    pairs = [(top, top), (low, top), (top - 3, low), (7, 3), (low, 5), (20, top), (top - 200, top), (0, 40), (40, 40), (-1, 41)]
    x = (rng.standard_normal((len(pairs), V)) * 2).astype(np.float32)
    for pen in (True, False):
        for r, (lo, hi) in enumerate(pairs):   # a row a call, beside one with entries of both kinds
            ask = Ask(rng, 2, V, history=40, rep=1.3, freq=0.4, pres=0.25, biases=40)
            n = {name: len(ask.a[name + "_ids"]) for name in ("pen", "bias")}
            name = "pen" if pen else "bias"
            ask.a[name + "_at"] = np.array([lo, hi, n[name]], np.int32)
            other = "bias" if pen else "pen"
            ask.a[other + "_at"] = np.array([0, n[other] // 2, n[other]], np.int32)
            got = ctx.adjust_logits(dev(x[:2]), ask.device()).numpy()
            for row in range(2):
                ends = [min(max(int(e), 0), n[name]) for e in ask.a[name + "_at"][row:row + 2]]
                one = Ask(rng, 1, V)
                one.a = {k: v[row:row + 1] if k in ("rep", "freq", "pres") else v for k, v in ask.a.items()}
                one.a[name + "_at"] = np.array([ends[0], max(ends)], np.int32)
                one.a[other + "_at"] = ask.a[other + "_at"][row:row + 2]
                with np.errstate(over="ignore", invalid="ignore"):
                    want = one.adjust(x[row:row + 1])[0].astype(np.float32)
                assert np.array_equal(got[row], want, equal_nan=True), (name, lo, hi, row)


def test_counts_that_pass_32_bits(ctx):
    """An id's counts add up past 2^31, to 2^32 - 1 at most, whatever their order and beside biases of the same ids."""
    rng = np.random.default_rng(40)
    V, top = 5000, 2**31 - 1
    x = (rng.standard_normal((1, V)) * 2).astype(np.float32)
    #           2^31          2^32 - 2      2^32 - 1          past it                two of 2^30      one and nothing
    sums = {3: [top, 1], 4: [top, top], 2500: [top, top, 1], 4999: [top] * 5 + [7], 70: [2**30] * 2, 71: [1, -5, 0]}
    ids = np.array([t for t, c in sums.items() for _ in c], np.int32)
    counts = np.array([v for c in sums.values() for v in c], np.int32)
    order = rng.permutation(len(ids))
    for freq, biases in ((2.0 ** -33, False), (2.0 ** -33, True), (0.0, False)):
        kw = dict(biases=3) if biases else {}
        ask = Ask(rng, 1, V, rep=1.5, freq=freq, pres=0.25, **kw)
        ask.a.update(pen_at=np.array([0, len(ids)], np.int32), pen_ids=ids[order], pen_counts=counts[order])
        if biases:
            ask.a["bias_ids"][:] = [4999, 3, 4]
        got = ctx.adjust_logits(dev(x), ask.device()).numpy()[0]
        held = {t: min(sum(v for v in c if v > 0), 2**32 - 1) for t, c in sums.items()}
        ask.a.update(pen_at=np.array([0, len(held)]), pen_ids=np.array(list(held)), pen_counts=np.array(list(held.values())))
        want = ask.adjust(x)[0]
        with np.errstate(over="ignore", invalid="ignore"):
            assert np.array_equal(got, want.astype(np.float32), equal_nan=True), (freq, biases)


def test_sample_follows_its_distribution(ctx):
    """4096 draws of one row: each token's share within five standard deviations of its weight."""
    rng = np.random.default_rng(34)
    rows, V = 4096, 50
    x = np.repeat((rng.standard_normal((1, V)) * 1.5).astype(np.float32), rows, 0)
    ids, probs = (a.numpy() for a in ctx.sample(dev(x), Ask(rng, rows, V, temp=1.0, u=(np.arange(rows) + 0.5) / rows).device()))
    w = np.exp(x[0].astype(np.float64) - x[0].max())
    w /= w.sum()
    share = np.bincount(ids, minlength=V) / rows
    assert (np.abs(share - w) <= 2.0 / rows).all()      # u in even steps: within a step at either end
    assert np.abs(probs - w[ids]).max() <= 1e-6


# ------------------------------------------------------ streams, graphs, runs ---

@pytest.fixture()
def hip(gpu):
    from tests.test_zz_no_alloc import _Hip
    h = _Hip()
    yield h
    h.free()


TORCH_STREAMS = """
import numpy as np, torch
from chattorrent_amd import ccdecode as cc, configs
ctx = cc.Context(configs.with_layers(configs.SMOLLM2, 1), n_max=256, t_max=8, slots=2)
V = 1 << 20
x = torch.randn(2, V, device="cuda")
ask = cc.Sampling(2, V, temp=torch.ones(2, device="cuda"), u=torch.tensor([0.3, 0.6], dtype=torch.float64, device="cuda"))
here = [t.clone() for t in (*ctx.sample(x, ask), ctx.adjust_logits(x, ask))]
torch.cuda.synchronize()
side = torch.cuda.Stream()
for stream in (side.cuda_stream, 0):
    got = [*ctx.sample(x, ask, stream=stream), ctx.adjust_logits(x, ask, stream=stream)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(here, got)), stream
    at = got[2].data_ptr()
    del got
    again = torch.empty(2, V, device="cuda")
    # what is let go is given on to the stream that wrote it, and to no other
    assert (again.data_ptr() != at) == (stream != 0), stream
    with torch.cuda.stream(side):
        other = torch.empty(2, V, device="cuda")
    assert (other.data_ptr() == at) == (stream != 0), stream
    del again, other
print("held")
"""


def test_torch_memory_of_a_call_belongs_to_its_stream(gpu):
    r = subprocess.run([sys.executable, "-c", TORCH_STREAMS], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True,
                       timeout=110)
    assert r.returncode == 0 and r.stdout.strip().endswith("held"), r.stdout


def test_operators_on_two_streams_at_once(ctx, hip):
    """Calls on two streams of the caller's, each with its own workspace, overlapping: each gives what it gives alone."""
    rng = np.random.default_rng(41)
    ref = filled(rng, 2, 128, 128, [3000, 2500])
    cache = ref.device()
    q = [dev(rng.standard_normal((1, 8 * 128)).astype(np.float32)) for _ in range(2)]
    x = [dev((rng.standard_normal((4, 30000)) * 3).astype(np.float32)) for _ in range(2)]
    ask = [Ask(rng, 4, 30000, temp=1.0, top_p=0.9, u=rng.random(4)).device() for _ in range(2)]
    alone = [(ctx.attend_pages(cache, [(i, 2400, 1)], q[i], 9).numpy(), ctx.sample(x[i], ask[i])[0].numpy()) for i in range(2)]
    st = [C.c_void_p() for _ in range(2)]
    for s in st:
        hip.check(hip.h.hipStreamCreate(C.byref(s)))
    held = []
    for _ in range(6):
        for i in range(2):
            held.append((i, ctx.attend_pages(cache, [(i, 2400, 1)], q[i], 9, stream=st[i].value),
                         ctx.sample(x[i], ask[i], stream=st[i].value)[0]))
    for s in st:
        hip.check(hip.h.hipStreamSynchronize(s))
    for i, a, b in held:
        assert same_bits(a.numpy(), alone[i][0]) and same_bits(b.numpy(), alone[i][1])
    for s in st:
        hip.check(hip.h.hipStreamDestroy(s))


def test_a_captured_step_replays(ctx, hip):
    """Append, attend, adjust and sample captured into one graph on the caller's stream, replayed four times over new inputs
    with eager calls between: every replay equals the eager calls' bits on that replay's inputs. Two graphs that hold their
    own workspaces do not disturb each other."""
    from chattorrent_amd.ccdecode import DeviceArray
    lib, rng = ctx.lib, np.random.default_rng(42)
    ref = filled(rng, 2, 64, 64, [700, 640])
    cache = ref.device()
    jobs = np.array([(0, 699, 1), (1, 639, 1)], np.int32)      # the second completes a page
    V, heads, budget = 12000, 6, 5
    k, v, q = (DeviceArray((2, w), np.float32) for w in (128, 128, heads * 64))
    x = DeviceArray((2, V), np.float32)
    ask = Ask(rng, 2, V, temp=0.9, top_p=0.8, top_k=200, history=40, rep=1.1, u=[0.3, 0.8])
    sampling = ask.device()
    need = lib.cc_attend_workspace(ctx.h, cache.ref, 2, heads, budget)
    need2 = lib.cc_sample_workspace(2, V, sampling.ref)
    graphs = []
    for g in range(2):
        ws, ws2 = DeviceArray((need,), np.uint8), DeviceArray((need2,), np.uint8)
        out, ids, probs = DeviceArray((2, heads * 64), np.float32), DeviceArray((2,), np.int32), DeviceArray((2,), np.float32)
        adj = DeviceArray((2, V), np.float32)
        st, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
        hip.check(hip.h.hipStreamCreate(C.byref(st)))
        hip.check(hip.h.hipStreamBeginCapture(st, 2))
        code = [lib.cc_kv_append(ctx.h, cache.ref, jobs.ctypes.data, 2, k.data_ptr(), 128, v.data_ptr(), 128, st),
                lib.cc_attend_pages(ctx.h, cache.ref, jobs.ctypes.data, 2, heads, budget, 1, 2, q.data_ptr(), heads * 64,
                                    out.data_ptr(), heads * 64, ws.data_ptr(), need, st),
                lib.cc_logits_adjust(ctx.h, x.data_ptr(), V, 2, V, sampling.ref, adj.data_ptr(), V, st),
                lib.cc_sample(ctx.h, x.data_ptr(), V, 2, V, sampling.ref, ids.data_ptr(), probs.data_ptr(), ws2.data_ptr(),
                              need2, st)]
        hip.check(hip.h.hipStreamEndCapture(st, C.byref(graph)))
        assert code == [0] * 4, lib.cc_last_error(ctx.h)
        hip.check(hip.h.hipGraphInstantiate(C.byref(exe), graph, None, None, 0))
        graphs.append((st, graph, exe, out, ids, adj, (ws, ws2, probs)))
    for rep in range(4):
        for a, scale in ((k, 1), (v, 1), (q, 1), (x, 3)):
            a.set((rng.standard_normal(a.shape) * scale).astype(np.float32))
        for st, _, exe, *_ in graphs:
            hip.check(hip.h.hipGraphLaunch(exe, st))
        for st, *_ in graphs:
            hip.check(hip.h.hipStreamSynchronize(st))
        got = [[a.numpy() for a in g[3:6]] + [ref.d[0].numpy(), ref.d[4].numpy()] for g in graphs]
        ctx.kv_append(cache, jobs, k, v)
        want = [ctx.attend_pages(cache, jobs, q, budget).numpy(), ctx.sample(x, sampling)[0].numpy(),
                ctx.adjust_logits(x, sampling).numpy(), ref.d[0].numpy(), ref.d[4].numpy()]
        for g in got:
            for a, b in zip(g, want):
                assert same_bits(a, b), rep
    for st, graph, exe, *_ in graphs:
        hip.h.hipGraphExecDestroy(exe)
        hip.h.hipGraphDestroy(graph)
        hip.check(hip.h.hipStreamDestroy(st))


def test_a_decode_loop_of_all_four(ctx):
    """Three chats decode 70 tokens each, past a page's end: append, attend over selected pages, logits from the output, and
    the draw under a growing history; every step against the plain steps."""
    rng = np.random.default_rng(43)
    nkv, D, heads, V = 2, 64, 6, 600
    lengths = [500, 130, 60]
    ref = filled(rng, nkv, D, D, [n + 70 for n in lengths], spare=1)
    cache = ref.device()
    W = rng.standard_normal((heads * D, V)).astype(np.float32) / 8
    history = [[] for _ in lengths]
    for step in range(70):
        jobs = [(s, n + step, 1) for s, n in enumerate(lengths)]
        k, v = (rng.standard_normal((3, nkv * D)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((3, heads * D)).astype(np.float32)
        ctx.kv_append(cache, jobs, dev(k), dev(v))
        ref.append(jobs, k, v)
        got = ctx.attend_pages(cache, jobs, dev(q), 4, sink=1, recent=1).numpy()
        want, vmax, smax = ref.attend(jobs, q, heads, 4, 1, 1)
        assert (np.abs(got - want).max(1) <= attend_bound(D, vmax, smax)).all(), step
        ask = Ask(rng, 3, V, temp=0.8, top_k=30, rep=1.2, freq=0.2, u=rng.random(3))
        ask.a["pen_at"] = np.concatenate([[0], np.cumsum([len(h) for h in history])]).astype(np.int32)
        ask.a["pen_ids"] = np.array(sum(history, []) or [0], np.int32)
        ids = check_sample(ctx, ask, (got @ W).astype(np.float32))
        for h, t in zip(history, ids):
            h.append(int(t))
    assert same_bits(ref.d[0].numpy(), ref.k) and same_bits(ref.d[1].numpy(), ref.v)


# ----------------------------------------------------------------- refusals ---

def refuses(ctx, word, call):
    from chattorrent_amd.ccdecode import CCError
    with pytest.raises((CCError, ValueError)) as e:
        call()
    assert word in str(e.value), str(e.value)


def test_refusals_of_the_cache_operators(ctx):
    rng = np.random.default_rng(51)
    ref = Plain(rng, 2, 64, 64, 8, 2, 4)
    cache = ref.device()
    bare = ref.device(bounds=False)
    rows, q = dev(np.zeros((1, 128), np.float32)), dev(np.zeros((1, 256), np.float32))
    for jobs in ([(2, 0, 1)], [(-1, 0, 1)], [(0, -1, 1)], [(0, 256, 1)], [(0, 2**31 - 1, 1)]):
        refuses(ctx, "job 0", lambda: ctx.kv_append(cache, jobs, rows, rows))
        refuses(ctx, "job 0", lambda: ctx.attend_pages(cache, jobs, q, 4))
    two = dev(np.zeros((2, 128), np.float32))
    refuses(ctx, "twice", lambda: ctx.kv_append(cache, [(1, 0, 1), (1, 5, 1)], two, two))
    refuses(ctx, "at least one", lambda: ctx.kv_append(cache, np.zeros((0, 3), np.int32), dev(np.zeros((0, 128), np.float32)),
                                                       dev(np.zeros((0, 128), np.float32))))
    refuses(ctx, "k:", lambda: ctx.kv_append(cache, [(0, 0, 1)], q, rows))
    refuses(ctx, "v:", lambda: ctx.kv_append(cache, [(0, 0, 1)], rows, dev(np.zeros((1, 128), np.float64))))
    refuses(ctx, "bounds", lambda: ctx.attend_pages(bare, [(0, 255, 1)], q, 3))
    refuses(ctx, "bounds", lambda: ctx.kv_bounds(bare, [(0, 0, 64)]))
    refuses(ctx, "budget", lambda: ctx.attend_pages(cache, [(0, 255, 1)], q, 0))
    for sink, recent in ((-1, 1), (0, 0), (3, 1), (2**31 - 1, 2)):
        refuses(ctx, "sink", lambda: ctx.attend_pages(cache, [(0, 255, 1)], q, 3, sink=sink, recent=recent))
    refuses(ctx, "multiple", lambda: ctx.attend_pages(cache, [(0, 5, 1)], dev(np.zeros((1, 192), np.float32)), 3))
    refuses(ctx, "whole heads", lambda: ctx.attend_pages(cache, [(0, 5, 1)], dev(np.zeros((1, 200), np.float32)), 3))
    lib, jobs = ctx.lib, np.array([(0, 255, 1)], np.int32)
    ws = dev(np.zeros(1 << 16, np.uint8))

    def attend(**kw):
        a = dict(ws=ws.data_ptr(), n=1 << 16, ldq=256, ldo=256)
        a.update(kw)
        return lib.cc_attend_pages(ctx.h, cache.ref, jobs.ctypes.data, 1, 4, 3, 1, 1, q.data_ptr(), a["ldq"], q.data_ptr(),
                                   a["ldo"], a["ws"], a["n"], None)

    assert attend(ws=None) == 5 and attend(n=16) == 5 and attend(ws=ws.data_ptr() + 4) == 5
    assert attend(ldq=255) == 5 and attend(ldo=0) == 5
    assert lib.cc_attend_pages(None, cache.ref, jobs.ctypes.data, 1, 4, 3, 1, 1, q.data_ptr(), 256, q.data_ptr(), 256,
                               ws.data_ptr(), 1 << 16, None) == 5
    assert lib.cc_kv_append(ctx.h, None, jobs.ctypes.data, 1, rows.data_ptr(), 128, rows.data_ptr(), 128, None) == 5
    for field, bad in (("head_dim", 96), ("rot_dim", 3), ("rot_dim", 66), ("n_kv_heads", 0), ("max_pages", 40000),
                       ("n_pages", 0), ("slots", 0), ("rope_rows", 0), ("k", None), ("rope", None), ("v", cache.c.v + 8)):
        old = getattr(cache.c, field)
        setattr(cache.c, field, bad)
        try:
            assert lib.cc_kv_append(ctx.h, cache.ref, jobs.ctypes.data, 1, rows.data_ptr(), 128, rows.data_ptr(), 128,
                                    None) == 5, field
        finally:
            setattr(cache.c, field, old)
    with pytest.raises(Exception):
        from chattorrent_amd.ccdecode import KVCache
        KVCache.of_context(ctx, 7)


def test_refusals_of_the_logits_operators(ctx):
    from chattorrent_amd.ccdecode import Sampling
    rng = np.random.default_rng(52)
    x = dev(np.zeros((2, 100), np.float32))
    lib = ctx.lib
    plain = Sampling(2, 100)
    refuses(ctx, "logits:", lambda: ctx.sample(dev(np.zeros((2, 99), np.float32)), plain))
    refuses(ctx, "logits:", lambda: ctx.adjust_logits(dev(np.zeros((3, 100), np.float32)), plain))
    refuses(ctx, "random", lambda: ctx.sample(x, Sampling(2, 100, temp=dev(np.ones(2, np.float32)))))
    refuses(ctx, "history", lambda: ctx.adjust_logits(x, Sampling(2, 100, rep=dev(np.ones(2, np.float32)))))
    refuses(ctx, "words", lambda: Sampling(2, 100, mask=dev(np.zeros((1, 3), np.uint32)), mask_of=dev(np.zeros(2, np.int32))))
    refuses(ctx, "mask_of", lambda: ctx.adjust_logits(x, Sampling(2, 100, mask=dev(np.zeros((1, 4), np.uint32)))))
    refuses(ctx, "temp", lambda: Sampling(2, 100, temp=dev(np.ones(3, np.float32))))
    refuses(ctx, "u:", lambda: Sampling(2, 100, u=dev(np.ones(2, np.float32))))
    refuses(ctx, "freq_cap", lambda: ctx.adjust_logits(x, Sampling(2, 100, freq_cap=-1.0)))
    refuses(ctx, "pen_ids", lambda: Sampling(2, 100, pen_ids=dev(np.zeros(4, np.int64))))
    ids, ws = dev(np.zeros(2, np.int32)), dev(np.zeros(1 << 20, np.uint8))
    need = lib.cc_sample_workspace(2, 100, plain.ref)
    assert 0 < need <= 1 << 20
    assert lib.cc_sample_workspace(0, 100, plain.ref) == 0 and lib.cc_sample_workspace(2, (1 << 20) + 1, plain.ref) == 0
    assert lib.cc_sample_workspace(2, 100, None) == 0

    def sample(rows=2, V=100, ld=100, ws_=ws.data_ptr(), n=need):
        return lib.cc_sample(ctx.h, x.data_ptr(), ld, rows, V, plain.ref, ids.data_ptr(), None, ws_, n, None)

    assert sample() == 0
    assert sample(rows=0) == 5 and sample(V=0) == 5 and sample(ld=99) == 5 and sample(n=need - 1) == 5
    assert sample(ws_=None) == 5 and sample(ws_=ws.data_ptr() + 8) == 5 and sample(rows=65536) == 5
    assert sample(V=(1 << 20) + 1, ld=1 << 21) == 5
    assert lib.cc_logits_adjust(ctx.h, x.data_ptr(), 100, 2, 90, plain.ref, x.data_ptr(), 95, None) == 5

"""The operators of a cache held within a bound (cc_kv_append_at, cc_attend_weigh,
cc_kv_evict) against plain implementations in numpy, in 64 bits, through the C
ABI, at the sizes and masks where they can go wrong; their use on streams, in
captured graphs and at addresses past 32 bits; and a run of them together."""
import math
import subprocess
import sys

import numpy as np
import pytest

from chattorrent_amd import configs
from test_gpu_operators import ROOT, Plain, Strided, code_index, dev, hip, quantise, same_bits, scale_index  # noqa: F401

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24      # half a step of f32, relative to the value


@pytest.fixture(scope="module")
def ctx(gpu):
    from chattorrent_amd.ccdecode import Context
    c = Context(configs.with_layers(configs.SMOLLM2, 1), n_max=256, t_max=8, slots=2)
    yield c
    c.close()


# ------------------------------------------------------------------- plain ---

class Kept(Plain):
    """Plain's paged cache with marks, and positions that are not the rows' indices."""

    def __init__(self, rng, nkv, D, rot, n_pages, slots, max_pages, rope_rows=700, **kw):
        super().__init__(rng, nkv, D, rot, n_pages, slots, max_pages, **kw)
        inv = 10000.0 ** (-2.0 * np.arange(rot // 2) / rot)
        ang = np.arange(rope_rows)[:, None] * inv
        self.rope = np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)
        self.weight = np.full((n_pages, nkv, 64), np.nan, np.float32)     # nothing set yet
        self.token = np.full((n_pages, nkv, 64), -7, np.int32)

    def device(self, bounds=False):
        from chattorrent_amd.ccdecode import Marks
        cache = super().device(bounds)
        self.m = dev(self.weight), dev(self.token)
        return cache, Marks(*self.m)

    def same(self):
        """Whether the device's cache and marks are these, bit for bit."""
        for a, b in ((self.d[0], self.k), (self.d[1], self.v), (self.m[0], self.weight), (self.m[1], self.token)):
            if not np.array_equal(a.numpy().view(np.uint8), b.view(np.uint8)):
                return False
        return True

    def angles(self, pos, axis_of):
        """(cos, sin) [rot/2, 2] of a row at positions pos [axes]."""
        j = np.arange(self.rot // 2)
        at = np.clip(pos, 0, len(self.rope) - 1)
        return self.rope[at[axis_of] if axis_of is not None else np.full(len(j), at[0]), j]

    def append_at(self, jobs, k, v, pos=None, axis_of=None, first=None):
        row = 0
        for j, (slot, past, n) in enumerate(jobs):
            for i in range(n):
                p = past + i
                page, t = self.table[slot, p // 64], p % 64
                cs = self.angles(np.array([p]) if pos is None else pos[row], None if pos is None else axis_of)
                x = k[row].reshape(self.nkv, self.D)
                h = self.rot // 2
                a, o, c, s = x[:, :h], x[:, h:2 * h], cs[:, 0], cs[:, 1]
                kr = np.concatenate([a * c - o * s, o * c + a * s, x[:, 2 * h:]], -1).astype(np.float32)
                for which, pool, y in ((0, self.k, kr), (1, self.v, v[row].reshape(self.nkv, self.D))):
                    code, scale = quantise(y)
                    for hd in range(self.nkv):
                        pool[page, hd, code_index(which, self.D)[t]] = (code[hd] + 128).astype(np.uint8)
                        pool.view(np.float32)[page, hd, 16 * self.D + scale_index(which, self.D)[t]] = scale[hd]
                self.weight[page, :, t] = 0.0
                self.token[page, :, t] = (past if first is None else first[j]) + i
                row += 1
            for p in range(past // 64, (past + n) // 64):
                self.make_bounds(self.table[slot, p])

    def weigh(self, jobs, q, heads, pos=None, axis_of=None, observe=1 << 30, fade=1.0):
        """(output and the slots' weights [n_pages, nkv, 64] in 64 bits, bounds on how far each may be off).

        A score is a sum of D products of pairs (q and, in the sums over many columns, k to 2^-22 of their values, the
        products of their lower halves left out), each addition rounded, scaled and shifted in one more rounding: off by
        es = smax * (3 * 2^-22 + (D + 12) * 2^-24) of the magnitudes' sum smax, plus 32 * 2^-24 for the shift and v_exp.
        Numerator and sum each carry it, and the f32 sums over T tokens, at most T/4 + 64 additions deep; a value's pair and
        the joins take another 2^-20. exp(es) - 1 and not es: a score of thousands is off by more than a little."""
        G, D = heads // self.nkv, self.D
        out, bound = np.zeros((len(q), heads, D)), np.zeros(len(q))
        weight, wbound = self.weight.astype(np.float64), np.zeros(self.weight.shape)
        row = 0
        for slot, past, n in jobs:
            T = past + n
            pages = self.table[slot, :-(-T // 64)]
            there = np.repeat(pages.astype(np.uint32) < len(self.k), 64)[:T]
            fine = np.where(pages.astype(np.uint32) < len(self.k), pages, 0)
            for h in range(self.nkv):
                kk, vv = (np.concatenate([self.exact_rows(w, p, h) for p in fine])[:T] for w in (0, 1))
                got, worst = np.zeros(T), 0.0
                for i in range(n):
                    r = row + i
                    cs = self.angles(np.array([past + i]) if pos is None else pos[r], None if pos is None else axis_of)
                    x = q[r].reshape(heads, D)[h * G:(h + 1) * G].astype(np.float64)
                    m = self.rot // 2
                    a, o, c, s = x[:, :m], x[:, m:2 * m], cs[:, 0].astype(np.float64), cs[:, 1].astype(np.float64)
                    x = np.concatenate([a * c - o * s, o * c + a * s, x[:, 2 * m:]], -1)
                    ok = there & (np.arange(T) <= past + i)
                    if not ok.any():
                        continue
                    s = x @ kk[ok].T / math.sqrt(D)
                    w = np.exp(s - s.max(-1, keepdims=True))
                    w /= w.sum(-1, keepdims=True)
                    out[r, h * G:(h + 1) * G] = w @ vv[ok]
                    smax = (np.abs(x) @ np.abs(kk[ok]).T).max() / math.sqrt(D)
                    e = np.expm1(smax * (3 * 2.0 ** -22 + (D + 12) * U32) + 32 * U32)
                    e = 2 * e + 2 * (T / 4 + 64) * U32 + 2.0 ** -20
                    bound[r] = max(bound[r], np.abs(vv[ok]).max() * e)
                    if i >= n - observe:
                        got[ok] += w.sum(0)
                        worst = max(worst, e)
                t = np.arange(T)[there]
                at = (pages[t // 64], h, t % 64)
                old = np.where(np.float32(fade) == 0, 0.0, weight[at] * np.float64(np.float32(fade)))
                if observe > 0:
                    weight[at] = old + got[t]
                    wbound[at] = (got[t] * (worst + n * G * U32) + 2 * U32 * (np.abs(old) + got[t])
                                  + n * G * 2.0 ** -125)       # what is below f32's least normal value counts as none
            row += n
        return out.reshape(len(q), -1), bound, weight, wbound

    def evict(self, jobs, sink, recent):
        for slot, rows, keep, seen in jobs:
            if rows <= keep:
                continue
            r = np.arange(rows)
            page = self.table[slot, r // 64]
            there = page.astype(np.uint32) < len(self.k)
            for h in range(self.nkv):
                w = np.full(rows, -np.inf)
                tok = np.full(rows, -1)
                w[there], tok[there] = (a[page[there], h, r[there] % 64] for a in (self.weight, self.token))
                safe = there & ((tok < sink) | (tok >= seen - recent))     # alike: the lower rows of them first
                rank = np.where(safe, np.inf, np.where(np.isnan(w), -np.inf, w))
                order = np.lexsort((r, -rank, np.isnan(w) & ~safe, ~there, ~safe))
                gone = np.ones(rows, bool)
                gone[order[:keep]] = False
                for to, of in zip(r[:keep][gone[:keep]], r[keep:][~gone[keep:]]):
                    if not (there[to] and there[of]):
                        continue
                    pt, po = page[to], page[of]
                    for a in (self.weight, self.token):
                        a[pt, h, to % 64] = a[po, h, of % 64]
                    for which, pool in ((0, self.k), (1, self.v)):
                        ci, si = code_index(which, self.D), 16 * self.D + scale_index(which, self.D)
                        pool[pt, h, ci[to % 64]] = pool[po, h, ci[of % 64]]
                        f = pool.view(np.float32)
                        f[pt, h, si[to % 64]] = f[po, h, si[of % 64]]


def filled(rng, nkv, D, rot, lengths, spare=1, **kw):
    """A cache whose slots hold `lengths` rows, with marks."""
    per = -(-max(max(lengths), 1) // 64)
    c = Kept(rng, nkv, D, rot, len(lengths) * per + spare, len(lengths), per, **kw)
    jobs = [(s, 0, n) for s, n in enumerate(lengths) if n]
    T = sum(lengths)
    x = rng.standard_normal((2, T, nkv * D)).astype(np.float32)
    x[0] += rng.standard_normal(nkv * D).astype(np.float32)
    c.append_at(jobs, x[0], x[1], rng.integers(0, len(c.rope), (T, 1)), None)
    c.weight[~np.isnan(c.weight)] = rng.exponential(1.0, (~np.isnan(c.weight)).sum())
    return c


def axes_of(rng, rot, axes, kind):
    pairs = rot // 2
    if kind == "runs":
        return np.minimum(np.arange(pairs) * axes // pairs, axes - 1)
    return rng.integers(0, axes, pairs)


# ------------------------------------------------------------------ append ---

@pytest.mark.parametrize("nkv,D,rot,axes,kind,jobs,pad", [
    (3, 64, 64, 1, "runs", [(0, 0, 1)], 0),
    (2, 128, 128, 3, "runs", [(1, 63, 1), (0, 0, 65)], 0),
    (2, 128, 128, 3, "any", [(1, 64, 128), (0, 5, 3)], 4),
    (1, 256, 64, 3, "any", [(0, 60, 70)], 0),
    (2, 64, 16, 2, "any", [(1, 1, 63), (0, 63, 2)], 1),
    (1, 128, 10, 4, "any", [(0, 0, 64)], 3),
    (1, 256, 256, 4, "any", [(0, 100, 1), (1, 191, 1)], 0),
])
def test_append_at_bits(ctx, nkv, D, rot, axes, kind, jobs, pad):
    from chattorrent_amd.ccdecode import Positions
    rng = np.random.default_rng(D + rot + axes)
    c = Kept(rng, nkv, D, rot, 9, 2, 4)
    T, W = sum(j[2] for j in jobs), nkv * D
    x = rng.standard_normal((2, T, W + pad)).astype(np.float32)
    pos = rng.integers(0, len(c.rope), (T, axes)).astype(np.int32)
    pos[rng.random((T, axes)) < 0.05] = 2 ** 31 - 1            # beyond the table, and before it
    pos[rng.random((T, axes)) < 0.05] = -5
    of = axes_of(rng, rot, axes, kind)
    first = rng.integers(0, 10 ** 6, len(jobs)).astype(np.int32)
    cache, marks = c.device(bounds=True)
    k, v = (Strided(a, W) for a in x)
    ctx.kv_append_at(cache, jobs, k, v, Positions(dev(pos), of), marks=marks, first=first)
    c.append_at(jobs, x[0][:, :W], x[1][:, :W], pos, of, first)
    assert c.same()
    # bounds are those of 64 stored rows: a page that a job completes over rows that never were has none to compare
    whole = ~np.isnan(c.k.view(np.float32)[:, :, 16 * D:]).any((1, 2))
    assert np.array_equal(c.d[4].numpy()[whole], c.bounds[whole])


def test_append_at_without_positions_is_append(ctx):
    """Rows at their indices: kv_append's bits; the marks say so too, and without marks none are touched."""
    rng = np.random.default_rng(5)
    jobs = [(0, 30, 100), (1, 0, 64)]
    a, b = (Kept(np.random.default_rng(5), 2, 128, 64, 8, 2, 3) for _ in range(2))
    x = rng.standard_normal((2, 164, 256)).astype(np.float32)
    k, v = dev(x[0]), dev(x[1])
    (ca, _), (cb, mb) = a.device(), b.device()
    ctx.kv_append(ca, jobs, k, v)
    ctx.kv_append_at(cb, jobs, k, v)
    assert np.array_equal(b.m[0].numpy().view(np.uint32), b.weight.view(np.uint32))
    ctx.kv_append_at(cb, jobs, k, v, marks=mb)
    b.append_at(jobs, x[0], x[1])
    assert b.same() and np.array_equal(a.d[0].numpy(), b.k) and np.array_equal(a.d[1].numpy(), b.v)


def test_append_at_many_jobs_and_a_page_outside(ctx):
    """300 jobs take three launches, each with its own token numbers; a page outside the cache gets neither rows nor marks."""
    rng = np.random.default_rng(6)
    c = Kept(rng, 1, 64, 64, 300, 300, 1)
    c.table[7] = 5000
    c.table[8] = -1
    jobs = [(s, int(rng.integers(0, 60)), int(rng.integers(1, 4))) for s in rng.permutation(300)]
    T = sum(j[2] for j in jobs)
    first = np.arange(300, dtype=np.int32) * 1000
    x = rng.standard_normal((2, T, 64)).astype(np.float32)
    cache, marks = c.device()
    ctx.kv_append_at(cache, jobs, dev(x[0]), dev(x[1]), marks=marks, first=first)
    keep = [(j, int(f)) for j, f in zip(jobs, first) if j[0] not in (7, 8)]
    rows = np.concatenate([np.full(j[2], j[0] not in (7, 8)) for j in jobs])
    c.append_at([j for j, _ in keep], x[0][rows], x[1][rows], first=[f for _, f in keep])
    assert c.same()


# ------------------------------------------------------------------- weigh ---

def check_weigh(ctx, c, jobs, heads, axes=1, kind="any", observe=None, fade=1.0, seed=1, q=None, pad=0, size=1.5):
    from chattorrent_amd.ccdecode import Positions
    rng = np.random.default_rng(seed)
    T, W = sum(j[2] for j in jobs), heads * c.D
    if q is None:
        q = (size * rng.standard_normal((T, W + pad))).astype(np.float32)
    pos = rng.integers(0, len(c.rope), (T, axes)).astype(np.int32)
    of = axes_of(rng, c.rot, axes, kind)
    cache, marks = c.device()
    at = Positions(dev(pos), of)
    out = ctx.attend_weigh(cache, jobs, Strided(q, W), at, marks=marks, observe=observe, fade=fade).numpy()
    want, bound, weight, wbound = c.weigh(jobs, q[:, :W], heads, pos, of, 1 << 30 if observe is None else observe, fade)
    off = np.abs(out - want)
    assert (off <= bound[:, None]).all(), (float(off.max()), float(bound.max()))
    got = c.m[0].numpy()
    touched = wbound > 0
    off = np.abs(got - weight)
    assert (off[touched] <= wbound[touched]).all(), float((off[touched] / wbound[touched]).max())
    assert np.array_equal(got[~touched].view(np.uint32), c.weight[~touched].view(np.uint32))      # other rows' weights
    assert np.array_equal(c.m[1].numpy(), c.token)
    assert np.array_equal(c.d[0].numpy(), c.k) and np.array_equal(c.d[1].numpy(), c.v)
    # the same call again gives the same bits
    again, other = c.device(), out
    assert same_bits(ctx.attend_weigh(again[0], jobs, Strided(q, W), at, marks=again[1], observe=observe, fade=fade).numpy(), other)
    assert same_bits(c.m[0].numpy(), got)
    return out


@pytest.mark.parametrize("heads,nkv,D,rot,axes,jobs,observe,fade", [
    (9, 3, 64, 64, 1, [(0, 0, 1)], None, 1.0),                          # the chat's first token
    (9, 3, 64, 64, 3, [(0, 62, 1), (1, 63, 1), (2, 64, 1)], None, 1.0),
    (10, 2, 128, 128, 3, [(0, 300, 1), (2, 5, 1), (1, 127, 1)], None, 0.0),
    (12, 2, 256, 64, 3, [(1, 200, 1), (0, 31, 1)], None, 0.5),
    (2, 2, 128, 32, 2, [(0, 100, 16), (1, 3, 1)], 3, 1.0),              # 16 rows of one head: one piece of columns
    (4, 2, 64, 64, 2, [(0, 100, 9), (1, 60, 5)], None, 1.0),            # 18 columns, and 10
    (10, 2, 128, 128, 3, [(0, 130, 8), (1, 64, 1), (2, 0, 8)], None, 1.0),   # verify rows beside a token
    (12, 2, 256, 64, 1, [(0, 65, 8), (1, 190, 7)], 2, 0.25),
    (8, 2, 128, 128, 1, [(0, 0, 130)], None, 1.0),                      # a prompt
    (3, 3, 64, 64, 4, [(1, 77, 70), (0, 3, 1), (2, 0, 200)], 64, 0.0),  # a prompt's end is looked at
    (6, 1, 256, 256, 3, [(0, 40, 100)], 33, 1.0),
    (2, 2, 128, 128, 1, [(0, 1, 65)], 1, 0.0),                          # the last row alone
    (34, 1, 64, 64, 1, [(0, 90, 1), (1, 0, 4)], None, 1.0),             # 34 heads of a kv head
    (5, 5, 128, 128, 3, [(0, 511, 1), (1, 448, 64), (2, 0, 1)], None, 1.0),
])
def test_weigh_against_64_bits(ctx, heads, nkv, D, rot, axes, jobs, observe, fade):
    rng = np.random.default_rng(heads + D)
    lengths = [0] * (1 + max(j[0] for j in jobs))
    for s, past, n in jobs:
        lengths[s] = past + n
    c = filled(rng, nkv, D, rot, lengths)
    check_weigh(ctx, c, jobs, heads, axes, observe=observe, fade=fade)


def test_weigh_at_strides_and_without_positions(ctx):
    """q's rows padded so that no 16-byte load fits; rows at their indices; no marks, and none looked at: none touched."""
    rng = np.random.default_rng(8)
    c = filled(rng, 2, 128, 128, [200, 90])
    check_weigh(ctx, c, [(0, 150, 50), (1, 89, 1)], 6, 3, pad=3)
    jobs, q = [(0, 199, 1), (1, 60, 30)], rng.standard_normal((31, 6 * 128)).astype(np.float32)
    cache, marks = c.device()
    want, bound = c.weigh(jobs, q, 6)[:2]
    for kw in (dict(), dict(marks=marks, observe=0)):
        out = ctx.attend_weigh(cache, jobs, dev(q), **kw).numpy()
        assert (np.abs(out - want) <= bound[:, None]).all()
    assert same_bits(c.m[0].numpy(), c.weight)


@pytest.mark.parametrize("D,heads", [(64, 3), (128, 5), (256, 6)])
@pytest.mark.parametrize("n", [1, 40])
def test_weigh_over_several_splits(ctx, D, heads, n):
    """A slot of many pages is split over workgroups, for a token and for a chunk."""
    rng = np.random.default_rng(D + n)
    c = filled(rng, 1, D, D, [1500 + n, 100])
    check_weigh(ctx, c, [(0, 1500, n), (1, 99, 1)], heads, 2, size=3.0)


@pytest.mark.parametrize("n", [1, 30])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_weigh_what_rows_do_not_see(ctx, D, n):
    """Rows behind the last one and pages outside the cache hold NaN and infinity: no output has them, and their weights stay
    as they are. A row whose every page is outside gives zeros."""
    rng = np.random.default_rng(D)
    c = filled(rng, 2, D, D, [150 + n, 70, 64 + n], spare=2)
    c.table[1, 1] = 100000
    c.table[2, :] = -1
    jobs = [(0, 150, n), (1, 69, 1), (2, 64, n)]
    out = check_weigh(ctx, c, jobs, 4)
    assert not out[n + 1:].any() and np.isfinite(out).all()


@pytest.mark.parametrize("D,heads", [(64, 2), (128, 10), (256, 12)])
@pytest.mark.parametrize("n", [2, 24])
def test_weigh_values_that_are_no_numbers(ctx, D, heads, n):
    """An infinite value of the last row's makes the channels of its group NaN in the rows that see it, and in no other."""
    rng = np.random.default_rng(D)
    c = filled(rng, 2, D, D, [70 + n])
    page, t = c.table[0, (69 + n) // 64], (69 + n) % 64
    c.v.view(np.float32)[page, :, 16 * D + scale_index(1, D)[t, 1]] = np.inf
    q = rng.standard_normal((n, heads * D)).astype(np.float32)
    cache, marks = c.device()
    out = ctx.attend_weigh(cache, [(0, 70, n)], dev(q), marks=marks).numpy().reshape(n, heads, D)
    c.v.view(np.float32)[page, :, 16 * D + scale_index(1, D)[t, 1]] = 0.0
    want, bound, weight, wbound = c.weigh([(0, 70, n)], q, heads)
    bad = np.zeros((n, heads, D), bool)
    bad[-1, :, 32:64] = True
    assert np.isnan(out[bad]).all() and np.isfinite(out[~bad]).all()
    off = np.abs(out - want.reshape(out.shape))
    assert (off[:-1] <= bound[:-1, None, None]).all()
    got = c.m[0].numpy()
    assert (np.abs(got - weight)[wbound > 0] <= wbound[wbound > 0]).all()


@pytest.mark.parametrize("n", [1, 20])
def test_weigh_keys_and_queries_that_are_no_numbers(ctx, n):
    """A NaN query spoils its own row and head, and the weights that it counts in."""
    rng = np.random.default_rng(3)
    c = filled(rng, 2, 128, 128, [70 + n])
    q = rng.standard_normal((n, 4 * 128)).astype(np.float32)
    q[n - 1, 128 + 5] = np.nan                       # head 1, of kv head 0
    cache, marks = c.device()
    out = ctx.attend_weigh(cache, [(0, 70, n)], dev(q), marks=marks).numpy().reshape(n, 4, 128)
    want, bound, weight, wbound = c.weigh([(0, 70, n)], np.nan_to_num(q), 4)
    bad = np.zeros((n, 4), bool)
    bad[n - 1, 1] = True
    assert np.isnan(out[bad]).all()
    assert (np.abs(out - want.reshape(out.shape))[~bad] <= np.broadcast_to(bound[:, None, None], out.shape)[~bad]).all()
    got = c.m[0].numpy()[c.table[0]]
    seen = np.arange(128) < 70 + n
    assert np.isnan(got[:, 0].reshape(-1)[seen]).all() and not np.isnan(got[:, 1].reshape(-1)[seen]).any()


@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("size", [1e-30, 1e-4, 300.0, 1e6, 1e12])
def test_weigh_scores_of_any_magnitude(ctx, n, size):
    """From scores that are all alike to ones where a single row takes everything."""
    rng = np.random.default_rng(int(math.log10(size)) + 50)
    c = filled(rng, 2, 128, 128, [130 + n])
    q = (size * rng.standard_normal((n, 4 * 128))).astype(np.float32)
    cache, marks = c.device()
    out = ctx.attend_weigh(cache, [(0, 130, n)], dev(q), marks=marks, fade=0.0).numpy()
    want, bound, weight, wbound = c.weigh([(0, 130, n)], q, 4, fade=0.0)
    got = c.m[0].numpy()[c.table[0]].reshape(-1, 2, 64)
    seen = np.arange(got.shape[0] * 64) < 130 + n
    total = got.transpose(1, 0, 2).reshape(2, -1)[:, seen].sum(1)
    assert np.isfinite(out).all()
    # 1e6 and more: f32 no longer says which of two scores is the larger, and many rows' are formed anew for the sums
    assert (total <= 2 * n * (1 + 1e-4)).all() and ((total >= 2 * n * (1 - 1e-4)).all() or (n > 1 and size > 300))
    if size <= 300:
        assert (np.abs(out - want) <= bound[:, None]).all()
        off = np.abs(c.m[0].numpy() - weight)
        assert (off[wbound > 0] <= wbound[wbound > 0]).all(), [a[off > wbound] for a in (off, wbound, weight)]


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("n", [1, 24])
def test_weigh_rows_whose_groups_differ_in_size(ctx, which, n):
    """Keys (which = 0) or values from 2^-40 to 2^40 times the others, by row and group: an output is off by no more than its
    group's largest value allows."""
    rng = np.random.default_rng(9)
    c = filled(rng, 1, 128, 128, [200 + n])
    pool = (c.k, c.v)[which]
    pages = c.table[0, :-(-(200 + n) // 64)]
    for g in range(4):
        f = 2.0 ** rng.integers(-40, 41 if which else 3, 64)
        pool.view(np.float32)[pages[:, None], 0, 16 * 128 + scale_index(which, 128)[:, g]] *= f.astype(np.float32)
    jobs, q = [(0, 200, n)], (0.5 * rng.standard_normal((n, 3 * 128))).astype(np.float32)
    cache, marks = c.device()
    out = ctx.attend_weigh(cache, jobs, dev(q), marks=marks).numpy()
    want, bound, weight, wbound = c.weigh(jobs, q, 3)
    T = 200 + n
    vv = np.concatenate([c.exact_rows(1, p, 0) for p in pages])[:T]
    of = np.abs(vv).reshape(T, 4, 32).max((0, 2)) / np.abs(vv).max()           # a group's part of the largest value
    lim = bound[:, None, None] * np.tile(np.repeat(of, 32), 3).reshape(1, 3, 128)
    assert (np.abs(out - want).reshape(n, 3, 128) <= lim).all()
    assert (np.abs(c.m[0].numpy() - weight)[wbound > 0] <= wbound[wbound > 0]).all()


def test_weigh_more_jobs_and_rows_than_a_launch_takes(ctx):
    """70 jobs of either kind; then one of more rows than a piece, whose weights fade once and whose last rows count."""
    rng = np.random.default_rng(12)
    lengths = [int(n) for n in rng.integers(1, 120, 140)]
    c = filled(rng, 1, 64, 64, lengths)
    jobs = [(s, 0, n) if s % 2 and n > 8 else (s, n - 1, 1) for s, n in enumerate(lengths)]
    check_weigh(ctx, c, jobs, 2, observe=5, fade=0.5)
    c = filled(rng, 1, 64, 64, [4230], rope_rows=5000)
    check_weigh(ctx, c, [(0, 10, 4220)], 1, observe=4000, fade=0.5, size=0.5)
    check_weigh(ctx, c, [(0, 10, 4220)], 1, observe=30, fade=0.5, size=0.5)


# ------------------------------------------------------------------- evict ---

def check_evict(ctx, c, jobs, sink=0, recent=0):
    cache, marks = c.device()
    ctx.kv_evict(cache, marks, jobs, sink=sink, recent=recent)
    c.evict(jobs, sink, recent)
    assert c.same()


@pytest.mark.parametrize("nkv,D,jobs,sink,recent", [
    (3, 64, [(0, 2, 1, 2)], 0, 0),
    (2, 128, [(0, 65, 64, 65), (1, 130, 64, 130), (2, 40, 64, 40)], 0, 0),     # one row; a page's worth; none
    (2, 128, [(0, 200, 64, 200), (1, 130, 100, 130)], 4, 30),
    (1, 256, [(0, 300, 70, 300)], 0, 64),
    (2, 64, [(0, 500, 1, 500), (1, 500, 499, 500)], 1, 0),
    (1, 64, [(0, 777, 388, 777)], 300, 300),                                   # more of them are safe than stay
    (2, 128, [(0, 1200, 700, 1200)], 3, 10),
])
def test_evict_bits(ctx, nkv, D, jobs, sink, recent):
    rng = np.random.default_rng(D + len(jobs) + sink)
    c = filled(rng, nkv, D, D, [j[1] for j in jobs])
    check_evict(ctx, c, jobs, sink, recent)


@pytest.mark.parametrize("rows", [4096, 4097, 8193, 16384, 16500])
def test_evict_sizes_around_the_variants(ctx, rows):
    rng = np.random.default_rng(rows)
    per = -(-rows // 64)
    c = Kept(rng, 1, 64, 64, per, 1, per)
    for a in (c.k, c.v):
        a[:] = rng.integers(0, 255, a.shape)
    c.weight[:] = rng.exponential(1.0, c.weight.shape)
    order = rng.permutation(3 * rows)[:per * 64].reshape(per, 64)
    c.token[c.table[0], 0] = order
    check_evict(ctx, c, [(0, rows, rows - 37, 3 * rows)], 2, 50)
    check_evict(ctx, c, [(0, rows - 37, rows // 3, 3 * rows)], 2, 50)


def test_evict_equal_weights_and_ones_that_are_no_numbers(ctx):
    """Ties go to the lower row, -0 is 0, infinities are weights like others, NaN counts least; a page outside the cache is
    neither read nor written, and counts least of all."""
    rng = np.random.default_rng(4)
    kinds = np.array([0.0, -0.0, 1.0, 1.0, np.inf, -np.inf, np.nan, 1e-45, 3e38, -2.0], np.float32)
    for keep in (1, 100, 130, 190, 319):
        c = filled(rng, 2, 64, 64, [320])
        c.weight[:] = rng.choice(kinds, c.weight.shape)
        check_evict(ctx, c, [(0, 320, keep, 320)], 1, 2)
    c = filled(rng, 2, 64, 64, [320], spare=1)
    c.weight[:] = rng.choice(kinds, c.weight.shape)
    c.table[0, 1] = 77
    c.table[0, 4] = -1
    check_evict(ctx, c, [(0, 320, 100, 320)], 1, 2)


def test_evict_many_jobs_beside_each_other(ctx):
    """More jobs than a launch takes, few and many moves among them; the other slots' pages stay as they are."""
    rng = np.random.default_rng(14)
    lengths = [int(n) for n in rng.integers(1, 400, 110)]
    c = filled(rng, 1, 64, 64, lengths)
    jobs = [(s, n, int(rng.integers(1, n + 1)), n + int(rng.integers(0, 100))) for s, n in enumerate(lengths) if s % 9]
    check_evict(ctx, c, jobs, 2, 5)


# ---------------------------------------------------------------- together ---

def step(ctx, cache, marks, jobs, first, keeps, k, v, q, at, stream=None, sink=1, recent=8):
    ctx.kv_append_at(cache, jobs, k, v, at, marks=marks, first=first, stream=stream)
    out = ctx.attend_weigh(cache, jobs, q, at, marks=marks, fade=0.9, stream=stream)
    ctx.kv_evict(cache, marks, keeps, sink=sink, recent=recent, stream=stream)
    return out


def test_chats_within_a_bound(ctx):
    """Chats whose caches are cut to 100 rows whenever they pass 128: prompts with an image, then tokens, against the plain
    operators on the same cache. Which rows go hangs on weights that are sums of f32: the device's own weights decide on both
    sides, within their bound of the plain ones."""
    rng = np.random.default_rng(21)
    from chattorrent_amd.ccdecode import Positions
    nkv, D, heads, rot = 2, 128, 6, 64
    c = Kept(rng, nkv, D, rot, 12, 3, 4)
    cache, marks = c.device()
    of = np.arange(rot // 2) % 3
    rows, seen, at_pos = [0, 0, 0], [0, 0, 0], [0, 0, 0]
    for turn in range(12):
        n = [int(rng.integers(30, 100)) for _ in range(3)] if turn == 0 else [1 + (turn + s) % 5 * 7 for s in range(3)]
        jobs = [(s, rows[s], n[s]) for s in range(3)]
        T = sum(n)
        pos = np.concatenate([np.stack([np.full(m, p), p + np.arange(m) // 8, p + np.arange(m) % 8], 1) if turn == 0 else
                              np.tile(p + np.arange(m)[:, None], (1, 3)) for p, m in zip(at_pos, n)]).astype(np.int32)
        x = rng.standard_normal((2, T, nkv * D)).astype(np.float32)
        q = rng.standard_normal((T, heads * D)).astype(np.float32)
        at, first = Positions(dev(pos), of), np.array(seen, np.int32)
        rows = [r + m for r, m in zip(rows, n)]
        seen = [r + m for r, m in zip(seen, n)]
        at_pos = [int(pos[i - 1].max()) + 1 for i in np.cumsum(n)]
        keeps = [(s, rows[s], 100, seen[s]) for s in range(3) if rows[s] > 128]
        k, v = dev(x[0]), dev(x[1])
        ctx.kv_append_at(cache, jobs, k, v, at, marks=marks, first=first)
        c.append_at(jobs, x[0], x[1], pos, of, first)
        out = ctx.attend_weigh(cache, jobs, dev(q), at, marks=marks, fade=0.9).numpy()
        want, bound, weight, wbound = c.weigh(jobs, q, heads, pos, of, fade=0.9)
        assert (np.abs(out - want) <= bound[:, None]).all()
        got = c.m[0].numpy()
        assert (np.abs(got - weight)[wbound > 0] <= wbound[wbound > 0]).all()
        c.weight[:] = got
        if keeps:
            ctx.kv_evict(cache, marks, keeps, sink=1, recent=8)
            c.evict(keeps, 1, 8)
            for s, *_ in keeps:
                rows[s] = 100
        assert c.same()
        for s in range(3):      # what is promised to stay is there, once
            r = np.arange(rows[s])
            for h in range(nkv):
                tok = c.token[c.table[s, r // 64], h, r % 64]
                assert len(set(tok.tolist())) == rows[s] and {0, *range(max(0, seen[s] - 8), seen[s])} <= set(tok.tolist())


def two_chats(ctx, seed):
    """A step's device inputs and the cache before it, as a function that puts them back."""
    from chattorrent_amd.ccdecode import Positions
    rng = np.random.default_rng(seed)
    c = filled(rng, 2, 128, 128, [150, 90], spare=0)
    c.table = np.concatenate([c.table, np.zeros_like(c.table)], 1)[:, :4]
    jobs = [(0, 149, 1), (1, 60, 30)]
    keeps = [(0, 150, 100, 400), (1, 90, 64, 90)]
    x = rng.standard_normal((2, 31, 256)).astype(np.float32)
    q = rng.standard_normal((31, 6 * 128)).astype(np.float32)
    pos = rng.integers(0, 600, (31, 3)).astype(np.int32)
    cache, marks = c.device()
    args = (cache, marks, jobs, [399, 60], keeps, dev(x[0]), dev(x[1]), dev(q), Positions(dev(pos), np.arange(64) % 3))

    def reset():
        for d, a in zip((*c.d[:2], *c.m), (c.k, c.v, c.weight, c.token)):
            d.set(a)

    def state():
        return [d.numpy().view(np.uint8).copy() for d in (*c.d[:2], *c.m)]
    return args, reset, state


def test_a_captured_step_of_the_bound_replays(ctx, hip):
    """Append, weigh and evict in one graph, replayed with the eager step in between: every replay gives its bits."""
    import ctypes as C
    import ctypes as C
    from chattorrent_amd.ccdecode import DeviceArray
    args, reset, state = two_chats(ctx, 31)
    want = step(ctx, *args).numpy()
    after = state()
    cache, marks, jobs, first, keeps, k, v, q, at = args
    L, h = ctx.lib, ctx.h
    ja, ka, fa = np.array(jobs, np.int32), np.array(keeps, np.int32), np.array(first, np.int32)
    out = DeviceArray(want.shape, np.float32)
    nw = L.cc_weigh_workspace(h, cache.ref, ja.ctypes.data, 2, 6, 1000)
    ne = L.cc_evict_workspace(cache.ref, ka.ctypes.data, 2)
    ws, we = DeviceArray(nw, np.uint8), DeviceArray(max(ne, 16), np.uint8)
    st, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    hip.check(hip.h.hipStreamCreate(C.byref(st)))
    hip.check(hip.h.hipStreamBeginCapture(st, 2))
    code = [L.cc_kv_append_at(h, cache.ref, at.ref, marks.ref, ja.ctypes.data, 2, fa.ctypes.data, k.data_ptr(), 256,
                              v.data_ptr(), 256, st),
            L.cc_attend_weigh(h, cache.ref, at.ref, marks.ref, ja.ctypes.data, 2, 6, 1000, C.c_float(0.9), q.data_ptr(), 768,
                              out.data_ptr(), 768, ws.data_ptr(), nw, st),
            L.cc_kv_evict(h, cache.ref, marks.ref, ka.ctypes.data, 2, 1, 8, we.data_ptr(), ne, st)]
    hip.check(hip.h.hipStreamEndCapture(st, C.byref(graph)))
    assert code == [0] * 3, L.cc_last_error(h)
    hip.check(hip.h.hipGraphInstantiate(C.byref(exe), graph, None, None, 0))
    for i in range(4):
        reset()
        ws.set(np.random.default_rng(i).integers(0, 255, nw).astype(np.uint8))     # a workspace of any contents
        hip.check(hip.h.hipGraphLaunch(exe, st))
        hip.check(hip.h.hipStreamSynchronize(st))
        assert same_bits(out.numpy(), want)
        assert all(np.array_equal(a, b) for a, b in zip(state(), after))
        reset()
        assert same_bits(step(ctx, *args).numpy(), want)
        assert all(np.array_equal(a, b) for a, b in zip(state(), after))
    hip.h.hipGraphExecDestroy(exe)
    hip.h.hipGraphDestroy(graph)
    hip.check(hip.h.hipStreamDestroy(st))


def test_two_streams_at_once(ctx, hip):
    """Two caches' steps on two streams that overlap give what each gives alone."""
    import ctypes as C
    both = two_chats(ctx, 41), two_chats(ctx, 42)
    want = []
    for args, reset, state in both:
        out = step(ctx, *args).numpy()
        want.append((out, state()))
        reset()
    st = [C.c_void_p() for _ in range(2)]
    for s in st:
        hip.check(hip.h.hipStreamCreate(C.byref(s)))
    for _ in range(3):
        outs = [step(ctx, *args, stream=s.value) for (args, _, _), s in zip(both, st)]
        for s in st:
            hip.check(hip.h.hipStreamSynchronize(s))
        for out, (args, reset, state), (o, after) in zip(outs, both, want):
            assert same_bits(out.numpy(), o) and all(np.array_equal(x, y) for x, y in zip(state(), after))
            reset()
    for s in st:
        hip.check(hip.h.hipStreamDestroy(s))


def test_rows_past_4_gib(ctx):
    """Blocks whose bytes lie past 2^31 and 2^32 of the pools: appended to, read, weighed and moved as a small cache's."""
    from chattorrent_amd.ccdecode import DeviceArray, KVCache, Marks
    rng = np.random.default_rng(17)
    nkv, D, n = 8, 256, 30000
    small = Kept(rng, nkv, D, D, 6, 1, 6)
    small.table[0] = np.arange(6)
    near, near_marks = small.device()
    pools = [DeviceArray((n, nkv, small.k.shape[2]), np.uint8) for _ in range(2)]
    marks = [DeviceArray((n, nkv, 64), t) for t in (np.float32, np.int32)]
    far = KVCache(*pools, dev(np.array([[29999, 3, 14800, 29400, 14650, 29250]], np.int32)), small.d[3], D)
    k, v = (dev(rng.standard_normal((380, nkv * D)).astype(np.float32)) for _ in range(2))
    q = [dev(rng.standard_normal((m, 2 * nkv * D)).astype(np.float32)) for m in (1, 30)]
    got = []
    for cache, m in ((near, near_marks), (far, Marks(*marks))):
        ctx.kv_append_at(cache, [(0, 0, 380)], k, v, marks=m)
        outs = [ctx.attend_weigh(cache, [(0, 380 - len_, len_)], x, marks=m).numpy() for x, len_ in zip(q, (1, 30))]
        ctx.kv_evict(cache, m, [(0, 380, 200, 380)], sink=1, recent=4)
        got.append(outs + [ctx.attend_weigh(cache, [(0, 199, 1)], q[0], marks=m).numpy()])
    assert all(same_bits(a, b) for a, b in zip(*got))


# ------------------------------------------------------ what nothing above asks ---

@pytest.mark.parametrize("heads,nkv,D,rot,axes,jobs,observe,fade", [
    (8, 1, 64, 2, 1, [(0, 127, 2), (1, 0, 2)], None, 1.0),              # 16 columns
    (17, 1, 64, 6, 4, [(0, 128, 1), (1, 200, 1)], None, 1.0),           # 17
    (8, 1, 128, 10, 2, [(0, 57, 8), (1, 121, 6)], 5, 0.5),              # 64, and 48: up to 64 columns, some that do not count
    (13, 1, 128, 128, 1, [(0, 190, 5)], 1, 1.0),                        # 65
    (64, 1, 64, 64, 2, [(0, 66, 1), (1, 190, 1)], None, 0.0),
    (1, 1, 256, 14, 3, [(0, 0, 64), (1, 63, 65)], 17, 1.0),             # as many rows of one head
    (130, 1, 64, 64, 1, [(0, 90, 5)], 3, 0.25),                         # tiles that end inside a row's heads
    (7, 1, 256, 2, 4, [(0, 61, 75)], 50, 0.0),
    (4, 4, 64, 64, 1, [(0, 3, 300)], 299, 0.5),                         # all but one row count
])
def test_weigh_at_the_borders_of_the_variants(ctx, heads, nkv, D, rot, axes, jobs, observe, fade):
    rng = np.random.default_rng(heads + D + rot)
    lengths = [0] * (1 + max(j[0] for j in jobs))
    for s, past, n in jobs:
        lengths[s] = past + n
    check_weigh(ctx, filled(rng, nkv, D, rot, lengths), jobs, heads, axes, observe=observe, fade=fade)


@pytest.mark.parametrize("D,heads,n", [(64, 2, 300), (128, 1, 300), (256, 2, 100)])
def test_weigh_many_tiles_over_several_splits(ctx, D, heads, n):
    """Tiles of a chunk that end before the slot's last pages, beside a shorter chunk."""
    rng = np.random.default_rng(D + n)
    c = filled(rng, 1, D, D, [2000 + n, 170], rope_rows=2500)
    check_weigh(ctx, c, [(0, 2000, n), (1, 40, 130)], heads, 1, observe=n // 2, size=2.0)


def test_weigh_more_splits_than_one_batch_of_loads(ctx):
    """196 pages: 33 splits for a token, 98 for 40 columns."""
    rng = np.random.default_rng(4)
    c = filled(rng, 1, 64, 64, [12500], rope_rows=700)
    check_weigh(ctx, c, [(0, 12499, 1)], 2, size=0.5)
    check_weigh(ctx, c, [(0, 12480, 20)], 2, size=0.5, observe=3, fade=0.5)


def test_weigh_slots_whose_pages_are_in_any_order(ctx):
    """Pages in falling order, between others' and with a slot that is not asked."""
    rng = np.random.default_rng(3)
    c = filled(rng, 2, 128, 128, [300, 310, 290], spare=4)
    moved = rng.permutation(len(c.k))
    for a in (c.k, c.v, c.weight, c.token):
        a[:] = a[np.argsort(moved)]
    c.table = moved[c.table].astype(c.table.dtype)[:, :]
    check_weigh(ctx, c, [(2, 250, 40), (0, 299, 1)], 6, 3)


def test_a_contexts_own_cache_kept(ctx):
    """The cache that the pass fills, with marks beside it: weighed as attend_pages reads it, and given up by weight."""
    from chattorrent_amd.ccdecode import Context, DeviceArray, KVCache, Marks
    d = configs.with_layers(configs.SMOLLM2, 1)
    c = Context(d, n_max=1024, t_max=8, slots=1)
    try:
        c.fill_random_kv(0, 900, 3, 1)
        rng = np.random.default_rng(9)
        q = rng.standard_normal((4, d["n_heads"] * d["head_dim"])).astype(np.float32)
        want = c.op_attend(0, 0, q, 890)
        cache = KVCache.of_context(c, 0)
        shape = cache.c.n_pages, cache.c.n_kv_heads, 64
        marks = Marks(dev(np.full(shape, 7, np.float32)), dev(np.tile(np.arange(64, dtype=np.int32), shape[:2] + (1,))))
        got = c.attend_weigh(cache, [(0, 890, 4)], dev(q), marks=marks, fade=0.0).numpy()
        assert np.abs(got - want).max() <= 2e-5 * np.abs(want).max() * 2
        weight = marks.kept[0].numpy()
        rows = weight != 7
        assert rows.sum() == 894 * shape[1]
        each = np.where(rows, weight, 0).sum((0, 2))       # the four rows' probabilities, of each head of a group
        assert np.abs(each - 4 * d["n_heads"] / shape[1]).max() <= 4 * 9 * 2.0 ** -14
        c.kv_evict(cache, marks, [(0, 894, 500, 894)])
        few = c.attend_weigh(cache, [(0, 499, 1)], dev(q[3:])).numpy()
        assert np.isfinite(few).all()
        table, left = np.asarray(c.pages(0))[:15], marks.kept[0].numpy()
        for h in range(shape[1]):
            before, after = (a[table, h].reshape(-1) for a in (weight, left))
            assert np.array_equal(np.sort(after[:500]), np.sort(before[:894])[-500:])
    finally:
        c.close()


TORCH_KEPT = """
import numpy as np, torch
from chattorrent_amd import ccdecode as cc, configs
ctx = cc.Context(configs.with_layers(configs.SMOLLM2, 1), n_max=256, t_max=8, slots=2)
nkv, D, heads, pages = 2, 128, 6, 6
def fresh():
    blk = 64 * D + 64 * (D // 32) * 4
    pools = [torch.full((pages, nkv, blk), 128, dtype=torch.uint8, device="cuda") for _ in range(2)]
    table = torch.arange(pages, dtype=torch.int32, device="cuda").reshape(2, 3)
    ang = torch.arange(192, device="cuda")[:, None] * torch.logspace(0, -4, D // 2, device="cuda")
    rope = torch.stack([ang.cos(), ang.sin()], -1).contiguous()
    marks = cc.Marks(torch.zeros(pages, nkv, 64, device="cuda"), torch.zeros(pages, nkv, 64, dtype=torch.int32, device="cuda"))
    return cc.KVCache(*pools, table, rope, D), marks
torch.manual_seed(1)
jobs, n = [(0, 0, 150), (1, 0, 70)], 220
k, v = (torch.randn(n, nkv * D + 8, device="cuda")[:, :nkv * D] for _ in range(2))
q = torch.randn(n, heads * D, device="cuda")
at = cc.Positions(torch.randint(0, 192, (n, 3), dtype=torch.int32, device="cuda"), np.arange(D // 2) % 3)
def run(stream):
    cache, marks = fresh()
    torch.cuda.synchronize()
    ctx.kv_append_at(cache, jobs, k, v, at, marks=marks, stream=stream)
    out = ctx.attend_weigh(cache, jobs, q, at, marks=marks, stream=stream)
    ctx.kv_evict(cache, marks, [(0, 150, 64, 150)], sink=1, recent=4, stream=stream)
    torch.cuda.synchronize()
    return [out.clone(), *(t.clone() for t in marks.kept)]
want = run(None)
side = torch.cuda.Stream()
with torch.cuda.stream(side):
    within = run(None)
for got in (within, run(side.cuda_stream), run(0)):
    assert all(torch.equal(a, b) for a, b in zip(want, got))
assert torch.isfinite(want[0]).all() and abs(float(want[1][3:].sum()) - 70 * heads) < 0.1
print("held")
"""


def test_torch_tensors_on_torchs_streams(gpu):
    r = subprocess.run([sys.executable, "-c", TORCH_KEPT], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True,
                       timeout=110)
    assert r.returncode == 0 and r.stdout.strip().endswith("held"), r.stdout


def test_two_graphs_with_workspaces_of_their_own(ctx, hip):
    """Two captured steps, each with its own workspaces, replayed at the same time: each gives the eager step's bits."""
    import ctypes as C
    from chattorrent_amd.ccdecode import DeviceArray
    L, h, held = ctx.lib, ctx.h, []
    for seed in (51, 52):
        args, reset, state = two_chats(ctx, seed)
        want = step(ctx, *args).numpy()
        after = state()
        cache, marks, jobs, first, keeps, k, v, q, at = args
        ja, ka, fa = np.array(jobs, np.int32), np.array(keeps, np.int32), np.array(first, np.int32)
        out = DeviceArray(want.shape, np.float32)
        nw, ne = L.cc_weigh_workspace(h, cache.ref, ja.ctypes.data, 2, 6, 1000), L.cc_evict_workspace(cache.ref, ka.ctypes.data, 2)
        ws, we = DeviceArray(nw, np.uint8), DeviceArray(max(ne, 16), np.uint8)
        st, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
        hip.check(hip.h.hipStreamCreate(C.byref(st)))
        hip.check(hip.h.hipStreamBeginCapture(st, 2))
        code = [L.cc_kv_append_at(h, cache.ref, at.ref, marks.ref, ja.ctypes.data, 2, fa.ctypes.data, k.data_ptr(), 256,
                                  v.data_ptr(), 256, st),
                L.cc_attend_weigh(h, cache.ref, at.ref, marks.ref, ja.ctypes.data, 2, 6, 1000, C.c_float(0.9), q.data_ptr(), 768,
                                  out.data_ptr(), 768, ws.data_ptr(), nw, st),
                L.cc_kv_evict(h, cache.ref, marks.ref, ka.ctypes.data, 2, 1, 8, we.data_ptr(), ne, st)]
        hip.check(hip.h.hipStreamEndCapture(st, C.byref(graph)))
        assert code == [0] * 3, L.cc_last_error(h)
        hip.check(hip.h.hipGraphInstantiate(C.byref(exe), graph, None, None, 0))
        held.append((st, graph, exe, args, reset, state, out, want, after, (ws, we)))
    for _ in range(3):
        for g in held:
            g[4]()
        for g in held:
            hip.check(hip.h.hipGraphLaunch(g[2], g[0]))
        for g in held:
            hip.check(hip.h.hipStreamSynchronize(g[0]))
        for st, graph, exe, args, reset, state, out, want, after, _ in held:
            assert same_bits(out.numpy(), want) and all(np.array_equal(a, b) for a, b in zip(state(), after))
    for st, graph, exe, *_ in held:
        hip.h.hipGraphExecDestroy(exe)
        hip.h.hipGraphDestroy(graph)
        hip.check(hip.h.hipStreamDestroy(st))

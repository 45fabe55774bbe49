"""cc_sample_pass: the tokens of a pass's own logits, drawn where they are,
against the same logits read back and drawn in numpy in 64 bits, and against
cc_sample over a copy of them."""
import base64
import json
import os
import subprocess

import numpy as np
import pytest

from chattorrent_amd import configs
from tests.test_gpu_operators import Ask, U32, dev

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
V = configs.SMOLLM2["vocab"]


@pytest.fixture(scope="module")
def ctx(gpu):
    from chattorrent_amd.ccdecode import Context
    c = Context(configs.with_layers(configs.SMOLLM2, 2), n_max=256, t_max=40, slots=8)
    c.fill_random(5)
    yield c
    c.close()


def feed(ctx, rng, sizes, sampled):
    """A pass of new chats; its logits as they read back."""
    for s in range(len(sizes)):
        ctx.release(s)
    ctx.step([dict(slot=s, past=0, n=n, sampled=k, ids=rng.integers(0, V, n).astype(np.uint32))
              for s, (n, k) in enumerate(zip(sizes, sampled))])
    return ctx.read_logits(sum(sampled))


@pytest.mark.parametrize("sizes,sampled", [([1], [1]), ([3, 1, 5], [1, 1, 5]), ([5] * 8, [5] * 8)])
@pytest.mark.parametrize("kw", [
    dict(), dict(temp=0.8), dict(temp=1.1, top_k=30, top_p=0.9, min_p=0.01),
    dict(temp=0.9, top_p=0.8, history=100, counts=True, rep=1.2, freq=0.3, pres=0.2, biases=30, masks=2)],
    ids=["greedy", "plain", "cuts", "lists"])
def test_tokens_of_a_pass(ctx, sizes, sampled, kw):
    rng = np.random.default_rng(len(sizes) + len(kw))
    rows = sum(sampled)
    x = feed(ctx, rng, sizes, sampled)
    ask = Ask(rng, rows, V, u=rng.random(rows), **kw)
    ids, probs = ctx.sample_pass(rows, freq_cap=ask.cap, **ask.a)
    other = [a.numpy() for a in ctx.sample(dev(x), ask.device())]
    assert np.array_equal(ids, other[0]) and np.array_equal(probs, other[1])
    for r, (t, p, near) in enumerate(ask.sample(x)):
        if near > 1e-9:     # as cc_sample's own test derives
            assert ids[r] == t and abs(probs[r] - p) <= (U32 + 1e-9) * p * 1.01, (r, ids[r], t)
    # a second draw of the same rows, and the rows themselves, stay as they were
    again = ctx.sample_pass(rows, freq_cap=ask.cap, **ask.a)
    assert np.array_equal(again[0], ids) and np.array_equal(again[1], probs)
    assert np.array_equal(ctx.read_logits(rows).view(np.uint32), x.view(np.uint32))


def test_a_chat_of_drawn_tokens(ctx):
    """Each drawn token fed on, without the rows leaving the device; the same chat with the rows read back."""
    def chat(draw):
        rng = np.random.default_rng(9)
        feed(ctx, rng, [4], [1])
        out = []
        for i in range(12):
            out.append(int(draw(rng.random())))
            ctx.step([dict(slot=0, past=4 + i, n=1, sampled=1, ids=np.array([out[-1]], np.uint32))])
        return out

    def back(u):
        return ctx.sample(dev(ctx.read_logits(1)), Ask(None, 1, V, temp=0.9, top_k=50, u=u).device())[0].numpy()[0]
    assert chat(lambda u: ctx.sample_pass(1, temp=[0.9], top_k=[50], u=[u])[0][0]) == chat(back)


def test_refusals(ctx):
    from chattorrent_amd.ccdecode import CCError, Context
    feed(ctx, np.random.default_rng(1), [2, 2], [1, 1])
    for rows, kw, text in ((1, {}, "last pass"), (3, {}, "last pass"), (2, dict(temp=[1, 1]), "random numbers"),
                           (2, dict(rep=[1.1, 1.1]), "history"), (2, dict(mask=np.zeros((1, 1 + V // 32))), "mask_of"),
                           (2, dict(freq_cap=-1.0), "freq_cap")):
        with pytest.raises(CCError, match=text):
            ctx.sample_pass(rows, **kw)
    with pytest.raises(ValueError, match="temp"):
        ctx.sample_pass(2, temp=[1.0])
    fresh = Context(configs.with_layers(configs.SMOLLM2, 1), n_max=64, t_max=2, slots=1)
    with pytest.raises(CCError, match="last pass"):
        fresh.sample_pass(1)
    fresh.close()
    assert (ctx.sample_pass(2)[0] >= 0).all()


HOST_DRAWS = """
const { sampleFromLogitsRow } = require(process.argv[1]);
const jobs = JSON.parse(require('fs').readFileSync(0, 'utf8'));
console.log(JSON.stringify(jobs.map(j => {
    const b = Buffer.from(j.row, 'base64');
    const row = new Float32Array(b.buffer.slice(b.byteOffset, b.byteOffset + b.length));
    return j.draws.map(d => sampleFromLogitsRow(row, d.opts, () => d.u));
})));
"""


def test_the_hosts_sampler_draws_the_same_tokens(ctx):
    """The same options through node/sampling.js over the rows read back and through cc_sample_pass: greedy, temperatures, top-k,
    penalties of distinct ids with counts of 1 and more, bans (all parameters whole in f32). Where u is not within 2^-20 of a border: there the host's walk,
    which adds weights rounded to f32 (2^-24 each, so 2^-24 of the sum behind a border and as much of the total), may differ."""
    rng = np.random.default_rng(12)
    rows = 8
    x = feed(ctx, rng, [2] * rows, [1] * rows)
    opts, u = [], []
    for i in range(12):
        for r in range(rows):
            o = dict(temp=[0, 0.75, 1.0, 1.875][i % 4], topK=[0, 40, 200][i % 3])
            if i % 2:
                top = np.argsort(-x[r])[:20]
                ids = np.unique(np.concatenate([rng.integers(0, V, 30), rng.choice(top, 10, replace=False)]))
                o.update(pen=[[int(t), int(rng.integers(1, 9))] for t in ids], rep=1.25, freq=0.5, pres=0.25)
                o["ban"] = [int(t) for t in rng.choice(top, 3, replace=False)]
            opts.append(o)
            u.append(float(rng.random()))
    jobs = [dict(row=base64.b64encode(x[r].tobytes()).decode(), draws=[dict(opts=opts[i * rows + r], u=u[i * rows + r]) for i in range(12)])
            for r in range(rows)]
    told = subprocess.run(["node", "-e", HOST_DRAWS, os.path.join(ROOT, "chattorrent_amd", "node", "sampling.js")],
                          input=json.dumps(jobs), capture_output=True, text=True, timeout=100)
    assert told.returncode == 0, told.stderr
    host, compared = json.loads(told.stdout), 0
    for i in range(12):
        mine = opts[i * rows:(i + 1) * rows]
        kw = dict(temp=[o["temp"] for o in mine], top_k=[o["topK"] for o in mine], u=u[i * rows:(i + 1) * rows])
        ask = Ask(rng, rows, V, **kw)
        if i % 2:
            flat = [e for o in mine for e in o["pen"]]
            ask.a.update(rep=np.full(rows, 1.25, np.float32), freq=np.full(rows, 0.5, np.float32), pres=np.full(rows, 0.25, np.float32),
                         pen_at=np.cumsum([0] + [len(o["pen"]) for o in mine]).astype(np.int32),
                         pen_ids=np.array([e[0] for e in flat], np.int32), pen_counts=np.array([e[1] for e in flat], np.int32),
                         bias_at=np.arange(0, 3 * rows + 1, 3, dtype=np.int32), bias=np.full(3 * rows, -np.inf, np.float32),
                         bias_ids=np.array([t for o in mine for t in o["ban"]], np.int32))
        ids, _ = ctx.sample_pass(rows, freq_cap=ask.cap, **ask.a)
        for r, (t, p, near) in enumerate(ask.sample(x)):
            if near > 2.0 ** -20:
                compared += 1
                assert ids[r] == host[r][i], (i, r, ids[r], host[r][i], t)
    assert compared >= 80

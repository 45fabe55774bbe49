"""The operators of one decode step of long chats whose speed is measured: from the paged int8 cache to the token.

  append   cc_kv_append: new keys (rotated to their positions) and values into a paged int8 cache, for a ragged batch of
           jobs, and the key bounds of every page that the rows complete
  attend   cc_attend_pages: attention of a job's rows over the pages of the cache that a cheap score, from the key bounds
           in 8 bits, selects for each row and kv head
  adjust   cc_logits_adjust: penalties for repeated tokens, biases and grammar masks on rows of logits
  sample   cc_sample: the same, then temperature, top-k, top-p and min-p, and the draw of a token with a given random number

Each is reached through `chattorrent_amd.ccdecode` where `own` is set; otherwise it is computed in elementary operations.
A cache is held as the library lays it out: a block for each (page of 64 tokens, kv head) with its codes (biased by 128) and
then one f32 scale for each token and 32 channels, `code_index` and `scale_index` saying where. Model shapes (heads, widths,
vocabularies) are those of `chattorrent_amd.configs`.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64
FREQ_CAP = 1.5     # the most that one token's frequency penalty takes, as node/sampling.js has it


# -------------------------------------------------------------------- cases ---

def append_case(name, **kw):
    return dict(dict(name=name, op="append", kv_heads=8, head_dim=128, rot_dim=128, chats=0, ctx_lo=128, ctx_hi=16384,
                     chunks=0, chunk_rows=0, chunk_past=0, ctx_seed=1234), **kw)


def attend_case(name, **kw):
    return dict(dict(name=name, op="attend", heads=40, kv_heads=8, head_dim=128, rot_dim=128, chats=1, rows=1, ctx_lo=4096,
                     ctx_hi=32768, budget=64, sink=1, recent=2, ctx_seed=1234), **kw)


def logits_case(name, op, **kw):
    return dict(dict(name=name, op=op, rows=1, vocab=151936, pad=0, history=0, biases=0, grammars=0, temp=0.0, top_k=0,
                     top_p=1.0, min_p=0.0, spread=2.5), **kw)


def listed():
    return [
        # one person chatting with the small model: one row, all latency
        append_case("append-one-chat", kv_heads=3, head_dim=64, rot_dim=64, chats=1, ctx_lo=300, ctx_hi=300),
        # the headline's batch: a token of each of 32 ragged chats on the 27B shape
        append_case("append-32-chats", chats=32),
        # decode rows beside two prompt chunks of the 8B shape's continuous batch
        append_case("append-chunks-beside-decode", chats=62, ctx_lo=32, ctx_hi=4096, chunks=2, chunk_rows=512,
                    chunk_past=1000),
        # a long prompt in the largest pass a context takes, beside the first tokens of others
        append_case("append-long-prompt", chats=3, ctx_lo=1, ctx_hi=64, chunks=1, chunk_rows=4000, chunk_past=8191),
        # one long chat on the 27B shape: few rows, all latency
        attend_case("attend-one-chat", ctx_lo=9000, ctx_hi=9000, budget=32),
        # 32 long chats on the 27B shape decode a token each
        attend_case("attend-32-chats", chats=32),
        # 16 chats verify seven drafts each on the hybrid's full-attention shape (heads of 256, a quarter rotary)
        attend_case("attend-verify", heads=24, kv_heads=4, head_dim=256, rot_dim=64, chats=16, rows=8, ctx_lo=2048,
                    ctx_hi=16384, budget=48),
        # the small model's row with a history and a few biases
        logits_case("adjust-one-row", "adjust", vocab=49152, history=300, biases=20),
        # 128 verify rows over the largest vocabulary, with histories, biases and grammars, rows padded
        logits_case("adjust-128-rows", "adjust", rows=128, vocab=248320, pad=64, history=2000, biases=100, grammars=4),
        # the small model's row with top-k
        logits_case("sample-one-row", "sample", vocab=49152, history=200, temp=0.8, top_k=40),
        # the headline's batch with everything a chat may ask for
        logits_case("sample-32-rows", "sample", rows=32, history=500, biases=30, grammars=3, temp=0.9, top_k=0, top_p=0.95,
                    min_p=0.0005),
        # 128 rows with a temperature alone: every token of the row takes part
        logits_case("sample-128-rows", "sample", rows=128, vocab=128256, temp=1.0),
    ]


def draw(rng):
    def logu(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "attend", "attend", "adjust", "sample", "sample"])
    if op == "append":
        head_dim = rng.choice([64, 128, 256])
        lo = logu(1, 4096)
        c = append_case("", kv_heads=rng.randint(1, 8), head_dim=head_dim, rot_dim=rng.choice([head_dim, head_dim // 4]),
                        chats=logu(1, 64), ctx_lo=lo, ctx_hi=logu(lo, 8192), chunks=rng.randint(0, 2),
                        chunk_rows=logu(2, 800), chunk_past=rng.choice([0, logu(1, 8000)]))
    elif op == "attend":
        lo, head_dim, kv = logu(1, 8192), rng.choice([64, 128, 128, 256]), rng.randint(1, 8)
        rows = rng.choice([1, 1, 1, rng.randint(2, 8)])
        chats = logu(1, 32) if rows == 1 else logu(1, 6)
        if head_dim == 256:
            chats = min(chats, 12)
        sink, recent = rng.randint(0, 2), rng.randint(1, 3)
        c = attend_case("", heads=kv * rng.randint(1, 8), kv_heads=kv, head_dim=head_dim,
                        rot_dim=rng.choice([head_dim, head_dim // 4]), chats=chats, rows=rows, ctx_lo=lo,
                        ctx_hi=logu(lo, 24000), budget=sink + recent + logu(1, 60), sink=sink, recent=recent)
    else:
        temp = rng.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.5]) if op == "sample" else 0.0
        c = logits_case("", op, rows=logu(1, 96), vocab=logu(1000, 160000), pad=rng.choice([0, 0, 1, 60]),
                        history=logu(1, 3000) if op == "adjust" else rng.choice([0, logu(1, 3000)]), biases=rng.choice([0, logu(1, 300)]),
                        grammars=rng.choice([0, rng.randint(1, 4)]), temp=temp,
                        top_k=rng.choice([0, 0, logu(1, 256)]) if temp else 0,
                        top_p=rng.choice([1.0, 0.95, 0.8, 0.5]) if temp else 1.0,
                        min_p=rng.choice([0.0, 0.0, 0.02]) if temp else 0.0, spread=rng.choice([0.5, 2.5, 4.0]))
    del c["name"]
    if "ctx_seed" in c:
        c["ctx_seed"] = rng.randrange(1 << 20)
    return c


def jobs_of(case):
    """(slot, past, rows) of each job, int32 [jobs, 3]: the chats, whose contexts are log-uniform, then the chunks."""
    rng = np.random.default_rng(case["ctx_seed"])
    past = np.round(np.exp(rng.uniform(math.log(case["ctx_lo"]), math.log(case["ctx_hi"]), case["chats"])))
    n = np.full(case["chats"], case.get("rows", 1))
    chunks = case.get("chunks", 0)
    past = np.concatenate([past, np.full(chunks, case.get("chunk_past", 0))])
    n = np.concatenate([n, np.full(chunks, case.get("chunk_rows", 0))])
    return np.stack([np.arange(len(n)), past, n], 1).astype(np.int32)


def rows_of(jobs):
    """Each row's slot and position, in job order."""
    n = jobs[:, 2]
    first = np.repeat(np.cumsum(n) - n, n)
    return np.repeat(jobs[:, 0], n), np.repeat(jobs[:, 1], n) + np.arange(n.sum()) - first


def work(case):
    if case["op"] in ("append", "attend"):
        jobs, D, nkv = jobs_of(case), case["head_dim"], case["kv_heads"]
        past, n = jobs[:, 1].astype(float), jobs[:, 2].astype(float)
    if case["op"] == "append":
        row = nkv * (D + D / 8)
        done = (past + n) // PAGE - past // PAGE                  # pages that the job completes
        early = np.where(done > 0, past % PAGE, 0)                # their rows that were there before
        return {"bytes": float(n.sum() * (8 * nkv * D + 2 * row) + early.sum() * row + done.sum() * nkv * (2 * D + D / 8)),
                "flops": float(n.sum() * nkv * D * 12)}
    if case["op"] == "attend":
        pos = rows_of(jobs)[1]
        seen = pos // PAGE + 1
        kept = np.minimum(seen, case["budget"])
        scored = np.where(seen > case["budget"], seen - case["sink"] - case["recent"], 0)
        tokens = kept * PAGE - (PAGE - 1 - pos % PAGE)
        per_slot = jobs[:, 2].max(initial=1)                      # a job's rows share the bounds, not the pages they keep
        return {"bytes": float(nkv * (scored.sum() / per_slot * (2 * D + D / 8) + tokens.sum() * 2 * (D + D / 8))
                               + 8.0 * len(pos) * case["heads"] * D),
                "flops": float(4.0 * case["heads"] * D * tokens.sum() + 2.0 * case["heads"] * D * scored.sum())}
    per = case["vocab"] * (8.0 if case["op"] == "adjust" else 4.0) + 8.0 * case["history"] + 8.0 * case["biases"]
    per += case["vocab"] / 8 if case["grammars"] else 0
    return {"bytes": case["rows"] * per, "flops": case["rows"] * case["vocab"] * (4.0 if case["op"] == "adjust" else 24.0)}


# ------------------------------------------------------------------- layout ---

def code_index(which, D, device="cuda"):
    """Byte of (token, channel)'s code in its block, [64, D]: which = 0 for keys, 1 for values."""
    t, d = torch.arange(PAGE, device=device)[:, None], torch.arange(D, device=device)[None]
    if which == 0:
        return t * D + (D // 4) * ((d % 32) // 8) + 8 * (d // 32) + d % 8
    v = 16 * ((t % 16) // 4) + 4 * (t // 16) + t % 4
    return ((v // 16) * D + d) * 16 + v % 16


def scale_index(which, D, device="cuda"):
    """Float, after the block's 64 * D code bytes, of (token, 32-channel group)'s scale, [64, D/32]."""
    ng = D // 32
    t, g = torch.arange(PAGE, device=device)[:, None], torch.arange(ng, device=device)[None]
    if which == 0:
        return t * ng + g
    v = 16 * ((t % 16) // 4) + 4 * (t // 16) + t % 4
    return ((v // 16) * ng + g) * 16 + v % 16


def bound_index(D, device="cuda"):
    """Byte of (largest 0 / smallest 1, channel)'s code in a page's 2 * D bound bytes of one kv head, [2, D]."""
    w, d = torch.arange(2, device=device)[:, None], torch.arange(D, device=device)[None]
    return (2 * w + (d % 32) // 16) * (D // 2) + 16 * (d // 32) + d % 16


def codes_view(pool, D):
    return pool[:, :, :PAGE * D]


def scales_view(pool, D):
    """The scales of a pool [pages, kv heads, block] as f32 [pages, kv heads, 64 * D/32], in place."""
    return pool.view(torch.float32)[:, :, PAGE * D // 4:]


def bound_codes_view(bounds, nkv, D):
    return bounds[:, :nkv * 2 * D].unflatten(1, (nkv, 2 * D))


def bound_scales_view(bounds, nkv, D):
    return bounds.view(torch.float32)[:, nkv * D // 2:].unflatten(1, (nkv, D // 32))


def quantise(x):
    """Codes (as f32 whole numbers) and scales of x [..., D] in groups of 32, as store_kv rounds them."""
    g = x.unflatten(-1, (-1, 32))
    d127 = torch.full((), 127.0, device=x.device)    # on the device: a host scalar would be multiplied by its reciprocal
    scale = g.abs().amax(-1) / d127
    inv = torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    return (g * inv[..., None]).round().clamp(-127, 127).flatten(-2), scale


def bounds_of(x):
    """Codes [..., 2, D] (largest, smallest) and scales [..., D/32] of the channels' range in x [..., tokens, D]."""
    mx, mn = x.amax(-2), x.amin(-2)
    d127 = torch.full((), 127.0, device=x.device)
    scale = torch.maximum(mx.abs(), mn.abs()).unflatten(-1, (-1, 32)).amax(-1) / d127
    s = scale.repeat_interleave(32, -1)
    some = s > 0
    s = torch.where(some, s, torch.ones_like(s))
    hi = torch.where(some, (mx / s).ceil().clamp(-127, 127), torch.zeros_like(s))
    lo = torch.where(some, (mn / s).floor().clamp(-127, 127), torch.zeros_like(s))
    return torch.stack([hi, lo], -2), scale


def rotate(x, cs, rot):
    """x [..., D] rotated by (cos, sin) cs [..., rot/2, 2] in the halves of its first `rot` channels."""
    a, o = x[..., :rot // 2], x[..., rot // 2:rot]
    c, s = cs[..., 0], cs[..., 1]
    return torch.cat([a * c - o * s, o * c + a * s, x[..., rot:]], -1)


# ------------------------------------------------------------------- inputs ---

def generator(seed, *key):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + sum((i + 1) * 7919 * k for i, k in enumerate(key))) % (1 << 62))
    return g


def normal(shape, seed, *key):
    return torch.randn(shape, generator=generator(seed, *key), device="cuda", dtype=torch.float32)


def rope_table(rows, rot):
    inv = 1000000.0 ** (-2.0 * torch.arange(rot // 2, device="cuda", dtype=torch.float64) / rot)
    ang = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float()


def prepare_cache(case, seed):
    """A paged cache that holds each job's rows before `past` (attend: before past + n): keys with a common offset and a
    topic that changes every hundred tokens or so, pages in any order, and behind a chat's last row what another left."""
    jobs, D, nkv, rot = jobs_of(case), case["head_dim"], case["kv_heads"], case["rot_dim"]
    total = jobs[:, 1] + jobs[:, 2]
    held = total if case["op"] == "attend" else jobs[:, 1]
    owned = -(-total // PAGE)
    n_pages, most = int(owned.sum()), int(owned.max())
    order = torch.randperm(n_pages, generator=generator(seed, 1), device="cuda").int()
    table = torch.zeros((len(jobs), most), dtype=torch.int32, device="cuda")
    table[torch.arange(most, device="cuda")[None] < torch.from_numpy(owned).cuda()[:, None]] = order
    offset, topics = normal((nkv, D), seed, 2), normal((n_pages + 1, nkv, D), seed, 3)
    first = np.cumsum(owned) - owned
    slot = torch.from_numpy(np.repeat(np.arange(len(jobs)), owned)).cuda()
    page = torch.from_numpy(np.arange(n_pages) - np.repeat(first, owned)).cuda()
    k = torch.empty((n_pages, nkv, PAGE * (D + D // 8)), dtype=torch.uint8, device="cuda")
    v = torch.empty_like(k)
    bounds = torch.empty((n_pages, nkv * (2 * D + D // 8)), dtype=torch.uint8, device="cuda")
    tok = page[:, None] * PAGE + torch.arange(PAGE, device="cuda")
    stale = tok >= torch.from_numpy(held).cuda()[slot][:, None]
    step = max(1, (1 << 28) // (PAGE * nkv * D))
    for at in range(0, n_pages, step):     # a piece at a time: the rows in f32 take four times the cache
        p = slice(at, min(at + step, n_pages))
        n = p.stop - at
        topic = topics[(slot[p] * 131 + page[p] // 2) % (n_pages + 1)]
        x = offset[None, :, None] + topic[:, :, None] + 0.7 * normal((n, nkv, PAGE, D), seed, 4, at)
        y = normal((n, nkv, PAGE, D), seed, 5, at)
        for which, pool, val in ((0, k, x), (1, v, y)):
            code, scale = quantise(val)
            bad = stale[p][:, None, :, None].expand_as(scale)
            where = order[p].long()
            blk = torch.empty((n, nkv, pool.shape[2]), dtype=torch.uint8, device="cuda")
            codes_view(blk, D)[:, :, code_index(which, D)] = (code + 128).to(torch.uint8)
            sc = torch.where(bad, torch.full_like(scale, math.nan), scale)
            scales_view(blk, D)[:, :, scale_index(which, D)] = sc
            pool[where] = blk
            if which == 0:
                b, bs = bounds_of(code * scale.repeat_interleave(32, -1))
                blk = torch.empty((n, bounds.shape[1]), dtype=torch.uint8, device="cuda")
                bound_codes_view(blk, nkv, D)[:, :, bound_index(D)] = b.to(torch.int8).view(torch.uint8)
                bound_scales_view(blk, nkv, D)[:] = bs
                bounds[where] = blk
    return dict(op=case["op"], jobs=jobs, k=k, v=v, bounds=bounds, table=table, nkv=nkv, D=D, rot=rot,
                rope=rope_table(int(total.max()), rot))


def prepare_logits(case, seed):
    rows, V = case["rows"], case["vocab"]
    full = normal((rows, V + case["pad"]), seed, 1)
    logits = full[:, :V]
    logits *= case["spread"]
    some = torch.randint(0, V, (rows, 12), generator=generator(seed, 2), device="cuda")
    logits.scatter_add_(1, some, normal((rows, 12), seed, 3).abs() * 3)   # a few likely tokens, as a model has them
    rng = np.random.default_rng(seed)
    s = dict(op=case["op"], rows=rows, V=V, logits=logits)

    def ragged(most):
        n = rng.integers(max(1, most // 2), most + 1, rows)
        return torch.from_numpy(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)).cuda(), int(n.sum())

    def per_row(value, dtype, also):
        a = np.full(rows, value, dtype)
        a[rng.random(rows) < 0.1] = also                  # one chat in ten asks for something else
        return torch.from_numpy(a).cuda()

    if case["history"]:     # the tokens so far, again and again the same ones
        s["pen_at"], n = ragged(case["history"])
        s["pen_ids"] = torch.from_numpy((V * rng.random(n) ** 3).astype(np.int32)).cuda()
        s["rep"], s["freq"] = per_row(1.1, np.float32, 1.0), per_row(0.2, np.float32, 0.0)
        s["pres"] = per_row(0.1, np.float32, 0.5)
    if case["biases"]:      # wishes and bans
        s["bias_at"], n = ragged(case["biases"])
        s["bias_ids"] = torch.from_numpy(rng.integers(0, V, n).astype(np.int32)).cuda()
        b = rng.normal(0, 3, n).astype(np.float32)
        b[rng.random(n) < 0.2] = -np.inf
        s["bias"] = torch.from_numpy(b).cuda()
    if case["grammars"]:    # the tokens that a grammar allows at this place: few, many or nearly all
        words = -(-V // 32)
        share = np.geomspace(0.02, 0.98, case["grammars"])
        bits = torch.rand((case["grammars"], words * 32), generator=generator(seed, 4), device="cuda")
        bits = (bits < torch.from_numpy(share).cuda()[:, None]).unflatten(1, (words, 32)).long()
        bits = (bits << torch.arange(32, device="cuda")).sum(-1)
        s["mask"] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).int()
        s["mask_of"] = torch.from_numpy(rng.integers(-1, case["grammars"], rows).astype(np.int32)).cuda()
    if case["op"] == "sample":
        s["u"] = torch.from_numpy(rng.random(rows)).cuda()
        if case["temp"] > 0:
            s["temp"] = per_row(case["temp"], np.float32, 0.0)
        if case["top_k"]:
            s["top_k"] = per_row(case["top_k"], np.int32, 0)
        if case["top_p"] < 1:
            s["top_p"] = per_row(case["top_p"], np.float32, 1.0)
        if case["min_p"] > 0:
            s["min_p"] = per_row(case["min_p"], np.float32, 0.0)
    return s


SAMPLING = ("temp", "top_k", "top_p", "min_p", "rep", "freq", "pres", "pen_at", "pen_ids", "bias_at", "bias_ids", "bias",
            "mask", "mask_of", "u")
_context = None


def context():
    """The program's one context: the device and the messages of the library's calls."""
    global _context
    if _context is None:
        from chattorrent_amd import ccdecode, configs
        _context = ccdecode.Context(configs.with_layers(configs.SMOLLM2, 1), n_max=64, t_max=1, slots=1, lo=1, hi=2)
    return _context


def prepare(case, seed):
    if case["op"] in ("append", "attend"):
        s = prepare_cache(case, seed)
        T = int(s["jobs"][:, 2].sum())
        if case["op"] == "append":
            # the projections' rows as a model leaves them: q | k | v beside each other would be wider; here k | v
            kv = normal((T, 2 * s["nkv"] * s["D"]), seed, 6)
            s["k_rows"], s["v_rows"] = kv[:, :s["nkv"] * s["D"]], kv[:, s["nkv"] * s["D"]:]
        else:
            s.update(q=normal((T, case["heads"] * s["D"]), seed, 6) * 1.5, heads=case["heads"], budget=case["budget"],
                     sink=case["sink"], recent=case["recent"])
    else:
        s = prepare_logits(case, seed)
    if own:      # the handles that a program keeps beside its buffers
        from chattorrent_amd import ccdecode
        s["ctx"] = context()
        if case["op"] in ("append", "attend"):
            s["cache"] = ccdecode.KVCache(s["k"], s["v"], s["table"], s["rope"], s["D"], bounds=s["bounds"])
        else:
            s["sampling"] = ccdecode.Sampling(s["rows"], s["V"], freq_cap=FREQ_CAP,
                                              **{n: s[n] for n in SAMPLING if n in s})
    return s


# ---------------------------------------------------------------------- run ---

def run(s):
    if own:
        c = s["ctx"]
        if s["op"] == "append":
            c.kv_append(s["cache"], s["jobs"], s["k_rows"], s["v_rows"])
            return pools(s)
        if s["op"] == "attend":
            return c.attend_pages(s["cache"], s["jobs"], s["q"], s["budget"], sink=s["sink"], recent=s["recent"])
        if s["op"] == "adjust":
            return c.adjust_logits(s["logits"], s["sampling"])
        return c.sample(s["logits"], s["sampling"])
    return {"append": plain_append, "attend": plain_attend, "adjust": plain_adjust, "sample": plain_sample}[s["op"]](s)


def pools(s):
    """The cache after an append, in place: every code as the whole number it is (the operator's definition fixes each bit),
    every scale as the f32 it is."""
    out = {}
    for name in ("k", "v"):
        out[name + "_codes"], out[name + "_scales"] = codes_view(s[name], s["D"]), scales_view(s[name], s["D"])
    out["bound_codes"] = bound_codes_view(s["bounds"], s["nkv"], s["D"])
    out["bound_scales"] = bound_scales_view(s["bounds"], s["nkv"], s["D"])
    return out


def plain_append(s):
    D, nkv, rot = s["D"], s["nkv"], s["rot"]
    slot, pos = rows_of(s["jobs"])
    slot, pos = torch.from_numpy(slot).cuda().long(), torch.from_numpy(pos).cuda().long()
    page = s["table"][slot, pos // PAGE].long()[:, None, None]
    head = torch.arange(nkv, device="cuda")[None, :, None]
    k = rotate(s["k_rows"].unflatten(1, (nkv, D)), s["rope"][pos][:, None], rot)
    for which, pool, x in ((0, s["k"], k), (1, s["v"], s["v_rows"].unflatten(1, (nkv, D)))):
        code, scale = quantise(x)
        codes_view(pool, D)[page, head, code_index(which, D)[pos % PAGE][:, None]] = (code + 128).to(torch.uint8)
        scales_view(pool, D)[page, head, scale_index(which, D)[pos % PAGE][:, None]] = scale
    past, n = s["jobs"][:, 1], s["jobs"][:, 2]
    first, last = past // PAGE, (past + n) // PAGE         # the pages that the rows complete
    done = last - first
    at = np.repeat(np.cumsum(done) - done, done)
    full = np.repeat(first, done) + np.arange(done.sum()) - at
    if len(full):
        of = s["table"][torch.from_numpy(np.repeat(s["jobs"][:, 0], done)).cuda().long(),
                        torch.from_numpy(full).cuda().long()].long()
        code = codes_view(s["k"][of], D)[:, :, code_index(0, D)].float() - 128
        scale = scales_view(s["k"][of], D)[:, :, scale_index(0, D)]
        b, bs = bounds_of(code * scale.repeat_interleave(32, -1))
        blk = torch.empty((len(of), s["bounds"].shape[1]), dtype=torch.uint8, device="cuda")
        bound_codes_view(blk, nkv, D)[:, :, bound_index(D)] = b.to(torch.int8).view(torch.uint8)
        bound_scales_view(blk, nkv, D)[:] = bs
        s["bounds"][of] = blk
    return pools(s)


def kept_pages(s, q, slot, pos):
    """The pages that each row and kv head keeps, [rows, kv heads, budget] (-1: none), from the rotated queries q."""
    D, nkv, budget = s["D"], s["nkv"], s["budget"]
    seen = pos // PAGE + 1
    most = int(s["table"].shape[1])
    qc, qs = quantise(q)                                                    # [R, nkv, G, D], [R, nkv, G, ng]
    pages = s["table"][slot].long()                                         # [R, P]
    b = bound_codes_view(s["bounds"], nkv, D)[pages][..., bound_index(D)].view(torch.int8).float()
    bs = bound_scales_view(s["bounds"], nkv, D)[pages]                      # [R, P, nkv, ng]
    b = b.permute(0, 2, 3, 4, 1)                                            # [R, nkv, 2, D, P]
    hi, lo = (b[:, :, w].unflatten(2, (-1, 32)) for w in (0, 1))            # [R, nkv, ng, 32, P]
    up = qc.clamp(min=0).unflatten(3, (-1, 32)).transpose(2, 3).contiguous()   # [R, nkv, ng, G, 32]
    down = qc.clamp(max=0).unflatten(3, (-1, 32)).transpose(2, 3).contiguous()
    dot = up @ hi.contiguous() + down @ lo.contiguous()                     # whole numbers under 2^24: exact
    scale = qs.transpose(2, 3).double()[..., None] * bs.permute(0, 2, 3, 1).double()[:, :, :, None]
    score = (scale * dot.double()).sum(2).amax(2).float()                   # [R, nkv, P]
    p = torch.arange(most, device="cuda")
    there = p < seen[:, None]
    always = there & ((p < s["sink"]) | (p >= (seen - s["recent"])[:, None]))
    score = torch.where(there[:, None], score, torch.full_like(score, -math.inf))
    score = torch.where(always[:, None], torch.full_like(score, math.inf), score)
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :budget]    # ties: the lower page first
    return torch.where(there[:, None].expand(-1, nkv, -1).gather(2, best), best, torch.full_like(best, -1))


def plain_attend(s):
    D, nkv, G = s["D"], s["nkv"], s["heads"] // s["nkv"]
    slot, pos = rows_of(s["jobs"])
    slot, pos = torch.from_numpy(slot).cuda().long(), torch.from_numpy(pos).cuda().long()
    q = rotate(s["q"].unflatten(1, (nkv, G, D)), s["rope"][pos][:, None, None], s["rot"])
    keep = kept_pages(s, q, slot, pos)
    page = s["table"][slot[:, None, None], keep.clamp(min=0)].long()
    head = torch.arange(nkv, device="cuda")[None, :, None]
    tok = keep[..., None] * PAGE + torch.arange(PAGE, device="cuda")
    there = ((keep >= 0)[..., None] & (tok <= pos[:, None, None, None])).flatten(2)     # [R, nkv, tokens]
    kv = []
    for which, pool in ((0, s["k"]), (1, s["v"])):
        blk = pool[page, head]                                                          # [R, nkv, B, block]
        code = blk[..., :PAGE * D][..., code_index(which, D)].float() - 128
        scale = blk.view(torch.float32)[..., PAGE * D // 4:][..., scale_index(which, D)]
        x = (code.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2).flatten(2, 3)
        kv.append(torch.where(there[..., None], x, torch.zeros_like(x)))                # what is not there may be NaN
    dots = (q @ kv[0].transpose(2, 3).contiguous()) / math.sqrt(D)
    dots = torch.where(there[:, :, None], dots, torch.full_like(dots, -math.inf))
    w = (dots - dots.amax(-1, keepdim=True)).exp()
    return ((w @ kv[1]) / w.sum(-1, keepdim=True)).flatten(1)


def row_of(at, n):
    """The row that each of n entries of a ragged list belongs to."""
    return torch.searchsorted(at, torch.arange(n, device="cuda", dtype=at.dtype), right=True) - 1


def adjusted(s):
    """Penalties, biases and masks on the rows, in 64 bits (their values lie next to borders), rounded once."""
    rows, V = s["rows"], s["V"]
    x = s["logits"]
    out = x.double()
    if "pen_at" in s:
        r = row_of(s["pen_at"], len(s["pen_ids"]))
        count = torch.zeros((rows, V), dtype=torch.int32, device="cuda")
        count.index_put_((r, s["pen_ids"].long()), torch.ones_like(r, dtype=torch.int32), accumulate=True)
        rep, freq, pres = (s[n].double()[:, None] for n in ("rep", "freq", "pres"))
        less = torch.where(out > 0, out / rep, out * rep) - (pres + (freq * count).clamp(max=FREQ_CAP))
        out = torch.where(count > 0, less, out)
    if "bias_at" in s:
        r = row_of(s["bias_at"], len(s["bias_ids"]))
        i = torch.arange(1, len(r) + 1, device="cuda")
        last = torch.zeros(rows * V, dtype=torch.int64, device="cuda")
        last.scatter_reduce_(0, r * V + s["bias_ids"].long(), i, "amax")
        last = last.view(rows, V)
        out = torch.where(last > 0, out + s["bias"].double()[(last - 1).clamp(min=0)], out)
    if "mask" in s:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        bits = bits.flatten(1)[:, :V].bool()
        of = s["mask_of"].long()
        out = torch.where(bits[of.clamp(min=0)] | (of < 0)[:, None], out, torch.full_like(out, -math.inf))
    return out.float()


def plain_adjust(s):
    return adjusted(s)


def plain_sample(s):
    rows, V = s["rows"], s["V"]
    x = adjusted(s)
    temp = s["temp"].double() if "temp" in s else torch.zeros(rows, dtype=torch.float64, device="cuda")
    greedy = temp <= 0
    first = (x == x.amax(1, keepdim=True)).int().argmax(1)
    t = (x.double() / torch.where(greedy, torch.ones_like(temp), temp)[:, None]).float()
    w = (t.double() - t.amax(1, keepdim=True).double()).exp()
    cut = torch.full((rows, 1), -math.inf, device="cuda")
    if "top_k" in s or "top_p" in s:
        best = t.sort(1, descending=True)[0]
        if "top_k" in s:
            k = s["top_k"].long()
            k = torch.where((k < 1) | (k > V), torch.full_like(k, V), k)
            cut = best.gather(1, k[:, None] - 1)
        if "top_p" in s:
            mass = torch.where(best >= cut, (best.double() - best[:, :1].double()).exp(), 0.0).cumsum(1)
            enough = mass >= s["top_p"].double()[:, None] * mass[:, -1:]
            at = torch.where(s["top_p"][:, None] < 1, enough.int().argmax(1, keepdim=True), V - 1)
            cut = torch.maximum(cut, best.gather(1, at))
    w = torch.where(t >= cut, w, 0.0)
    if "min_p" in s:
        w = torch.where(w >= s["min_p"].double()[:, None], w, 0.0)
    run_ = w.cumsum(1)
    total = run_[:, -1:]
    drawn = (run_ > s["u"][:, None] * total).int().argmax(1)
    prob = w.gather(1, drawn[:, None])[:, 0] / total[:, 0]
    return (torch.where(greedy, first, drawn).int(), torch.where(greedy, torch.ones_like(prob), prob).float())


# ------------------------------------------------------------- in 64 bits ---

def exact(case, seed):
    s = prepare_cache(case, seed) if case["op"] in ("append", "attend") else prepare_logits(case, seed)
    return {"append": exact_append, "attend": exact_attend, "adjust": exact_adjust, "sample": exact_sample}[case["op"]](
        case, seed, s)


def exact_append(case, seed, s):
    """The scales alone: codes are whole numbers that a rounding decides."""
    D, nkv, rot = s["D"], s["nkv"], s["rot"]
    T = int(s["jobs"][:, 2].sum())
    kv = normal((T, 2 * nkv * D), seed, 6).double().view(T, 2, nkv, D)
    slot, pos = rows_of(s["jobs"])
    cs = s["rope"][torch.from_numpy(pos).cuda().long()].double()[:, None]
    turned = torch.complex(kv[:, 0, :, :rot // 2], kv[:, 0, :, rot // 2:rot]) * torch.complex(cs[..., 0], cs[..., 1])
    x = [torch.cat([turned.real, turned.imag, kv[:, 0, :, rot:]], -1), kv[:, 1]]
    out = {"k_codes": None, "v_codes": None, "bound_codes": None, "bound_scales": None}
    page = s["table"].cpu().numpy()[slot, pos // PAGE]
    for which, name in ((0, "k"), (1, "v")):
        amax = x[which].reshape(T, nkv, D // 32, 32).abs().max(-1)[0] / 127.0
        pool = scales_view(s[name], D).double().clone()
        at = scale_index(which, D)[torch.from_numpy(pos % PAGE).cuda()]
        for h in range(nkv):
            pool[torch.from_numpy(page).cuda().long()[:, None], h, at] = amax[:, h]
        out[name + "_scales"] = pool
    return out


def exact_attend(case, seed, s):
    """Row by row and head by head, over the pages that the selection keeps (its scores are whole numbers times scales, and
    the queries in 8 bits come from the queries rotated in 32, as its definition has it)."""
    D, nkv, heads, jobs = s["D"], s["nkv"], case["heads"], s["jobs"]
    G, ng = heads // nkv, s["D"] // 32
    T = int(jobs[:, 2].sum())
    if T * nkv > 1500:
        return None
    q32 = (normal((T, heads * D), seed, 6) * 1.5).view(T, nkv, G, D)
    out = torch.empty((T, heads * D), dtype=torch.float64, device="cuda")
    ki, vi, ksi, vsi = code_index(0, D), code_index(1, D), scale_index(0, D), scale_index(1, D)
    half = s["rot"] // 2
    row = 0
    for slot, past, n in jobs.tolist():
        for i in range(n):
            p = past + i
            seen = p // PAGE + 1
            ids = s["table"][slot, :seen].long()
            c, sn = s["rope"][p, :, 0], s["rope"][p, :, 1]
            for h in range(nkv):
                qf = q32[row, h]
                r32 = qf.clone()
                r32[:, :half] = qf[:, :half] * c - qf[:, half:2 * half] * sn
                r32[:, half:2 * half] = qf[:, half:2 * half] * c + qf[:, :half] * sn
                qd = qf.double().clone()
                qd[:, :half] = qf[:, :half].double() * c.double() - qf[:, half:2 * half].double() * sn.double()
                qd[:, half:2 * half] = qf[:, half:2 * half].double() * c.double() + qf[:, :half].double() * sn.double()
                keep = torch.arange(seen, device="cuda")
                if seen > case["budget"]:
                    code, sc = quantise(r32)
                    b = bound_codes_view(s["bounds"], nkv, D)[ids, h][:, bound_index(D)].view(torch.int8).double()
                    bs = bound_scales_view(s["bounds"], nkv, D)[ids, h].double()
                    code = code.double()
                    best = torch.where(code[:, None] > 0, code[:, None] * b[None, :, 0], code[:, None] * b[None, :, 1])
                    best = best.view(G, seen, ng, 32).sum(-1) * sc.double()[:, None] * bs[None]
                    score = best.sum(-1).max(0)[0].float()
                    a, z = case["sink"], seen - case["recent"]
                    rank = torch.sort(score[a:z], descending=True, stable=True)[1][:case["budget"] - a - case["recent"]] + a
                    keep = torch.cat([keep[:a], rank.sort()[0], keep[z:]])
                kb, vb = s["k"][ids[keep], h], s["v"][ids[keep], h]
                kc = (kb[:, ki].double() - 128).view(-1, 64, ng, 32)
                kc = kc * kb.view(torch.float32)[:, 16 * D:][:, ksi].double()[..., None]
                vc = (vb[:, vi].double() - 128).view(-1, 64, ng, 32)
                vc = vc * vb.view(torch.float32)[:, 16 * D:][:, vsi].double()[..., None]
                tok = (keep[:, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)
                ok = tok <= p
                kc, vc = kc.reshape(-1, D)[ok], vc.reshape(-1, D)[ok]
                a = torch.softmax(qd @ kc.t() / math.sqrt(D), -1)
                out[row].view(nkv, G, D)[h] = a @ vc
            row += 1
    return out


def exact_rows(s):
    """Each row's adjusted logits in 64 bits, entry by entry as the definition says, on the host."""
    V = s["V"]
    x = s["logits"].cpu().numpy().astype(np.float64)
    get = {n: s[n].cpu().numpy() for n in SAMPLING if n in s}
    for r in range(s["rows"]):
        if "pen_at" in get:
            ids, count = np.unique(get["pen_ids"][get["pen_at"][r]:get["pen_at"][r + 1]], return_counts=True)
            v, rep = x[r, ids], np.float64(get["rep"][r])
            v = np.where(v > 0, v / rep, v * rep)
            x[r, ids] = v - (np.float64(get["pres"][r]) + np.minimum(np.float64(get["freq"][r]) * count, FREQ_CAP))
        if "bias_at" in get:
            a, z = get["bias_at"][r:r + 2]
            wish = dict(zip(get["bias_ids"][a:z].tolist(), get["bias"][a:z].tolist()))   # a later entry replaces
            for t, b in wish.items():
                x[r, t] += b
        if "mask" in get and get["mask_of"][r] >= 0:
            bits = np.unpackbits(get["mask"][get["mask_of"][r]].view(np.uint8), bitorder="little")[:V]
            x[r, bits == 0] = -np.inf
    return x, get


def exact_adjust(case, seed, s):
    return torch.from_numpy(exact_rows(s)[0])


def exact_sample(case, seed, s):
    """The draw over the row's scaled logits, which the definition rounds to 32 bits twice, and sums in 64."""
    x, get = exact_rows(s)
    ids, probs = np.zeros(s["rows"], np.int32), np.ones(s["rows"])
    for r in range(s["rows"]):
        v = x[r].astype(np.float32)
        temp = float(get["temp"][r]) if "temp" in get else 0.0
        if temp <= 0:
            ids[r] = int(np.argmax(v))
            continue
        t = (v.astype(np.float64) / temp).astype(np.float32).astype(np.float64)
        w = np.exp(t - t.max())
        k = int(get["top_k"][r]) if "top_k" in get else 0
        if 0 < k < s["V"]:
            w[t < np.partition(t, -k)[-k]] = 0
        if "top_p" in get and get["top_p"][r] < 1:
            order = np.argsort(-t, kind="stable")
            mass = np.cumsum(w[order])
            w[t < t[order[int(np.argmax(mass >= float(get["top_p"][r]) * mass[-1]))]]] = 0
        if "min_p" in get:
            w[w < float(get["min_p"][r])] = 0
        run_ = np.cumsum(w)
        ids[r] = int(np.argmax(run_ > get["u"][r] * run_[-1]))
        probs[r] = w[ids[r]] / run_[-1]
    return torch.from_numpy(ids), torch.from_numpy(probs)

"""The operators of chats whose cache is kept within a bound that are measured: what a token's row goes through in a cache
that holds images beside text and gives up the tokens that nothing attends to.

  append   cc_kv_append_at: new keys, rotated to positions of one or several axes (time, height, width), and values into the
           rows of a paged int8 cache, whatever those positions are, and a fresh mark for each row
  weigh    cc_attend_weigh: attention of a job's rows over all rows of its cache, and the attention weight that each of these
           has received, added up over query rows and the query heads of its kv head
  evict    cc_kv_evict: of each kv head's rows the `keep` with the largest weight stay, the chat's first and latest tokens
           whatever theirs; those from row `keep` on move into the rows that others leave

Each is reached through `chattorrent_amd.ccdecode` where `own` is set; otherwise it is computed in elementary operations.
A cache is held as the library lays it out: a block for each (page of 64 tokens, kv head) with its codes (biased by 128) and
then one f32 scale for each token and 32 channels, `code_index` and `scale_index` saying where; its marks are, for each such
block, 64 weights and 64 token numbers. Model shapes (heads, widths) are those of `chattorrent_amd.configs`.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64


# -------------------------------------------------------------------- cases ---

def append_case(name, **kw):
    return dict(dict(name=name, op="append", kv_heads=8, head_dim=128, rot_dim=128, axes=3, interleaved=True, chats=0,
                     ctx_lo=128, ctx_hi=16384, rows=1, chunks=0, chunk_rows=0, chunk_past=0, ctx_seed=1234), **kw)


def weigh_case(name, **kw):
    return dict(dict(name=name, op="weigh", heads=40, kv_heads=8, head_dim=128, rot_dim=128, axes=3, interleaved=True,
                     chats=0, ctx_lo=2048, ctx_hi=16384, rows=1, chunks=0, chunk_rows=0, chunk_past=0, observe=1 << 20,
                     fade=1.0, ctx_seed=1234), **kw)


def evict_case(name, **kw):
    return dict(dict(name=name, op="evict", kv_heads=8, head_dim=128, chats=1, ctx_lo=4096, ctx_hi=16384, keep=2048,
                     over=0, sink=4, recent=64, ctx_seed=1234), **kw)


def listed():
    return [
        # the next token of one chat with the small model, behind an image: all latency
        append_case("append-one-chat", kv_heads=3, head_dim=64, rot_dim=64, chats=1, ctx_lo=300, ctx_hi=300),
        # an image's patches of two chats, 32 x 32 of them each, beside 30 chats' tokens, on the hybrid's full-attention
        # shape (heads of 256, a quarter rotary)
        append_case("append-images-beside-decode", kv_heads=4, head_dim=256, rot_dim=64, chats=30, chunks=2,
                    chunk_rows=1024, chunk_past=37),
        # a long prompt with images in the largest pass a context takes, axes in runs of pairs
        append_case("append-long-prompt", chats=3, ctx_lo=1, ctx_hi=64, chunks=1, chunk_rows=4000, chunk_past=8191,
                    interleaved=False),
        # one long chat on the 27B shape, whose tokens' weights add up: few rows, all latency
        weigh_case("weigh-one-chat", chats=1, ctx_lo=9000, ctx_hi=9000),
        # 32 chats on the 27B shape decode a token each; the last step's weights alone will say what goes
        weigh_case("weigh-32-chats", chats=32, fade=0.0),
        # 16 chats verify seven drafts each on the hybrid's full-attention shape
        weigh_case("weigh-verify", heads=24, kv_heads=4, head_dim=256, rot_dim=64, chats=16, rows=8, ctx_hi=8192),
        # the end of a prompt on the 8B shape: its last 64 rows say what of it stays; one axis
        weigh_case("weigh-prompt-end", heads=32, axes=1, chunks=1, chunk_rows=512, chunk_past=4000, observe=64, fade=0.0),
        # a prompt's chunk far into it, every row of which counts, beside seven chats' tokens
        weigh_case("weigh-chunk-beside-decode", chats=7, chunks=1, chunk_rows=512, chunk_past=8192),
        # 32 chats at their bound: a page's worth of new rows goes
        evict_case("evict-32-chats-at-the-bound", chats=32, ctx_lo=4160, ctx_hi=4160, keep=4096, over=64),
        # one chat with the small model gives up the one row that is over
        evict_case("evict-one-row", kv_heads=3, head_dim=64, ctx_lo=1025, ctx_hi=1025, keep=1024, over=1),
        # long prompts are cut down to their bound
        evict_case("evict-32-prompts", chats=32),
        # one prompt on the hybrid's full-attention shape
        evict_case("evict-one-prompt", kv_heads=4, head_dim=256, ctx_lo=16001, ctx_hi=16001, keep=5000),
    ]


def draw(rng):
    def logu(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "weigh", "weigh", "weigh", "evict", "evict"])
    D, kv = rng.choice([64, 128, 128, 256]), rng.randint(1, 8)
    rot = rng.choice([D, D // 4])
    lo = logu(1, 6000)
    at = dict(kv_heads=kv, head_dim=D, rot_dim=rot, axes=rng.choice([1, 2, 3, 3, 4]), interleaved=rng.random() < 0.5)
    if op == "append":
        c = append_case("", chats=logu(1, 64), ctx_lo=lo, ctx_hi=logu(lo, 8192), chunks=rng.randint(0, 2),
                        chunk_rows=logu(2, 1000), chunk_past=rng.choice([0, logu(1, 8000)]), **at)
    elif op == "weigh":
        group = rng.randint(1, 8)
        rows = rng.choice([1, 1, 1, rng.randint(2, 8)])
        c = weigh_case("", heads=kv * group, chats=logu(1, 32 if rows == 1 else 12), rows=rows, ctx_lo=lo,
                       ctx_hi=logu(lo, 12000), chunks=rng.choice([0, 0, 1, 2]),
                       chunk_rows=logu(9, 400 if D < 256 else 150), chunk_past=rng.choice([0, logu(1, 5000)]),
                       observe=rng.choice([1 << 20, 1 << 20, 1, logu(1, 200)]), fade=rng.choice([0.0, 0.5, 1.0, 1.0]),
                       **at)
    else:
        keep, over = logu(80, 6000), rng.choice([0, 1, logu(1, 300)])
        hi = logu(max(lo, keep), 16000)
        sink = rng.randint(0, 8)
        c = evict_case("", kv_heads=kv, head_dim=D, chats=logu(1, 32), ctx_lo=keep + over if over else lo,
                       ctx_hi=keep + over if over else hi, keep=keep, over=over, sink=sink, recent=rng.randint(0, 64))
    del c["name"]
    c["ctx_seed"] = rng.randrange(1 << 20)
    return c


def contexts(case):
    rng = np.random.default_rng(case["ctx_seed"])
    return np.round(np.exp(rng.uniform(math.log(case["ctx_lo"]), math.log(case["ctx_hi"]), case["chats"]))).astype(np.int64)


def jobs_of(case):
    """(slot, past, rows) of each job, int32 [jobs, 3]: the chats, whose contexts are log-uniform, then the chunks."""
    past = np.concatenate([contexts(case), np.full(case["chunks"], case["chunk_past"])])
    n = np.concatenate([np.full(case["chats"], case["rows"]), np.full(case["chunks"], case["chunk_rows"])])
    return np.stack([np.arange(len(n)), past, n], 1).astype(np.int32)


def evictions(case):
    """(slot, rows, keep, tokens seen) of each chat, int32 [chats, 4]: prompts hold every token that they have seen, chats at
    their bound have seen three times as many."""
    rows = contexts(case)
    seen = 3 * rows if case["over"] else rows
    return np.stack([np.arange(len(rows)), rows, np.full(len(rows), case["keep"]), seen], 1).astype(np.int32)


def rows_of(jobs):
    """Each row's slot and index in the cache, in job order."""
    n = jobs[:, 2]
    first = np.repeat(np.cumsum(n) - n, n)
    return np.repeat(jobs[:, 0], n), np.repeat(jobs[:, 1], n) + np.arange(n.sum()) - first


def work(case):
    D, nkv = case["head_dim"], case["kv_heads"]
    row = nkv * (D + D / 8)                       # a row's codes and scales, of K or V
    if case["op"] == "evict":
        j = evictions(case).astype(float)
        over = np.maximum(j[:, 1] - case["keep"], 0)
        # as many rows move as there are rows below `keep` to give up: those of them that the cut falls on
        free = np.maximum(j[:, 1] - case["sink"] - case["recent"], 1)
        moved = over * np.minimum(np.maximum(case["keep"] - case["sink"], 0) / free, 1)
        read = np.where(over > 0, j[:, 1], 0).sum() * nkv * 8
        return {"bytes": float(read + moved.sum() * (4 * row + 16 * nkv)) + 64.0, "flops": float(read / 8)}
    jobs = jobs_of(case)
    past, n = jobs[:, 1].astype(float), jobs[:, 2].astype(float)
    if case["op"] == "append":
        return {"bytes": float(n.sum() * (8 * nkv * D + 2 * row + 8 * nkv + 4 * case["axes"])),
                "flops": float(n.sum() * nkv * D * 12)}
    seen = (past + (n + 1) / 2) * n
    looked = np.minimum(n, case["observe"])
    tokens = (past + n).sum()
    return {"bytes": float(tokens * (2 * row + 4 * nkv * (2 if case["fade"] else 1)) + 8.0 * n.sum() * case["heads"] * D),
            "flops": float(4.0 * case["heads"] * D * seen.sum() + case["heads"] * ((past + n) * looked).sum())}


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


def codes_view(pool, D):
    return pool[:, :, :PAGE * D]


def scales_view(pool, D):
    """The scales of a pool [pages, kv heads, block] as f32 [pages, kv heads, 64 * D/32], in place."""
    return pool.view(torch.float32)[:, :, PAGE * D // 4:]


def quantise(x):
    """Codes (as f32 whole numbers) and scales of x [..., D] in groups of 32, as store_kv rounds them."""
    g = x.unflatten(-1, (-1, 32))
    d127 = torch.full((), 127.0, device=x.device)    # on the device: a host scalar would be multiplied by its reciprocal
    scale = g.abs().amax(-1) / d127
    inv = torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    return (g * inv[..., None]).round().clamp(-127, 127).flatten(-2), scale


def axis_of(case):
    """The axis that each pair of rotary channels turns by, uint8 [rot/2]: the first axis has the most, and either the axes
    take turns as long as all have pairs left, or each has a run of its own."""
    pairs, axes = case["rot_dim"] // 2, case["axes"]
    if case["interleaved"]:
        a = np.arange(pairs) % axes
        a[pairs - pairs // 8:] = 0
        return a.astype(np.uint8)
    return np.minimum(np.arange(pairs) * axes // max(1, pairs), axes - 1).astype(np.uint8)


def turned(x, s):
    """x [rows, ..., D] rotated to the rows' positions in the halves of its first `rot` channels."""
    rot, half = s["rot"], s["rot"] // 2
    which = torch.from_numpy(s["axis_of"].astype(np.int64)).cuda()
    cs = s["rope"][s["pos"].long()[:, which], torch.arange(half, device="cuda")]       # [rows, rot/2, 2]
    cs = cs.view(len(x), *([1] * (x.dim() - 2)), half, 2)
    a, o, c, n = x[..., :half], x[..., half:rot], cs[..., 0], cs[..., 1]
    return torch.cat([a * c - o * n, o * c + a * n, x[..., rot:]], -1)


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


def positions(case, jobs, seed):
    """int32 [rows, axes]: a chat's text goes on where its images and the tokens that it gave up have left it, the same on
    every axis; of a chunk's rows every second run of 32 x 32 is an image's patches, whose time stands still."""
    rng = np.random.default_rng(seed)
    out = np.zeros((int(jobs[:, 2].sum()), case["axes"]), np.int64)
    row = 0
    for slot, past, n in jobs.tolist():
        i = np.arange(n)
        text = int(past * rng.uniform(0.6, 1.8)) + i
        out[row:row + n] = text[:, None]
        image = (i // 1024) % 2 == 0
        if slot >= case["chats"] and case["axes"] > 1:
            start = text - i % 1024
            parts = [start, start + (i % 1024) // 32, start + i % 32, start]
            out[row:row + n] = np.where(image[:, None], np.stack(parts[:case["axes"]], 1), out[row:row + n])
        row += n
    return out.astype(np.int32)


def prepare_pages(total, seed):
    """(page table, [pages] slot, page within the slot, index in the cache) of slots that hold `total` rows each, their pages in
    any order."""
    owned = -(-total // PAGE)
    n_pages, most = int(owned.sum()), int(owned.max())
    order = torch.randperm(n_pages, generator=generator(seed, 1), device="cuda").int()
    table = torch.zeros((len(total), most), dtype=torch.int32, device="cuda")
    table[torch.arange(most, device="cuda")[None] < torch.from_numpy(owned).cuda()[:, None]] = order
    first = np.cumsum(owned) - owned
    slot = torch.from_numpy(np.repeat(np.arange(len(total)), owned)).cuda()
    page = torch.from_numpy(np.arange(n_pages) - np.repeat(first, owned)).cuda()
    return table, slot, page, order.long()


def prepare_cache(case, seed, total, held):
    """A paged cache with `held` rows of each slot: keys with a common offset, a few that stand out and a topic that changes
    every hundred tokens or so; behind a chat's last row what another left."""
    D, nkv = case["head_dim"], case["kv_heads"]
    table, slot, page, order = prepare_pages(total, seed)
    n_pages = len(order)
    offset, topics = normal((nkv, D), seed, 2), normal((n_pages + 1, nkv, D), seed, 3)
    k = torch.empty((n_pages, nkv, PAGE * (D + D // 8)), dtype=torch.uint8, device="cuda")
    v = torch.empty_like(k)
    stale = page[:, None] * PAGE + torch.arange(PAGE, device="cuda") >= torch.from_numpy(held).cuda()[slot][:, None]
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
            blk = torch.empty((n, nkv, pool.shape[2]), dtype=torch.uint8, device="cuda")
            codes_view(blk, D)[:, :, code_index(which, D)] = (code + 128).to(torch.uint8)
            scales_view(blk, D)[:, :, scale_index(which, D)] = torch.where(bad, torch.full_like(scale, math.nan), scale)
            pool[order[p]] = blk
    # the marks: a weight and a token number of each row, in one piece of memory
    marks = torch.zeros((2, n_pages, nkv, PAGE), dtype=torch.int32, device="cuda")
    return dict(op=case["op"], k=k, v=v, table=table, nkv=nkv, D=D, marks=marks, weight=marks[0].view(torch.float32),
                token=marks[1], slot_of=slot, page_of=page, order=order)


def prepare(case, seed):
    if case["op"] == "evict":
        j = evictions(case)
        s = prepare_cache(case, seed, j[:, 1].astype(np.int64), j[:, 1].astype(np.int64))
        s.update(jobs=j, sink=case["sink"], recent=case["recent"])
        # weights as attention leaves them, most of them small and a few large; token numbers: all of a prompt's in order, at
        # the bound a part of those seen, in any order but for the new rows'
        s["weight"].copy_(torch.exp(2.0 * normal(s["weight"].shape, seed, 7)))
        tok = s["page_of"][:, None] * PAGE + torch.arange(PAGE, device="cuda")
        if case["over"]:
            rows = int(j[0, 1])
            mix = torch.stack([torch.randperm(3 * rows - case["over"], generator=generator(seed, 8, i), device="cuda")
                               for i in range(len(j))])
            old = mix[s["slot_of"][:, None], tok.clamp(max=rows - 1)]
            tok = torch.where(tok >= case["keep"], 2 * rows + tok, old)
        s["token"][s["order"]] = tok.int()[:, None].expand(-1, s["nkv"], -1)
        s["marks_before"] = s["marks"].clone()
        s["rope"] = rope_table(1, 2)
    else:
        jobs = jobs_of(case)
        total = (jobs[:, 1] + jobs[:, 2]).astype(np.int64)
        s = prepare_cache(case, seed, total, total if case["op"] == "weigh" else jobs[:, 1].astype(np.int64))
        pos = positions(case, jobs, seed)
        s.update(jobs=jobs, rot=case["rot_dim"], axis_of=axis_of(case), rope=rope_table(int(pos.max()) + 1, case["rot_dim"]),
                 pos=torch.from_numpy(pos).cuda())
        T = len(pos)
        if case["op"] == "append":
            # the projections' rows as a model leaves them, k | v beside each other
            kv = normal((T, 2 * s["nkv"] * s["D"]), seed, 6)
            s["k_rows"], s["v_rows"] = kv[:, :s["nkv"] * s["D"]], kv[:, s["nkv"] * s["D"]:]
            s["first"] = (jobs[:, 1] * 2).astype(np.int32)          # half of a chat's tokens are gone
        else:
            s.update(q=normal((T, case["heads"] * s["D"]), seed, 6) * 1.5, heads=case["heads"], observe=case["observe"],
                     fade=case["fade"])
            s["weight"].copy_(torch.exp(normal(s["weight"].shape, seed, 7)))
            s["marks_before"] = s["marks"].clone()
    if own:      # the handles that a program keeps beside its buffers
        from chattorrent_amd import ccdecode
        s["ctx"] = context()
        s["cache"] = ccdecode.KVCache(s["k"], s["v"], s["table"], s["rope"], s["D"])
        s["held"] = ccdecode.Marks(s["weight"], s["token"])
        if "pos" in s:
            s["at"] = ccdecode.Positions(s["pos"], s["axis_of"])
    return s


_context = None


def context():
    """The program's one context: the device and the messages of the library's calls."""
    global _context
    if _context is None:
        from chattorrent_amd import ccdecode, configs
        _context = ccdecode.Context(configs.with_layers(configs.SMOLLM2, 1), n_max=64, t_max=1, slots=1, lo=1, hi=2)
    return _context


# ---------------------------------------------------------------------- run ---

def run(s):
    """One pass. Weights that add up, and a cache that was cut down, start from what their marks were before: the same pass
    can be made again."""
    if s["op"] == "evict" or (s["op"] == "weigh" and s["fade"]):
        s["marks"].copy_(s["marks_before"])
    if own:
        c = s["ctx"]
        if s["op"] == "append":
            c.kv_append_at(s["cache"], s["jobs"], s["k_rows"], s["v_rows"], s["at"], marks=s["held"], first=s["first"])
            return pools(s)
        if s["op"] == "weigh":
            out = c.attend_weigh(s["cache"], s["jobs"], s["q"], s["at"], marks=s["held"], observe=s["observe"],
                                 fade=s["fade"])
            return {"out": out, "weight": s["weight"]}
        c.kv_evict(s["cache"], s["held"], s["jobs"], sink=s["sink"], recent=s["recent"])
        return pools(s)
    return {"append": plain_append, "weigh": plain_weigh, "evict": plain_evict}[s["op"]](s)


def pools(s):
    """The cache and its marks after a pass, in place: every code as the whole number it is, every scale as the f32 it is."""
    out = {"weight": s["weight"], "token": s["token"]}
    for name in ("k", "v"):
        out[name + "_codes"], out[name + "_scales"] = codes_view(s[name], s["D"]), scales_view(s[name], s["D"])
    return out


def plain_append(s):
    D, nkv = s["D"], s["nkv"]
    slot, row = rows_of(s["jobs"])
    i = row - np.repeat(s["jobs"][:, 1], s["jobs"][:, 2])
    number = torch.from_numpy((np.repeat(s["first"], s["jobs"][:, 2]) + i).astype(np.int32)).cuda()
    slot, row = torch.from_numpy(slot).cuda().long(), torch.from_numpy(row).cuda().long()
    page = s["table"][slot, row // PAGE].long()[:, None]
    head = torch.arange(nkv, device="cuda")[None]
    s["weight"][page, head, (row % PAGE)[:, None]] = 0.0
    s["token"][page, head, (row % PAGE)[:, None]] = number[:, None]
    page, head = page[..., None], head[..., None]
    k = turned(s["k_rows"].unflatten(1, (nkv, D)), s)
    for which, pool, x in ((0, s["k"], k), (1, s["v"], s["v_rows"].unflatten(1, (nkv, D)))):
        code, scale = quantise(x)
        codes_view(pool, D)[page, head, code_index(which, D)[row % PAGE][:, None]] = (code + 128).to(torch.uint8)
        scales_view(pool, D)[page, head, scale_index(which, D)[row % PAGE][:, None]] = scale
    return pools(s)


def plain_weigh(s):
    D, nkv, G = s["D"], s["nkv"], s["heads"] // s["nkv"]
    q = turned(s["q"].unflatten(1, (nkv, G, D)), s)
    out = torch.empty_like(s["q"])
    at = 0
    for slot, past, n in s["jobs"].tolist():
        T = past + n
        page = s["table"][slot, :-(-T // PAGE)].long()
        kv = []
        for which, pool in ((0, s["k"]), (1, s["v"])):
            blk = pool[page].transpose(0, 1)                                            # [nkv, P, block]
            code = blk[..., :PAGE * D][..., code_index(which, D)].float() - 128
            scale = blk.contiguous().view(torch.float32)[..., PAGE * D // 4:][..., scale_index(which, D)]
            kv.append((code.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2).flatten(1, 2)[:, :T])
        rows = q[at:at + n].permute(1, 0, 2, 3).reshape(nkv, n * G, D)
        dots = (rows @ kv[0].transpose(1, 2).contiguous()) / math.sqrt(D)               # [nkv, n * G, T]
        last = past + torch.arange(n, device="cuda").repeat_interleave(G)
        dots.masked_fill_(torch.arange(T, device="cuda") > last[:, None], -math.inf)
        w = (dots - dots.amax(-1, keepdim=True)).exp()
        w = w / w.sum(-1, keepdim=True)
        out[at:at + n] = (w @ kv[1]).unflatten(1, (n, G)).transpose(0, 1).reshape(n, -1)
        got = w[:, max(0, n - s["observe"]) * G:].sum(1)                                # [nkv, T]
        t = torch.arange(T, device="cuda")
        at_page, h = page[t // PAGE][None], torch.arange(nkv, device="cuda")[:, None]
        before = s["weight"][at_page, h, (t % PAGE)[None]]
        s["weight"][at_page, h, (t % PAGE)[None]] = before * s["fade"] + got if s["fade"] else got
        at += n
    return {"out": out, "weight": s["weight"]}


def plain_evict(s):
    D, nkv = s["D"], s["nkv"]
    for slot, rows, keep, seen in s["jobs"].tolist():
        if rows <= keep:
            continue
        r = torch.arange(rows, device="cuda")
        page, h = s["table"][slot, r // PAGE].long()[None], torch.arange(nkv, device="cuda")[:, None]
        w, tok = s["weight"][page, h, (r % PAGE)[None]], s["token"][page, h, (r % PAGE)[None]]
        safe = (tok < s["sink"]) | (tok >= seen - s["recent"])
        w = torch.where(safe, torch.full_like(w, math.inf), w)
        best = torch.sort(w, dim=-1, descending=True, stable=True)[1][:, :keep]        # ties: the lower row first
        kept = torch.zeros((nkv, rows), dtype=torch.bool, device="cuda").scatter_(1, best, True)
        hh, to = (~kept[:, :keep]).nonzero(as_tuple=True)       # both in (head, row) order, and as many of a head
        _, of = kept[:, keep:].nonzero(as_tuple=True)
        of = of + keep
        p, pt, po = s["table"][slot].long(), to // PAGE, of // PAGE
        for marks in (s["weight"], s["token"]):
            marks[p[pt], hh, to % PAGE] = marks[p[po], hh, of % PAGE]
        for which, pool in ((0, s["k"]), (1, s["v"])):
            for view, index in ((codes_view(pool, D), code_index(which, D)), (scales_view(pool, D), scale_index(which, D))):
                view[p[pt][:, None], hh[:, None], index[to % PAGE]] = view[p[po][:, None], hh[:, None], index[of % PAGE]]
    return pools(s)


# ------------------------------------------------------------- in 64 bits ---

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"append": exact_append, "weigh": exact_weigh, "evict": exact_evict}[case["op"]](case, s)


def exact_turned(x, case, s):
    """x f64 [rows, heads, D]: every pair as a complex number, turned by its axis's position."""
    half = case["rot_dim"] // 2
    z = torch.complex(x[..., :half], x[..., half:2 * half])
    out = x.clone()
    for j, a in enumerate(s["axis_of"].tolist()):
        cs = s["rope"][s["pos"][:, a].long(), j].double()
        t = z[..., j] * torch.complex(cs[:, 0], cs[:, 1])[:, None]
        out[..., j], out[..., half + j] = t.real, t.imag
    return out


def exact_append(case, s):
    """The scales alone: codes are whole numbers that a rounding decides, marks are set and not computed."""
    D, nkv = s["D"], s["nkv"]
    x = [exact_turned(s["k_rows"].double().unflatten(1, (nkv, D)), case, s), s["v_rows"].double().unflatten(1, (nkv, D))]
    slot, row = rows_of(s["jobs"])
    page = torch.from_numpy(s["table"].cpu().numpy()[slot, row // PAGE]).cuda().long()
    out = {"weight": None, "token": None, "k_codes": None, "v_codes": None}
    for which, name in ((0, "k"), (1, "v")):
        amax = x[which].reshape(len(row), nkv, D // 32, 32).abs().max(-1)[0] / 127.0
        pool = scales_view(s[name], D).double().clone()
        at = scale_index(which, D)[torch.from_numpy(row % PAGE).cuda()]
        for h in range(nkv):
            pool[page[:, None], h, at] = amax[:, h]
        out[name + "_scales"] = pool
    return out


def exact_weigh(case, s):
    """Job by job and head by head, the softmax of each row from the whole line of its scores."""
    D, nkv, heads = s["D"], s["nkv"], case["heads"]
    G, ng = heads // nkv, D // 32
    q = exact_turned(s["q"].double().unflatten(1, (heads, D)), case, s)
    out = torch.empty((len(q), heads, D), dtype=torch.float64, device="cuda")
    weight = s["weight"].double()
    index = [(code_index(w, D), scale_index(w, D)) for w in (0, 1)]
    at = 0
    for slot, past, n in s["jobs"].tolist():
        T = past + n
        ids = s["table"][slot, :(T + PAGE - 1) // PAGE].long()
        future = torch.ones((n, T), dtype=torch.bool, device="cuda").triu(past + 1)
        for h in range(nkv):
            kv = []
            for pool, (ci, si) in zip((s["k"], s["v"]), index):
                blk = pool[ids, h].contiguous()
                c = (blk[:, ci].double() - 128).reshape(-1, ng, 32)
                kv.append((c * blk.view(torch.float32)[:, 16 * D:][:, si].double().reshape(-1, ng, 1)).reshape(-1, D)[:T])
            got = torch.zeros(T, dtype=torch.float64, device="cuda")
            for g in range(G):
                a = q[at:at + n, h * G + g] @ kv[0].t().contiguous() / math.sqrt(D)
                a[future] = -math.inf
                a = torch.softmax(a, 1)
                out[at:at + n, h * G + g] = a @ kv[1]
                got += a[max(0, n - case["observe"]):].sum(0)
            flat = torch.zeros(len(ids) * PAGE, dtype=torch.float64, device="cuda")
            flat[:T] = got
            there = (torch.arange(len(flat), device="cuda") < T).view(-1, PAGE)
            old = weight[ids, h]
            weight[ids, h] = torch.where(there, (old * case["fade"] if case["fade"] else 0.0) + flat.view(-1, PAGE), old)
        at += n
    return {"out": out.flatten(1), "weight": weight}


def exact_evict(case, s):
    """Where a row's marks end, chat by chat and head by head on the host; codes and scales move with them, unchanged."""
    weight, token = s["weight"].cpu().numpy().astype(np.float64), s["token"].cpu().numpy()
    table = s["table"].cpu().numpy()
    for slot, rows, keep, seen in s["jobs"].tolist():
        if rows <= keep:
            continue
        r = np.arange(rows)
        page = table[slot, r // PAGE]
        for h in range(s["nkv"]):
            w, t = weight[page, h, r % PAGE], token[page, h, r % PAGE]
            w = np.where((t < case["sink"]) | (t >= seen - case["recent"]), np.inf, w)
            gone = np.ones(rows, bool)
            gone[np.lexsort((r, -w))[:keep]] = False
            to, of = r[:keep][gone[:keep]], r[keep:][~gone[keep:]]
            for m in (weight, token):
                m[page[to], h, to % PAGE] = m[page[of], h, of % PAGE]
    return {"weight": torch.from_numpy(weight), "token": torch.from_numpy(token), "k_codes": None, "v_codes": None,
            "k_scales": None, "v_scales": None}

"""The host side of the operators on device buffers, on the CPU: which calls are
refused, how a call goes over launches, and whose errors it reports. The HIP
runtime is the stand-in of test_host_path.py, with the device calls that these
entries make added."""
import json
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

ADDED = """
#include "hip_stand_in.cc"
extern "C" {
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
void stand_in_stale() { last = hipErrorInvalidValue; }   // what a caller's own failed call leaves
}
"""

PRELUDE = """
import ctypes as C, json, sys
import numpy as np
sys.path.insert(0, %r)
from chattorrent_amd import ccdecode as cc, configs
hip = C.CDLL(%r)
hip.stand_in_reset.argtypes = [C.c_long]
hip.stand_in_launches.restype = C.c_char_p
out = []
ctx = cc.Context(configs.with_layers(configs.SMOLLM2, 1), n_max=256, t_max=8, slots=2)
held = []

def launched():
    return [k for n in hip.stand_in_launches().decode().split()
            for k in ("k_kv_append", "k_page_score", "k_attend_pages", "k_logits_adjust", "k_sample_scale", "k_sample_mass",
                      "k_sample_cut", "k_sample_weights", "k_sample_pick") if k in n]

class A:                      # an array in "device" memory
    def __init__(self, *shape, of=np.float32):
        self.a = np.zeros(shape, of)
        self.shape, self.dtype = self.a.shape, self.a.dtype
        held.append(self.a)
    def data_ptr(self):
        return self.a.ctypes.data // 16 * 16 + 16 if self.a.nbytes > 4096 else self.a.ctypes.data
    def stride(self, d):
        return int(np.prod(self.shape[1:])) if d == 0 else 1

def cache(nkv=2, D=128, pages=8, per=8, slots=4, bounds=True, rope=None):
    rope = per * 64 if rope is None else rope
    blk = 64 * D + 64 * D // 32 * 4
    mem = [np.zeros(pages * nkv * blk + 64, np.uint8) for _ in range(2)]
    b, t, r = np.zeros(pages * (nkv * 2 * D + 1024) + 64, np.uint8), np.zeros((slots, per), np.uint32), np.zeros((rope, D), np.float32)
    held.extend(mem + [b, t, r])
    at = lambda a: (a.ctypes.data + 15) // 16 * 16
    c = cc.CCache()
    c.n_kv_heads, c.head_dim, c.rot_dim, c.n_pages, c.max_pages, c.slots, c.rope_rows = nkv, D, D, pages, per, slots, rope
    c.k, c.v, c.bounds, c.page_table, c.rope = at(mem[0]), at(mem[1]), at(b) if bounds else None, t.ctypes.data, at(r)
    return c

F = np.zeros(1 << 22, np.float32)
f = (F.ctypes.data + 15) // 16 * 16

def jobs(*j):
    a = np.array(j, np.int32)
    held.append(a)
    return a.ctypes.data, len(j)

def append(c, *j, k=f, v=f, ldk=None, ldv=None):
    w = c.n_kv_heads * c.head_dim
    return ctx.lib.cc_kv_append(ctx.h, C.byref(c), *jobs(*j), k, ldk or w, v, ldv or w, None)

def attend(c, *j, heads=4, budget=3, sink=1, recent=1, q=f, ldq=None, o=f + (1 << 23), ldo=None, ws=f + (1 << 21), n=1 << 22):
    w = heads * c.head_dim
    return ctx.lib.cc_attend_pages(ctx.h, C.byref(c), *jobs(*j), heads, budget, sink, recent, q, ldq or w, o, ldo or w, ws, n, None)

def why():
    return ctx.lib.cc_last_error(ctx.h).decode()
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("hip")
    so = str(d / "stand_in.so")
    (d / "stand_in.cc").write_text(ADDED)
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I",
                    os.path.join(ROCM, "include"), "-I", HERE, str(d / "stand_in.cc"), "-o", so], check=True)

    def run(code):
        r = subprocess.run([sys.executable, "-c", PRELUDE % (ROOT, so) + code + "\nprint(json.dumps(out))"], cwd=ROOT,
                           env=dict(os.environ, LD_PRELOAD=so), stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True,
                           timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
        return json.loads(r.stdout.splitlines()[-1])

    return run


def test_cache_refusals(host):
    out = host("""
c = cache()
def no(text, st):
    out.append([text, st, why()])
hip.stand_in_reset(-1)
for j in ((4, 0, 1), (-1, 0, 1), (0, -1, 1), (0, 0, 0), (0, 512, 1), (0, 2**31 - 1, 1), (0, 1, 512), (0, 5, -3)):
    no("job 0", append(c, j))
    no("job 0", attend(c, j))
no("job 1", attend(c, (0, 0, 1), (9, 0, 1)))
no("rope", append(cache(rope=100), (0, 99, 2)))
no("twice", append(c, (1, 0, 1), (2, 0, 1), (1, 5, 1)))
no("at least one", ctx.lib.cc_kv_append(ctx.h, C.byref(c), None, 1, f, 256, f, 256, None))
no("at least one", ctx.lib.cc_kv_append(ctx.h, C.byref(c), jobs((0, 0, 1))[0], 0, f, 256, f, 256, None))
no("ldk", append(c, (0, 0, 1), ldk=255))
no("ldk", append(c, (0, 0, 1), ldv=255))
no("must be set", append(c, (0, 0, 1), k=None))
no("must be set", attend(c, (0, 0, 1), o=None))
no("bounds", attend(cache(bounds=False), (0, 200, 1)))
no("bounds", ctx.lib.cc_kv_bounds(ctx.h, C.byref(cache(bounds=False)), *jobs((0, 0, 64)), None))
for s, r, b in ((-1, 1, 3), (0, 0, 3), (3, 1, 3), (2**31 - 1, 2, 3), (2**31 - 1, 2**31 - 1, 2**31 - 1)):
    no("sink", attend(c, (0, 200, 1), sink=s, recent=r, budget=b))
no("budget", attend(c, (0, 200, 1), budget=0))
no("multiple", attend(c, (0, 200, 1), heads=3))
no("multiple", attend(c, (0, 200, 1), heads=0))
no("multiple", attend(c, (0, 200, 1), heads=2 * 1025))
no("ldq", attend(c, (0, 200, 1), ldq=511))
no("ldq", attend(c, (0, 200, 1), ldo=511))
no("workspace", attend(c, (0, 200, 1), ws=None))
no("workspace", attend(c, (0, 200, 1), n=64))
no("workspace", attend(c, (0, 200, 1), ws=f + 8))
no("share memory", attend(c, (0, 200, 1), o=f))
no("share memory", attend(c, (0, 200, 2), o=f + 4 * 512))
no("share memory", attend(c, (0, 200, 2), ldq=1024, ldo=1024, o=f + 4 * 511))
for field, bad in (("head_dim", 96), ("head_dim", 32), ("rot_dim", 3), ("rot_dim", 0), ("rot_dim", 130), ("n_kv_heads", 0),
                   ("n_kv_heads", 2000), ("max_pages", 0), ("max_pages", 32769), ("n_pages", 0), ("slots", 0), ("rope_rows", 0),
                   ("k", None), ("v", None), ("page_table", None), ("rope", None), ("k", c.k + 8), ("bounds", c.bounds + 4)):
    d = cache()
    setattr(d, field, bad)
    no("cache:", append(d, (0, 0, 1)))
    no("cache:", attend(d, (0, 0, 1)))
    out.append(["", 5 if ctx.lib.cc_attend_workspace(ctx.h, C.byref(d), 1, 4, 3) == 0 else 0, ""])
out.append(["", 5 if launched() == [] else 0, "nothing launched"])
""")
    for text, st, said in out:
        assert st == 5 and text in said, (text, st, said)


def test_a_call_over_launches(host):
    """At most 128 jobs a launch, whole calls of few; kv_bounds launches nothing where no page is whole."""
    out = host("""
def n(st):
    assert st == 0, why()
    got = launched()
    hip.stand_in_reset(-1)
    return got
hip.stand_in_reset(-1)
c = cache(slots=300)
out = dict(one=n(append(c, (0, 0, 1))), many=n(append(c, *[(s, 0, 1) for s in range(300)])),
           seen=n(attend(c, (0, 100, 1))), scored=n(attend(c, (0, 300, 1))), all=n(attend(c, (0, 300, 1), budget=8)),
           rows=n(attend(c, *[(s % 300, 0, 1) for s in range(130)])),
           beside=n(attend(c, (0, 200, 3), ldq=1024, ldo=1024, o=f + 4 * 512)),
           none=n(ctx.lib.cc_kv_bounds(ctx.h, C.byref(c), *jobs((0, 1, 126)), None)),
           some=n(ctx.lib.cc_kv_bounds(ctx.h, C.byref(c), *jobs((0, 1, 127)), None)))
""")
    assert out["one"] == ["k_kv_append"] and out["many"] == ["k_kv_append"] * 3
    assert out["seen"] == ["k_attend_pages"] or out["seen"] == ["k_page_score", "k_attend_pages"]
    assert out["scored"] == ["k_page_score", "k_attend_pages"]
    assert out["all"][-1] == "k_attend_pages" and out["beside"][-1] == "k_attend_pages"
    assert out["rows"].count("k_attend_pages") == 2
    assert out["none"] == [] and out["some"] == ["k_kv_append"]


def test_logits_refusals(host):
    out = host("""
V = 100
def ask(**kw):
    s = cc.CSampling()
    s.freq_cap = 1.5
    for n, v in kw.items():
        setattr(s, n, v)
    return s
def adjust(s, x=f, ld=V, rows=2, vocab=V, o=f + (1 << 20), ldo=V):
    return ctx.lib.cc_logits_adjust(ctx.h, x, ld, rows, vocab, C.byref(s), o, ldo, None)
def sample(s, x=f, ld=V, rows=2, vocab=V, ids=f + (1 << 20), ws=f + (1 << 21), n=1 << 22):
    return ctx.lib.cc_sample(ctx.h, x, ld, rows, vocab, C.byref(s), ids, None, ws, n, None)
def no(text, st):
    out.append([text, st, why()])
hip.stand_in_reset(-1)
for kw in (dict(rows=0), dict(rows=-1), dict(rows=65536), dict(vocab=0), dict(vocab=(1 << 20) + 1, ld=1 << 21), dict(ld=99), dict(x=None),
           dict(ld=(1 << 31) + 1)):
    no("logits:", adjust(ask(), **kw))
    no("logits:", sample(ask(), **kw))
for text, kw in (("history", dict(rep=f)), ("history", dict(freq=f)), ("history", dict(pres=f)), ("negative", dict(n_pen=-1)),
                 ("negative", dict(n_bias=-1)), ("negative", dict(n_masks=-1)), ("pen_ids", dict(pen_at=f, n_pen=3)),
                 ("bias_ids", dict(bias_at=f, n_bias=3)), ("bias_ids", dict(bias_at=f, n_bias=3, bias_ids=f)),
                 ("mask_of", dict(mask=f, mask_words=4, n_masks=1)), ("mask_words", dict(mask=f, mask_of=f, mask_words=3, n_masks=1)),
                 ("mask_words", dict(mask=f, mask_of=f, mask_words=-1, n_masks=1)), ("freq_cap", dict(freq_cap=-1.0)),
                 ("freq_cap", dict(freq_cap=float("nan")))):
    no(text, adjust(ask(**kw)))
    no(text, sample(ask(**kw)))
no("random", sample(ask(temp=f)))
no("workspace", sample(ask(), ws=None))
no("workspace", sample(ask(), ws=f + 4))
no("workspace", sample(ask(), n=8))
no("must be set", sample(ask(), ids=None))
no("must be set", adjust(ask(), o=None))
no("ldo", adjust(ask(), ldo=99))
no("ldo", adjust(ask(), o=f, ld=128, ldo=127))
no("shares", adjust(ask(), o=f + 4))
no("shares", adjust(ask(), o=f + 4 * 100))
no("shares", adjust(ask(), o=f + 4 * 150, ld=200, ldo=300))
no("shares", adjust(ask(), o=f + 4 * 101, ld=200, ldo=200))
out.append(["", 5 if launched() == [] else 0, "nothing launched"])
ok = [adjust(ask(), o=f), adjust(ask(), o=f + 4 * 100, ld=200, ldo=200), adjust(ask(), o=f + 4 * 200), adjust(ask(), rows=1, o=f + 4 * 100)]
out.append(["", 5 if ok == [0] * 4 else 0, str(ok)])
for bad in ((0, 100), (-1, 100), (65536, 100), (2, 0), (2, (1 << 20) + 1)):
    out.append(["", 5 if ctx.lib.cc_sample_workspace(*bad, C.byref(ask())) == 0 else 0, str(bad)])
""")
    for text, st, said in out:
        assert st == 5 and text in said, (text, st, said)


def test_launches_of_the_sampler_and_their_errors(host):
    """Two launches without cuts, two with min-p alone, three with top-k or top-p; the one that fails is reported and ends the
    call; an error that the caller's own earlier call left is not this call's."""
    out = host("""
V = 20000
def sample(*names, fail=-1, stale=False):
    s = cc.CSampling()
    s.freq_cap = 1.5
    for n in names:
        setattr(s, n, f)
    hip.stand_in_reset(fail)
    if stale:
        hip.stand_in_stale()
    st = ctx.lib.cc_sample(ctx.h, f, V, 2, V, C.byref(s), f + (1 << 20), None, f + (1 << 21), 1 << 23, None)
    left = hip.hipGetLastError()
    return [st, left, launched()]
def append_(stale):
    hip.stand_in_reset(-1)
    if stale:
        hip.stand_in_stale()
    st = append(cache(), (0, 0, 1))
    hip.hipGetLastError()
    return st
T = ("temp", "u")
out = dict(greedy=sample(), plain=sample(*T), minp=sample(*T, "min_p"), topk=sample(*T, "top_k"), topp=sample(*T, "top_p", "min_p"),
           failed=[sample(*T, "top_k", fail=k) for k in range(3)] + [sample(*T, fail=k) for k in range(2)],
           stale=sample(*T, "top_k", stale=True)[0], stale_append=append_(True))
""")
    assert out["greedy"] == [0, 0, ["k_sample_weights", "k_sample_pick"]] == out["plain"]
    assert out["minp"][2] == ["k_sample_scale", "k_sample_mass"]
    cut = ["k_sample_scale", "k_sample_mass", "k_sample_cut"]
    assert out["topk"] == [0, 0, cut] == out["topp"]
    assert out["failed"] == [[8, 0, cut[:k + 1]] for k in range(3)] + [[8, 0, ["k_sample_weights", "k_sample_pick"][:k + 1]] for k in range(2)]
    assert out["stale"] == 0 and out["stale_append"] == 0

"""The host side of the operators of a bounded cache (cc_kv_append_at,
cc_attend_weigh, cc_kv_evict), on the CPU: which calls are refused, how a call
goes over launches, whose errors it reports, and which arrays the Python binding
takes. The HIP runtime is the stand-in of test_host_operators.py, and of
test_host_binding.py with two GPUs."""
import json
import os
import subprocess
import sys

import pytest
import test_host_binding as two
import test_host_operators as one

MORE = """
NAMES = ("k_kv_append_at", "k_weigh_query", "k_weigh_page", "k_weigh_many", "k_weigh_finish", "k_weigh_join", "k_weigh_sums", "k_weigh_add",
         "k_evict_select", "k_evict_move")
def launched():
    return [next(k for k in NAMES if k in n) for n in hip.stand_in_launches().decode().split() if any(k in n for k in NAMES)]

def positions(n=3, pos=f, of=None):
    p = cc.CPositions()
    p.n_axes, p.pos = n, pos
    if of is not None:
        a = np.array(of, np.uint8)
        held.append(a)
        p.axis_of = a.ctypes.data
    return p

def marks(weight=f, token=f):
    m = cc.CMarks()
    m.weight, m.token = weight, token
    return m

def ref(x):
    return None if x is None else C.byref(x)

def append_at(c, *j, at=None, m=None, first=None, k=f, v=f, ldk=None, ldv=None):
    w = c.n_kv_heads * c.head_dim
    fa = None if first is None else np.array(first, np.int32)
    held.append(fa)
    return ctx.lib.cc_kv_append_at(ctx.h, C.byref(c), ref(at), ref(m), *jobs(*j), None if fa is None else fa.ctypes.data, k,
                                   ldk or w, v, ldv or w, None)

def weigh(c, *j, at=None, m=marks(), heads=4, observe=1000, fade=1.0, q=f, ldq=None, o=f + (1 << 23), ldo=None,
          ws=f + (1 << 21), n=1 << 22):
    w = heads * c.head_dim
    return ctx.lib.cc_attend_weigh(ctx.h, C.byref(c), ref(at), ref(m), *jobs(*j), heads, observe, C.c_float(fade), q, ldq or w,
                                   o, ldo or w, ws, n, None)

def room(c, *j, heads=4, observe=1000):
    return ctx.lib.cc_weigh_workspace(ctx.h, C.byref(c), *jobs(*j), heads, observe)

def evict(c, *j, m=marks(), sink=0, recent=0, ws=f + (1 << 21), n=1 << 22):
    return ctx.lib.cc_kv_evict(ctx.h, C.byref(c), ref(m), *jobs(*j), sink, recent, ws, n, None)
"""


def runner(tmp_path_factory, source, prelude):
    d = tmp_path_factory.mktemp("hip")
    so = str(d / "stand_in.so")
    (d / "stand_in.cc").write_text(source)
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I",
                    os.path.join(one.ROCM, "include"), "-I", one.HERE, str(d / "stand_in.cc"), "-o", so], check=True)

    def run(code):
        r = subprocess.run([sys.executable, "-c", prelude % (one.ROOT, so) + code + "\nprint(json.dumps(out))"], cwd=one.ROOT,
                           env=dict(os.environ, LD_PRELOAD=so), stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True,
                           timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
        return json.loads(r.stdout.splitlines()[-1])

    return run


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    return runner(tmp_path_factory, one.ADDED, one.PRELUDE + MORE.replace("%", "%%"))


@pytest.fixture(scope="module")
def gpus(tmp_path_factory):
    return runner(tmp_path_factory, two.TWO_GPUS, two.PRELUDE)


def test_refusals(host):
    out = host("""
c = cache()
def no(text, st):
    out.append([text, st, why()])
hip.stand_in_reset(-1)
for j in ((4, 0, 1), (-1, 0, 1), (0, -1, 1), (0, 0, 0), (0, 512, 1), (0, 2**31 - 1, 1), (0, 1, 512), (0, 5, -3)):
    for at in (None, positions()):
        no("job 0", append_at(c, j, at=at))
        no("job 0", weigh(c, j, at=at))
    out.append(["", 5 if room(c, j) == 0 else 0, str(j)])
no("rope", append_at(cache(rope=100), (0, 99, 2)))
no("rope", weigh(cache(rope=100), (0, 99, 2)))
for f_ in (append_at, weigh):
    no("twice", f_(c, (1, 0, 1), (2, 0, 1), (1, 5, 1)))
    no("axes", f_(c, (0, 0, 1), at=positions(0)))
    no("axes", f_(c, (0, 0, 1), at=positions(5)))
    no("pos must", f_(c, (0, 0, 1), at=positions(pos=None)))
    no("pos must", f_(c, (0, 0, 1), at=positions(pos=f + 2)))
    no("axis_of[63]", f_(c, (0, 0, 1), at=positions(2, of=[0, 1] * 31 + [0, 2])))
    no("marks", f_(c, (0, 0, 1), m=marks(weight=None)))
    no("marks", f_(c, (0, 0, 1), m=marks(token=f + 4)))
no("at least one", append_at(c))
no("at least one", weigh(c))
no("ldk", append_at(c, (0, 0, 1), ldk=255))
no("ldk", append_at(c, (0, 0, 1), ldv=255))
no("must be set", append_at(c, (0, 0, 1), v=None))
no("token numbers", append_at(c, (0, 0, 1), first=[-1]))
no("token numbers", append_at(c, (0, 0, 1), (1, 0, 3), first=[2**31 - 2, 2**31 - 3]))
no("must be set", weigh(c, (0, 0, 1), q=None))
no("must be set", weigh(c, (0, 0, 1), o=None))
for h in (3, 0, -2, 2 * 1025):
    no("multiple", weigh(c, (0, 200, 1), heads=h, ldq=1 << 20, ldo=1 << 20))
no("observe", weigh(c, (0, 200, 1), observe=-1))
out.append(["", 5 if room(c, (0, 200, 1), observe=-1) == 0 else 0, "observe"])
for bad in (-0.5, 1.5, float("nan"), float("inf")):
    no("fade", weigh(c, (0, 200, 1), fade=bad))
no("ldq", weigh(c, (0, 200, 1), ldq=511))
no("ldq", weigh(c, (0, 200, 1), ldo=511))
no("workspace", weigh(c, (0, 200, 1), ws=None))
no("workspace", weigh(c, (0, 200, 1), n=64))
no("workspace", weigh(c, (0, 200, 1), ws=f + 8))
no("share memory", weigh(c, (0, 200, 1), o=f))
no("share memory", weigh(c, (0, 200, 2), ldq=1024, ldo=1024, o=f + 4 * 511))
for j in ((4, 10, 5, 10), (-1, 10, 5, 10), (0, -1, 5, 10), (0, 513, 5, 10), (0, 10, 0, 10), (0, 10, -1, 10), (0, 10, 5, -1)):
    no("job 0", evict(c, j))
no("at least one", evict(c))
no("twice", evict(c, (1, 10, 5, 10), (1, 10, 5, 10)))
no("must be set", evict(c, (0, 10, 5, 10), m=None))
no("marks", evict(c, (0, 10, 5, 10), m=marks(weight=f + 8)))
no("negative", evict(c, (0, 10, 5, 10), sink=-1))
no("negative", evict(c, (0, 10, 5, 10), recent=-1))
no("workspace", evict(c, (0, 400, 200, 400), ws=None))
need = ctx.lib.cc_evict_workspace(C.byref(c), *jobs((0, 400, 200, 400)))
no("workspace", evict(c, (0, 400, 200, 400), n=need - 4))
out.append(["", 5 if need >= 2 * 4 * 2 * 200 else 0, str(need)])
no("workspace", evict(c, (0, 400, 200, 400), ws=f + 4))
for field, bad in (("head_dim", 96), ("rot_dim", 0), ("n_kv_heads", 0), ("n_kv_heads", 2000), ("max_pages", 32769),
                   ("n_pages", 0), ("slots", 0), ("rope_rows", 0), ("k", None), ("page_table", None), ("rope", None), ("v", c.v + 8)):
    d = cache()
    setattr(d, field, bad)
    no("cache:", append_at(d, (0, 0, 1)))
    no("cache:", weigh(d, (0, 0, 1)))
    no("cache:", evict(d, (0, 10, 5, 10)))
    out.append(["", 5 if room(d, (0, 0, 1)) == 0 else 0, field])
out.append(["", 5 if launched() == [] else 0, str(launched())])
""")
    for text, st, said in out:
        assert st == 5 and text in said, (text, st, said)


def test_launches_and_their_errors(host):
    """What a call launches: few and many columns apart, a job of many rows in pieces; nothing where nothing is to be given up;
    the launch that fails is reported and ends the call, an error that an earlier call of the caller's left is not."""
    out = host("""
def n(st):
    assert st == 0, why()
    got = launched()
    hip.stand_in_reset(-1)
    return got
hip.stand_in_reset(-1)
c, long = cache(slots=300), cache(nkv=1, D=64, pages=200, per=200)
big = dict(ws=f, n=1 << 40)     # nothing runs
out = dict(append=n(append_at(c, (0, 0, 1))), many=n(append_at(c, *[(s, 0, 1) for s in range(300)], first=range(300))),
           token=n(weigh(c, (0, 10, 1), m=None)), weighed=n(weigh(c, (0, 10, 1))), off=n(weigh(c, (0, 10, 1), observe=0)),
           chunk=n(weigh(c, (0, 100, 60), **big)), alone=n(weigh(c, (0, 100, 60), m=None, **big)),
           both=n(weigh(c, (0, 100, 60), (1, 5, 1), **big)), jobs=n(weigh(c, *[(s, 0, 1) for s in range(130)], **big)),
           pieces=n(weigh(long, (0, 10, 9000), heads=1, **big)),
           none=n(evict(c, (0, 64, 64, 64), (1, 3, 10, 5), ws=None, n=0)), one=n(evict(c, (0, 65, 64, 65), ws=None, n=0)),
           lot=n(evict(c, (0, 400, 200, 400))), jobs_=n(evict(c, *[(s, 300, 200, 300) for s in range(200)], **big)))
def fails(k, call):
    hip.stand_in_reset(k)
    st = call()
    left = hip.hipGetLastError()
    got = launched()
    hip.stand_in_reset(-1)
    return [st, left, len(got)]
out["failed"] = [fails(k, lambda: weigh(c, (0, 100, 60), (1, 5, 1), **big)) for k in range(3)]
out["failed"] += [fails(k, lambda: evict(c, (0, 400, 200, 400))) for k in range(2)] + [fails(0, lambda: append_at(c, (0, 0, 1)))]
hip.stand_in_stale()
out["stale"] = [weigh(c, (0, 100, 60), **big), append_at(c, (0, 0, 1)), evict(c, (0, 400, 200, 400))]
hip.hipGetLastError()
""")
    assert out["append"] == ["k_kv_append_at"] and out["many"] == ["k_kv_append_at"] * 3
    page = ["k_weigh_page"]      # which rotates up to 16 columns itself
    assert out["token"] == page == out["off"] and out["weighed"] == page + ["k_weigh_finish"]
    many = ["k_weigh_query", "k_weigh_many", "k_weigh_join", "k_weigh_sums", "k_weigh_add"]
    assert [k for k in many if k in out["chunk"]] == out["chunk"] and "k_weigh_sums" in out["chunk"]
    assert "k_weigh_sums" not in out["alone"] and "k_weigh_finish" not in out["token"]
    assert out["both"][:2] == page + ["k_weigh_finish"] and out["both"][2:] == out["chunk"]
    assert out["jobs"].count("k_weigh_page") == 3 and out["pieces"].count("k_weigh_sums") == 3
    assert out["none"] == [] and out["one"] == ["k_evict_select"] and out["lot"] == ["k_evict_select", "k_evict_move"]
    assert out["jobs_"] == ["k_evict_select", "k_evict_move"] * 3
    assert out["failed"] == [[8, 0, k + 1] for k in range(3)] + [[8, 0, 1], [8, 0, 2], [8, 0, 1]]
    assert out["stale"] == [0, 0, 0]


def test_the_bindings_arrays(gpus):
    """Positions and marks of other shapes, types or GPUs are refused by the binding before anything is launched."""
    out = gpus("""
out = []
c = cache(0, 0, 0, 0, 0)
k, q = on(0, 3, 128), on(0, 3, 256)
pos = lambda g=0, rows=3, axes=3, of=np.int32: on(g, rows, axes, of=of)
of = [0, 1, 2] * 10 + [0, 0]
m = cc.Marks(on(0, 4, 2, 64), on(0, 4, 2, 64, of=np.int32))
def no(call):
    hip.stand_in_reset(-1)
    try:
        call()
    except ValueError as e:
        out.append([hip.stand_in_launches() == b"", str(e)])
    else:
        out.append([False, "taken"])
j = [(0, 5, 3)]
both = (lambda p, m_=None: ctx[0].kv_append_at(c, j, k, k, p, marks=m_), lambda p, m_=None: ctx[0].attend_weigh(c, j, q, p, marks=m_))
for call in both:
    no(lambda: call(cc.Positions(pos(rows=2), of)))
    no(lambda: call(cc.Positions(pos(g=1), of)))
    no(lambda: call(cc.Positions(pos(), of[:-1])))
    no(lambda: call(None, cc.Marks(on(0, 5, 2, 64), on(0, 5, 2, 64, of=np.int32))))
    no(lambda: call(None, cc.Marks(on(1, 4, 2, 64), on(1, 4, 2, 64, of=np.int32))))
no(lambda: cc.Positions(pos(of=np.int64), of))
no(lambda: cc.Positions(on(0, 3, of=np.int32), of))
no(lambda: cc.Positions(pos(), [0, 3] * 16))
no(lambda: cc.Positions(pos(), [0, -1] * 16))
no(lambda: cc.Positions(pos(), [0.5] * 32))
no(lambda: cc.Marks(on(0, 4, 2, 64), on(1, 4, 2, 64, of=np.int32)))
no(lambda: cc.Marks(on(0, 4, 2, 64), on(0, 4, 3, 64, of=np.int32)))
no(lambda: cc.Marks(on(0, 4, 2, 32), on(0, 4, 2, 32, of=np.int32)))
no(lambda: cc.Marks(on(0, 4, 2, 64, of=np.float64), on(0, 4, 2, 64, of=np.int32)))
no(lambda: ctx[0].kv_append_at(c, j, k, k, first=[1, 2]))
no(lambda: ctx[0].kv_append_at(c, j, k, k, first=[0.5]))
no(lambda: ctx[0].attend_weigh(c, j, on(0, 3, 100), marks=m))
no(lambda: ctx[0].kv_evict(c, m, [(0, 5, 3)]))
no(lambda: ctx[0].kv_evict(c, m, [(0, 2**31, 3, 5)]))
no(lambda: ctx[1].kv_evict(c, m, [(0, 65, 64, 65)]))
hip.stand_in_reset(-1)
ctx[0].kv_append_at(c, j, k, k, cc.Positions(pos(), of), marks=m, first=[9])
ctx[0].attend_weigh(c, j, q, cc.Positions(pos()), marks=m)
ctx[0].kv_evict(c, m, [(0, 65, 64, 65)])
out.append([hip.stand_in_launches().count(b"k_") >= 4, ""])
""")
    for ok, said in out:
        assert ok, said


def test_the_bindings_numbers_past_32_bits(gpus):
    """A count that 32 bits do not hold means all of the rows, a negative one is refused, however far below 0."""
    out = gpus("""
out = []
c = cache(0, 0, 0, 0, 0)
q = on(0, 3, 256)
m = cc.Marks(on(0, 4, 2, 64), on(0, 4, 2, 64, of=np.int32))
for observe in (3, 1 << 32, 1 << 40):
    hip.stand_in_reset(-1)
    ctx[0].attend_weigh(c, [(0, 5, 3)], q, marks=m, observe=observe)
    out.append([b"k_weigh_finish" in hip.stand_in_launches(), str(observe)])
def no(call):
    try:
        call()
    except cc.CCError as e:
        out.append(["negative" in str(e), str(e)])
    else:
        out.append([False, "taken"])
no(lambda: ctx[0].attend_weigh(c, [(0, 5, 3)], q, marks=m, observe=-(1 << 32)))
no(lambda: ctx[0].kv_evict(c, m, [(0, 65, 64, 65)], sink=-(1 << 32)))
no(lambda: ctx[0].kv_evict(c, m, [(0, 65, 64, 65)], recent=-(1 << 40)))
ctx[0].kv_evict(c, m, [(0, 65, 64, 65)], sink=1 << 32, recent=1 << 40)
""")
    for ok, said in out:
        assert ok, said


def test_the_memory_of_a_launch(host):
    """What a launch with several jobs holds in memory stays near 1 GiB: more jobs use the memory again in further
    launches. What a call asks for evict's lists hangs on no job that it would refuse."""
    out = host("""
c = cache(nkv=8, slots=64, per=512)
verify, token, chunk = ([(s, 32000, n) for s in range(64)] for n in (8, 1, 600))
out = dict(one=[room(c, j[0], heads=64) for j in (verify, token, chunk)], all=[room(c, *j, heads=64) for j in (verify, token, chunk)])
hip.stand_in_reset(-1)
assert weigh(c, *verify, heads=64, o=f + (1 << 40), ws=f, n=1 << 40) == 0, why()     # nothing runs
out["launches"] = launched().count("k_weigh_page")
out["evict"] = [ctx.lib.cc_evict_workspace(C.byref(c), *jobs(j)) for j in ((0, 100, -5, 100), (0, 2**31 - 1, 2**31 - 2, 0), (0, 100, 0, 1))]
""")
    scores = 8 * 504 * 64 * 256
    assert out["one"][0] > scores and out["launches"] > 1
    assert all(n < (1 << 30) * 1.25 for n in out["all"]) and all(a >= b for a, b in zip(out["all"], out["one"]))
    assert out["evict"] == [0, 0, 0]

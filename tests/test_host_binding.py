"""The Python binding of the operators on device buffers, on the CPU: which GPU a
call's arrays are on. The HIP runtime is the stand-in of test_host_path.py with
two GPUs, each of whose allocations is known."""
import json
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

TWO_GPUS = """
#define hipSetDevice one_gpu_set
#define hipMalloc one_gpu_malloc
#define hipFree one_gpu_free
#include "hip_stand_in.cc"
#undef hipSetDevice
#undef hipMalloc
#undef hipFree
static int current = 0;
static std::map<void*, int> where;
extern "C" {
hipError_t hipGetDevice(int* d) { *d = current; return hipSuccess; }
hipError_t hipSetDevice(int d) {
    if (d < 0 || d > 1) return hipErrorInvalidDevice;
    current = d;
    return hipSuccess;
}
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) {
    const hipError_t e = one_gpu_malloc(p, n);
    where[*p] = current;
    return e;
}
hipError_t hipFree(void* p) {
    where.erase(p);
    return one_gpu_free(p);
}
int stand_in_gpu_of(void* p) { return where.count(p) ? where[p] : -1; }
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
hip.stand_in_gpu_of.argtypes = [C.c_void_p]
hip.hipMalloc.argtypes = [C.POINTER(C.c_void_p), C.c_size_t]
hip.hipFree.argtypes = [C.c_void_p]
hip.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
hip.hipGetDevice.argtypes = [C.POINTER(C.c_int)]
cc._hip = lambda: hip
ctx = [cc.Context(configs.with_layers(configs.SMOLLM2, 1), n_max=256, t_max=8, slots=2, device=g) for g in (0, 1)]
hip.hipSetDevice(0)
hip.stand_in_reset(-1)

def now():
    d = C.c_int()
    hip.hipGetDevice(C.byref(d))
    return d.value

def on(g, *shape, of=np.float32):
    hip.hipSetDevice(g)
    a = cc.DeviceArray.of(np.zeros(shape, of))
    hip.hipSetDevice(0)
    return a

def cache(*gpus, D=64, nkv=2, pages=4):
    shapes = [(pages, nkv, 64 * D + 128 * D // 16), (pages, nkv, 64 * D + 128 * D // 16), (2, pages), (64 * pages, D // 2, 2),
              (pages, nkv * (2 * D + D // 8))]
    k, v, t, r, b = (on(g, *s, of=of) for g, s, of in zip(gpus, shapes, (np.uint8, np.uint8, np.int32, np.float32, np.uint8)))
    return cc.KVCache(k, v, t, r, D, bounds=b)

def refused(call):
    hip.stand_in_reset(-1)
    try:
        call()
    except ValueError as e:
        return "GPU" in str(e) and hip.stand_in_launches() == b""
    return False
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("hip")
    so = str(d / "stand_in.so")
    (d / "stand_in.cc").write_text(TWO_GPUS)
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I",
                    os.path.join(ROCM, "include"), "-I", HERE, str(d / "stand_in.cc"), "-o", so], check=True)

    def run(code):
        r = subprocess.run([sys.executable, "-c", PRELUDE % (ROOT, so) + code + "\nprint(json.dumps(out))"], cwd=ROOT,
                           env=dict(os.environ, LD_PRELOAD=so), stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True,
                           timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
        return json.loads(r.stdout.splitlines()[-1])

    return run


def test_an_array_is_in_the_memory_of_its_gpu(host):
    """The one that is asked for or is current; the current one is as before after, also after copies."""
    out = host("""
out = []
hip.hipSetDevice(1)
a, b = cc.DeviceArray(5, np.float32), cc.DeviceArray((2, 3), np.int32, device=0)
c = cc.DeviceArray.of(np.arange(4, dtype=np.float32), device=0)
b.set(np.ones((2, 3)))
out.append([hip.stand_in_gpu_of(x.data_ptr()) for x in (a, b, c)] + [a.device, b.device, c.device, now()])
out.append(c.numpy().tolist() + b.numpy().tolist() + [now()])
try:
    cc.DeviceArray(5, np.float32, device=2)
except RuntimeError as e:
    out.append(str(e))
""")
    assert out == [[1, 0, 0, 1, 0, 0, 1], [0.0, 1.0, 2.0, 3.0, [1, 1, 1], [1, 1, 1], 1], "no GPU 2"]


def test_outputs_and_workspaces_are_on_the_contexts_gpu(host):
    """Whichever GPU is current: every allocation of a call."""
    out = host("""
out = []
real, made = cc.DeviceArray.__init__, []
def noted(self, *a, **kw):
    real(self, *a, **kw)
    made.append(hip.stand_in_gpu_of(self.data_ptr()))
for g in (0, 1):
    x, s = on(g, 2, 100), cc.Sampling(2, 100, temp=on(g, 2), u=on(g, 2, of=np.float64))
    c, q = cache(*[g] * 5), on(g, 1, 4 * 64)
    for current in (0, 1):
        hip.hipSetDevice(current)
        cc.DeviceArray.__init__ = noted
        got = [ctx[g].adjust_logits(x, s), *ctx[g].sample(x, s), ctx[g].attend_pages(c, [(0, 200, 1)], q, 3)]
        cc.DeviceArray.__init__ = real
        out.append([g, sorted(set(made)), sorted({a.device for a in got}), now() == current])
        made.clear()
""")
    assert out == [[g, [g], [g], True] for g in (0, 0, 1, 1)]


def test_arrays_of_another_gpu_are_refused(host):
    out = host("""
x, q, kv = [on(g, 2, 100) for g in (0, 1)], [on(g, 1, 256) for g in (0, 1)], [on(g, 1, 128) for g in (0, 1)]
s, c = [cc.Sampling(2, 100, temp=on(g, 2), u=on(g, 2, of=np.float64)) for g in (0, 1)], [cache(*[g] * 5) for g in (0, 1)]
own = cc.KVCache.of_context(ctx[1], 0)
job = [(0, 200, 1)]
calls = dict(
    logits=lambda: ctx[0].adjust_logits(x[1], s[0]), out=lambda: ctx[0].adjust_logits(x[0], s[0], out=x[1]),
    sampling=lambda: ctx[0].sample(x[0], s[1]), sample=lambda: ctx[1].sample(x[0], s[1]),
    cache=lambda: ctx[0].attend_pages(c[1], job, q[0], 3), q=lambda: ctx[0].attend_pages(c[0], job, q[1], 3),
    attended=lambda: ctx[0].attend_pages(c[0], job, q[0], 3, out=q[1]),
    k=lambda: ctx[0].kv_append(c[0], job, kv[1], kv[0]), v=lambda: ctx[0].kv_append(c[0], job, kv[0], kv[1]),
    bounds=lambda: ctx[0].kv_bounds(c[1], [(0, 0, 64)]), own=lambda: ctx[0].attend_pages(own, job, on(0, 1, 9 * 64), 4),
    mixed_cache=lambda: cache(0, 0, 1, 0, 0), mixed_bounds=lambda: cache(0, 0, 0, 0, 1),
    mixed_sampling=lambda: cc.Sampling(2, 100, temp=on(0, 2), u=on(1, 2, of=np.float64)),
    own_bounds=lambda: cc.KVCache.of_context(ctx[1], 0, bounds=on(0, own.c.n_pages, ctx[1].lib.cc_bounds_bytes(own.ref), of=np.uint8)))
out = [n for n, call in calls.items() if not refused(call)]
hip.stand_in_reset(-1)
for g in (0, 1):
    ctx[g].kv_append(c[g], [(0, 0, 1)], kv[g], kv[g])
    ctx[g].kv_bounds(c[g], [(0, 0, 64)])
out.append(hip.stand_in_launches().count(b"k_kv_append"))
""")
    assert out == [4]


TENSORS = """
class Tensor(cc.DeviceArray):      # stands for torch's: on GPU 0, contiguous
    requires_grad = False
    def get_device(self):
        return self.gpu
    def is_contiguous(self):
        return True
def tensor(*shape, of=np.float32, gpu=0):
    hip.hipSetDevice(0)
    t = Tensor(shape, of)
    t.gpu = gpu
    return t
cc._is_torch = lambda t: isinstance(t, Tensor)
def outcome(call):
    hip.stand_in_reset(-1)
    try:
        call()
    except (ValueError, RuntimeError) as e:
        return [str(e), hip.stand_in_launches().count(b"k_")]
    return ["", hip.stand_in_launches().count(b"k_")]
x, q, kv = on(0, 2, 100), on(0, 1, 256), on(0, 1, 128)
s, c, job = cc.Sampling(2, 100), cache(*[0] * 5), [(0, 70, 1)]
"""


def test_tensors_beside_other_arrays_need_a_stream(host):
    """The call's arrays are each ordered on the stream of their kind: a mixed call must say where it runs."""
    out = host(TENSORS + """
mixed = cc.Sampling(2, 100, temp=tensor(2), u=on(0, 2, of=np.float64))
c2 = cc.KVCache(*[a for a in c.kept[:4]], 64, bounds=tensor(*c.kept[4].shape, of=np.uint8))
calls = [lambda **kw: ctx[0].kv_append(c, job, kv, tensor(1, 128), **kw), lambda **kw: ctx[0].kv_append(c2, job, kv, kv, **kw),
         lambda **kw: ctx[0].attend_pages(c, job, q, 3, out=tensor(1, 256), **kw), lambda **kw: ctx[0].attend_pages(c2, job, q, 3, **kw),
         lambda **kw: ctx[0].adjust_logits(x, s, out=tensor(2, 100), **kw), lambda **kw: ctx[0].adjust_logits(x, mixed, **kw),
         lambda **kw: ctx[0].sample(x, mixed, **kw)]
out = [outcome(c) for c in calls] + [outcome(lambda: c(stream=0))[0] for c in calls]
""")
    assert all("stream must be given" in said and n == 0 for said, n in out[:7]), out
    assert out[7:] == [""] * 7


def test_tensors_on_the_cpu_are_refused_beside_device_arrays(host):
    out = host(TENSORS + """
cpu = lambda *a: tensor(*a, gpu=-1)
out = [outcome(c) for c in (lambda: ctx[0].kv_append(c, job, kv, cpu(1, 128), stream=0), lambda: ctx[0].kv_append(c, job, cpu(1, 128), kv),
                            lambda: ctx[0].attend_pages(c, job, q, 3, out=cpu(1, 256), stream=0),
                            lambda: ctx[0].adjust_logits(x, s, out=cpu(2, 100), stream=0), lambda: ctx[0].sample(cpu(2, 100), s))]
""")
    assert all("not on the context's GPU" in said and n == 0 for said, n in out), out


def test_gradients_do_not_end_silently(host):
    """A tensor that requires a gradient is refused in each place, except where gradients are off."""
    out = host(TENSORS + """
import types
grad = [True]
sys.modules["torch"] = types.SimpleNamespace(is_grad_enabled=lambda: grad[0])
def learnt(*a, **kw):
    t = tensor(*a, **kw)
    t.requires_grad = True
    return t
calls = [lambda: ctx[0].kv_append(c, job, learnt(1, 128), kv), lambda: ctx[0].kv_append(c, job, kv, learnt(1, 128), stream=0),
         lambda: ctx[0].attend_pages(c, job, learnt(1, 256), 3), lambda: ctx[0].attend_pages(c, job, q, 3, out=learnt(1, 256), stream=0),
         lambda: ctx[0].adjust_logits(learnt(2, 100), s), lambda: ctx[0].adjust_logits(x, s, out=learnt(2, 100), stream=0),
         lambda: ctx[0].sample(learnt(2, 100), s), lambda: cc.Sampling(2, 100, temp=learnt(2))]
out = [outcome(c) for c in calls]
grad[0] = False
out += [outcome(c) for c in (calls[1], calls[3], calls[5], calls[7])]
""")
    assert all("gradient" in said and n == 0 for said, n in out[:8]), out
    assert all(said == "" for said, n in out[8:]), out


def test_wishes_that_are_no_32_bit_numbers(host):
    """What does not fit is refused, not wrapped or cut; what fits keeps its bits."""
    out = host("""
bad = [("top_k", np.array([2**32 + 5])), ("top_k", [1.5]), ("top_k", [np.nan]), ("pen_at", [0, 2**31]), ("pen_ids", np.array([-2**40])),
       ("mask_of", [np.inf]), ("bias_ids", np.array([2**63], np.uint64)), ("mask", np.array([[2**32]])), ("mask", [[0.5]])]
out = []
for name, a in bad:
    try:
        cc._HostArray(name, a)
        out.append([name, str(a)])
    except ValueError as e:
        out += [] if name in str(e) else [str(e)]
good = [("top_k", [3.0, -2**31, 2**31 - 1]), ("mask", np.array([[-1, 7]], np.int32)), ("mask", np.array([[2**32 - 1, 0]])), ("pen_ids", []),
        ("mask", np.zeros((1, 2))), ("top_k", np.array([1, 2], np.uint8)), ("temp", [1, 0.5]), ("u", [0.1]), ("mask_of", [True])]
out += [[a.tolist(), str(a.dtype)] for a in (cc._HostArray(n, v).a for n, v in good)]
""")
    assert out == [[[3, -2**31, 2**31 - 1], "int32"], [[[2**32 - 1, 7]], "uint32"], [[[2**32 - 1, 0]], "uint32"], [[], "int32"],
                   [[[0, 0]], "uint32"], [[1, 2], "int32"], [[1.0, 0.5], "float32"], [[0.1], "float64"], [[1], "int32"]]

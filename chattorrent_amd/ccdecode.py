"""ctypes binding of the C ABI (include/ccdecode.h) of libccdecode.so.

This is the Python host over the MI355X library: the tests and bench.py use
it; the JS Runner shim (node/runner.js) uses the N-API addon over the same
ABI. There is no CPU fallback: if the HIP library is missing, loading fails.
"""
import ctypes as C
import os
import sys

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libccdecode.so")

CC_OK, CC_BUSY, CC_COLD, CC_STALE, CC_NOSPEC, CC_EARG, CC_EPOOL, CC_EOOM, CC_EDEVICE = range(9)
STATUS_NAMES = ["ok", "busy", "cold", "stale", "nospec", "bad-job", "pool-too-small", "out-of-memory",
                "device"]
(T_Q, T_K, T_V, T_O, T_GATE, T_UP, T_DOWN, T_LN1, T_LN2, T_WTE, T_NORM, T_LM_HEAD) = range(12)
# a hybrid checkpoint's full_attention extras and linear_attention tensors
(T_ATTN_GATE, T_Q_NORM, T_K_NORM, T_IN_Q, T_IN_K, T_IN_V, T_IN_Z, T_IN_B, T_IN_A, T_CONV_Q, T_CONV_K, T_CONV_V,
 T_GATE_PARAMS, T_GATED_NORM, T_OUT_PROJ) = range(12, 27)
# the MTP draft head; its block's tensors are the block ids at LAYER_MTP
(T_MTP_ENORM, T_MTP_HNORM, T_MTP_FC_E, T_MTP_FC_H, T_MTP_NORM, T_MTP_EMBED, T_MTP_HEAD) = range(27, 34)
LAYER_MTP = -2
FULL_ATTENTION, LINEAR_ATTENTION = 0, 1
EXPORTS = [
    "cc_create", "cc_destroy", "cc_last_error", "cc_upload", "cc_fill_random", "cc_step", "cc_release",
    "cc_slot_pages", "cc_free_pages", "cc_fill_random_kv", "cc_read_kv", "cc_write_kv", "cc_read_pages",
    "cc_stats_get", "cc_op_matmul_q8", "cc_op_store_kv", "cc_op_round_f16", "cc_op_topk", "cc_op_rmsnorm",
    "cc_op_attend", "cc_profile", "cc_profile_read", "cc_read_logits", "cc_mtp_draft", "cc_topk_noalloc",
    "cc_decode_steps", "cc_cache_of", "cc_bounds_bytes", "cc_kv_append", "cc_kv_bounds", "cc_attend_workspace",
    "cc_attend_pages", "cc_logits_adjust", "cc_sample_workspace", "cc_sample", "cc_sample_pass",
]


class Dims(C.Structure):
    _fields_ = [("hidden", C.c_int32), ("n_layer", C.c_int32), ("n_heads", C.c_int32),
                ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32), ("ffn", C.c_int32), ("vocab", C.c_int32),
                ("q8_group", C.c_int32), ("rms_eps", C.c_float), ("rope_theta", C.c_double),
                ("rope_scaling", C.c_int32), ("rs_factor", C.c_double), ("rs_low_freq", C.c_double),
                ("rs_high_freq", C.c_double), ("rs_orig_max_pos", C.c_double), ("tied", C.c_int32),
                ("rot_dim", C.c_int32), ("hybrid", C.c_int32), ("layer_kinds", C.POINTER(C.c_uint8)),
                ("lin_nk", C.c_int32), ("lin_nv", C.c_int32), ("lin_dk", C.c_int32), ("lin_dv", C.c_int32),
                ("lin_conv", C.c_int32), ("mtp_vocab", C.c_int32)]


class Opts(C.Structure):
    _fields_ = [("lo", C.c_int32), ("hi", C.c_int32), ("n_max", C.c_int32), ("t_max", C.c_int32),
                ("slots", C.c_int32), ("sessions", C.c_int32), ("page_tokens", C.c_int32),
                ("max_jobs", C.c_int32), ("device", C.c_int32)]


class Job(C.Structure):
    _fields_ = [("slot", C.c_int32), ("past", C.c_int32), ("n", C.c_int32), ("sampled", C.c_int32),
                ("ids", C.POINTER(C.c_int32)), ("hidden", C.POINTER(C.c_uint16)), ("snap", C.c_int32),
                ("rollback", C.c_int32), ("keep", C.c_int32), ("mtp", C.c_int32)]


class Stats(C.Structure):
    _fields_ = [("vram_bytes", C.c_uint64), ("weight_bytes", C.c_uint64), ("kv_bytes", C.c_uint64),
                ("scratch_bytes", C.c_uint64), ("passes", C.c_int64), ("rows", C.c_int64),
                ("last_pass_ms", C.c_double)]


class CCache(C.Structure):
    """cc_cache: a paged int8 cache in device memory (KVCache builds it)."""
    _fields_ = [("n_kv_heads", C.c_int32), ("head_dim", C.c_int32), ("rot_dim", C.c_int32), ("n_pages", C.c_int32),
                ("max_pages", C.c_int32), ("slots", C.c_int32), ("rope_rows", C.c_int32), ("k", C.c_void_p),
                ("v", C.c_void_p), ("bounds", C.c_void_p), ("page_table", C.c_void_p), ("rope", C.c_void_p)]


class CSampling(C.Structure):
    """cc_sampling: what each row of a call asks for (Sampling builds it)."""
    _fields_ = [("temp", C.c_void_p), ("top_k", C.c_void_p), ("top_p", C.c_void_p), ("min_p", C.c_void_p),
                ("rep", C.c_void_p), ("freq", C.c_void_p), ("pres", C.c_void_p), ("freq_cap", C.c_float),
                ("pen_at", C.c_void_p), ("pen_ids", C.c_void_p), ("pen_counts", C.c_void_p), ("n_pen", C.c_int32),
                ("bias_at", C.c_void_p), ("bias_ids", C.c_void_p), ("bias", C.c_void_p), ("n_bias", C.c_int32),
                ("mask", C.c_void_p), ("mask_words", C.c_int32), ("n_masks", C.c_int32), ("mask_of", C.c_void_p),
                ("u", C.c_void_p)]


_lib = None
_torch_first = False   # torch was there when the library was loaded: they share one HIP runtime


def load():
    """Loads libccdecode.so; raises if it is not built (no fallback)."""
    global _lib, _torch_first
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is missing: build it with `python -m chattorrent_amd.build`")
    _torch_first = "torch" in sys.modules
    L = C.CDLL(LIB_PATH)
    P = C.c_void_p
    i32, i64, u64, size = C.c_int32, C.c_int64, C.c_uint64, C.c_size_t
    sig = {
        "cc_create": (i32, [C.POINTER(Dims), C.POINTER(Opts), C.POINTER(P)]),
        "cc_destroy": (None, [P]),
        "cc_last_error": (C.c_char_p, [P]),
        "cc_upload": (i32, [P, i32, i32, P, C.c_size_t, P, C.c_size_t, i32, i32]),
        "cc_fill_random": (i32, [P, u64]),
        "cc_step": (i32, [P, C.POINTER(Job), i32, i32, i32, i32, P, P, P, P]),
        "cc_release": (i32, [P, i32]),
        "cc_slot_pages": (i32, [P, i32]),
        "cc_free_pages": (i32, [P]),
        "cc_fill_random_kv": (i32, [P, i32, i32, u64, u64]),
        "cc_read_kv": (i32, [P, i32, i32, i32, i32, i32, i32, P]),
        "cc_write_kv": (i32, [P, i32, i32, i32, i32, i32, i32, P]),
        "cc_read_pages": (i32, [P, i32, P, i32]),
        "cc_stats_get": (i32, [P, C.POINTER(Stats)]),
        "cc_op_matmul_q8": (i32, [P, P, i32, i32, P, P, i32, P]),
        "cc_op_store_kv": (i32, [P, i32, i32, i32, P, i32, i32]),
        "cc_op_round_f16": (i32, [P, P, i64]),
        "cc_op_topk": (i32, [P, P, i32, i32, i32, P, P]),
        "cc_op_rmsnorm": (i32, [P, P, P, i32, i32, P]),
        "cc_op_attend": (i32, [P, i32, i32, P, i32, i32, P]),
        "cc_read_logits": (i32, [P, i32, P]),
        "cc_mtp_draft": (i32, [P, i32, i32, i32, i32, i32, P]),
        "cc_decode_steps": (i32, [P, C.POINTER(Job), i32, i32, i32, P, P]),
        "cc_cache_of": (i32, [P, i32, C.POINTER(CCache)]),
        "cc_bounds_bytes": (size, [C.POINTER(CCache)]),
        "cc_kv_append": (i32, [P, P, P, i32, P, i64, P, i64, P]),
        "cc_kv_bounds": (i32, [P, P, P, i32, P]),
        "cc_attend_workspace": (size, [P, P, i32, i32, i32]),
        "cc_attend_pages": (i32, [P, P, P, i32, i32, i32, i32, i32, P, i64, P, i64, P, size, P]),
        "cc_logits_adjust": (i32, [P, P, i64, i32, i32, P, P, i64, P]),
        "cc_sample_workspace": (size, [i32, i32, P]),
        "cc_sample": (i32, [P, P, i64, i32, i32, P, P, P, P, size, P]),
        "cc_sample_pass": (i32, [P, i32, P, P, P]),
        "cc_profile": (i32, [P, i32]),
        "cc_profile_read": (i32, [P, i32, C.POINTER(C.c_double), C.POINTER(C.c_int64), C.POINTER(C.c_double)]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


def _p(a):
    return a.ctypes.data_as(C.c_void_p)


class CCError(RuntimeError):
    """A failed call; `.status` is the cc_status, `.kind` its name."""

    def __init__(self, status, msg):
        super().__init__(msg)
        self.status = status
        self.kind = STATUS_NAMES[status] if 0 <= status < len(STATUS_NAMES) else str(status)


# --- device buffers: the operators on the caller's own memory -------------------------
# They take torch tensors or DeviceArrays. A call whose k, q or logits are torch's runs on torch's current stream, else on the
# context's; where a call on the one reads what a call on the other wrote, the caller orders them, or gives both one stream.

def _hip():
    """The HIP runtime that the library itself uses."""
    load()
    h = C.CDLL("libamdhip64.so.7")
    h.hipMalloc.argtypes = [C.POINTER(C.c_void_p), C.c_size_t]
    h.hipFree.argtypes = [C.c_void_p]
    h.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
    h.hipGetDevice.argtypes = [C.POINTER(C.c_int)]
    return h


class _Gpu:
    """GPU `device` is the thread's current one within; None: the one that is, as `device`."""

    def __init__(self, h, device=None):
        self.h, self.device = h, device

    def __enter__(self):
        now = C.c_int()
        if self.h.hipGetDevice(C.byref(now)):
            raise RuntimeError("no current GPU")
        if self.device is None:
            self.device = now.value
        self.before = now.value
        if self.before != self.device and self.h.hipSetDevice(self.device):
            raise RuntimeError(f"no GPU {self.device}")
        return self

    def __exit__(self, *exc):
        if self.before != self.device:
            self.h.hipSetDevice(self.before)


class DeviceArray:
    """A C-contiguous array in the memory of one GPU (`device`; None: the
    thread's current one), for callers without torch."""

    def __init__(self, shape, dtype, device=None):
        self.shape, self.dtype = tuple(int(n) for n in np.atleast_1d(shape)), np.dtype(dtype)
        self.nbytes = int(np.prod(self.shape)) * self.dtype.itemsize
        self._h, p = _hip(), C.c_void_p()
        with _Gpu(self._h, device) as gpu:
            self.device = gpu.device
            if self._h.hipMalloc(C.byref(p), max(self.nbytes, 16)):
                raise MemoryError(f"no device memory for {self.nbytes} bytes")
        self._p = p.value

    @classmethod
    def of(cls, a, device=None):
        """A copy of a numpy array on the device."""
        a = np.ascontiguousarray(a)
        out = cls(a.shape, a.dtype, device)
        out.set(a)
        return out

    def set(self, a):
        a = np.ascontiguousarray(a, self.dtype)
        if a.shape != self.shape:
            raise ValueError(f"shape {a.shape}, not {self.shape}")
        self._copy(self._p, a.ctypes.data, 1)

    def numpy(self):
        """A copy on the host, once everything on the device is done."""
        out = np.empty(self.shape, self.dtype)
        self._copy(out.ctypes.data, self._p, 2)
        return out

    def _copy(self, to, of, kind):
        with _Gpu(self._h, self.device):
            if self._h.hipDeviceSynchronize() or (self.nbytes and self._h.hipMemcpy(to, of, self.nbytes, kind)):
                raise RuntimeError("a copy between host and device failed")

    def data_ptr(self):
        return self._p

    def stride(self, dim):
        return int(np.prod(self.shape[dim:][1:])) if dim >= 0 else self.stride(dim + len(self.shape))

    def __del__(self):
        if getattr(self, "_p", None):
            self._h.hipFree(self._p)
            self._p = None


def _is_torch(t):
    torch = sys.modules.get("torch")
    return torch is not None and isinstance(t, torch.Tensor)


def _gpu_of(t):
    """The GPU whose memory t is in (-1: a CPU tensor's); None where it does not say."""
    return t.get_device() if _is_torch(t) else getattr(t, "device", None)


def _no_gradient(t):
    """Refuses a tensor whose gradient would end at a call: the operators have no backward pass."""
    if t.requires_grad and sys.modules["torch"].is_grad_enabled():
        raise ValueError("a tensor that requires a gradient: none passes through a call (detach it, or call under no_grad)")


_dtypes = {}   # a dtype object's name


def _dtype(t):
    d = t.dtype
    name = _dtypes.get(d)
    if name is None:
        name = _dtypes[d] = str(d).rsplit(".", 1)[-1]
    return name


class _Buffers:
    """Buffers that one C struct points into: checked, kept alive, on one device."""

    def __init__(self):
        self.kept, self.device, self.torch = [], None, False

    def take(self, t, name, dtypes, shape, nullable=True):
        """The pointer of a contiguous device array of one of `dtypes` and of `shape` (None: any extent)."""
        if t is None and nullable:
            return None
        if _dtype(t) not in dtypes:
            raise ValueError(f"{name}: {' or '.join(dtypes)}, not {t.dtype}")
        have = tuple(t.shape)
        if have != shape and (len(have) != len(shape) or any(w is not None and n != w for n, w in zip(have, shape))):
            raise ValueError(f"{name}: shape {have}, not {shape}")
        device = _gpu_of(t)
        if device is not None:
            if device < 0 or (_is_torch(t) and not t.is_contiguous()):
                raise ValueError(f"{name}: a contiguous tensor on the GPU")
            if self.device is not None and device != self.device:
                raise ValueError(f"{name}: on another GPU than the others")
            self.device = device
        if _is_torch(t):
            _no_gradient(t)
            self.torch = True
        self.kept.append(t)
        return t.data_ptr()


class _HostArray:
    """A wish of cc_sample_pass, in host memory and in the type that Sampling
    takes; whole numbers as they are given, or refused (a mask's words may be
    signed or not)."""

    def __init__(self, name, a):
        kind = {"u": np.float64, "mask": np.uint32}.get(name, np.float32)
        if name in ("top_k", "pen_at", "pen_ids", "pen_counts", "bias_at", "bias_ids", "mask_of"):
            kind = np.int32
        given = np.asarray(a)
        if kind in (np.int32, np.uint32) and given.size:
            low, high = np.min(given), np.max(given)      # NaN: in neither's range
            if not (low >= -2**31 and high < (2**31 if kind is np.int32 else 2**32) and (given == np.trunc(given)).all()):
                raise ValueError(f"{name}: whole numbers of 32 bits")
            if kind is np.uint32:
                given = given.astype(np.int64)
        self.a = np.ascontiguousarray(given, kind)
        self.shape, self.dtype = self.a.shape, self.a.dtype

    def data_ptr(self):
        return self.a.ctypes.data


class KVCache(_Buffers):
    """A paged int8 cache in the caller's device memory, K and V of one layer,
    laid out as include/ccdecode.h says (cc_cache): k, v uint8 [pages, kv heads,
    64*D + 64*D/32*4], page_table int32 [slots, pages a slot], rope f32
    [positions, rot_dim/2, 2], and key bounds uint8 [pages, kv heads*(2*D +
    D/8)] or None. KVCache.of_context gives a context's own."""

    def __init__(self, k, v, page_table, rope, head_dim, bounds=None):
        super().__init__()
        D = int(head_dim)
        n_pages, n_kv = int(k.shape[0]), int(k.shape[1])
        block = 64 * D + 64 * (D // 32) * 4
        self.c = CCache(n_kv_heads=n_kv, head_dim=D, rot_dim=2 * int(rope.shape[1]), n_pages=n_pages,
                        max_pages=int(page_table.shape[1]), slots=int(page_table.shape[0]),
                        rope_rows=int(rope.shape[0]),
                        k=self.take(k, "k", ("uint8", "int8"), (n_pages, n_kv, block), False),
                        v=self.take(v, "v", ("uint8", "int8"), (n_pages, n_kv, block), False),
                        page_table=self.take(page_table, "page_table", ("int32", "uint32"), (None, None), False),
                        rope=self.take(rope, "rope", ("float32",), (None, None, 2), False),
                        bounds=self.take(bounds, "bounds", ("uint8", "int8"), (n_pages, n_kv * (2 * D + D // 8))))
        self._done()

    def _done(self):
        """What every call on the cache needs of it: its struct, the width of a row, workspaces' sizes as they come up."""
        self.ref, self.width, self.workspace = C.byref(self.c), self.c.n_kv_heads * self.c.head_dim, {}

    @classmethod
    def of_context(cls, ctx, layer, bounds=None):
        """The context's own cache of block `layer`; `bounds`: key bounds of the caller's."""
        self = cls.__new__(cls)
        _Buffers.__init__(self)
        self.c = CCache()
        ctx._chk(ctx.lib.cc_cache_of(ctx.h, layer, C.byref(self.c)))
        self.kept.append(ctx)
        self.device = ctx.opts.device
        self.c.bounds = self.take(bounds, "bounds", ("uint8", "int8"),
                                  (self.c.n_pages, int(ctx.lib.cc_bounds_bytes(C.byref(self.c)))))
        self._done()
        return self


class Sampling(_Buffers):
    """What the rows of a call ask for (cc_sampling): device arrays, None where
    no row asks for it. temp, top_p, min_p, rep, freq, pres f32 [rows]; top_k
    int32 [rows]; u f64 [rows]; the history pen_at int32 [rows + 1], pen_ids
    int32 [entries], pen_counts int32 [entries] or None (1 each); bias_at,
    bias_ids likewise and bias f32 [entries]; mask 32-bit words [masks,
    ceil(vocab/32) or more] and mask_of int32 [rows]."""

    def __init__(self, rows, vocab, temp=None, top_k=None, top_p=None, min_p=None, rep=None, freq=None, pres=None,
                 freq_cap=1.5, pen_at=None, pen_ids=None, pen_counts=None, bias_at=None, bias_ids=None, bias=None,
                 mask=None, mask_of=None, u=None):
        super().__init__()
        self.rows, self.vocab = int(rows), int(vocab)
        n_pen = 0 if pen_ids is None else int(pen_ids.shape[0])
        n_bias = 0 if bias_ids is None else int(bias_ids.shape[0])
        f32, i32, row = ("float32",), ("int32", "uint32"), (self.rows,)
        if mask is not None and int(mask.shape[1]) * 32 < self.vocab:
            raise ValueError(f"mask: {mask.shape[1]} words are fewer than the vocabulary takes")
        self.c = CSampling(
            temp=self.take(temp, "temp", f32, row), top_k=self.take(top_k, "top_k", i32, row),
            top_p=self.take(top_p, "top_p", f32, row), min_p=self.take(min_p, "min_p", f32, row),
            rep=self.take(rep, "rep", f32, row), freq=self.take(freq, "freq", f32, row),
            pres=self.take(pres, "pres", f32, row), freq_cap=freq_cap,
            pen_at=self.take(pen_at, "pen_at", i32, (self.rows + 1,)),
            pen_ids=self.take(pen_ids, "pen_ids", i32, (n_pen,)),
            pen_counts=self.take(pen_counts, "pen_counts", i32, (n_pen,)), n_pen=n_pen,
            bias_at=self.take(bias_at, "bias_at", i32, (self.rows + 1,)),
            bias_ids=self.take(bias_ids, "bias_ids", i32, (n_bias,)),
            bias=self.take(bias, "bias", f32, (n_bias,)), n_bias=n_bias,
            mask=self.take(mask, "mask", i32, (None, None)), mask_words=0 if mask is None else int(mask.shape[1]),
            n_masks=0 if mask is None else int(mask.shape[0]), mask_of=self.take(mask_of, "mask_of", i32, row),
            u=self.take(u, "u", ("float64",), row))
        self.ref, self.workspace = C.byref(self.c), None


def _job_rows(jobs):
    """(slot, past, n) of each job as int32 [jobs, 3], its address, and the rows they hold."""
    a = np.asarray(jobs)
    if a.dtype != np.int32:
        if a.size and (a.dtype.kind not in "iu" or a.min() < -2**31 or a.max() >= 2**31):
            raise ValueError("jobs: 32-bit integers (slot, past, n)")
        a = a.astype(np.int32)
    if a.ndim != 2 or a.shape[1] != 3:
        raise ValueError("jobs: one (slot, past, n) each")
    if not a.flags.c_contiguous:
        a = np.ascontiguousarray(a)
    n = len(a)
    rows = int(a[0, 2]) if n == 1 else int(np.add.reduce(a[:, 2], dtype=np.int64))
    return a, a.__array_interface__["data"][0], n, rows


def layer_kinds(d):
    """Block kinds from `layer_types` (the manifest's strings), or None (all full)."""
    lt = d.get("layer_types")
    if not lt:
        return None
    return [LINEAR_ATTENTION if t == "linear_attention" else FULL_ATTENTION for t in lt]


def make_dims(d):
    sc = d.get("rope_scaling")
    dims = Dims(hidden=d["hidden"], n_layer=d["n_layer"], n_heads=d["n_heads"], n_kv_heads=d["n_kv_heads"],
                head_dim=d["head_dim"], ffn=d["ffn"], vocab=d["vocab"], q8_group=d.get("group_q8", 32),
                rms_eps=d["rms_eps"], rope_theta=d["rope_theta"], rope_scaling=1 if sc else 0,
                rs_factor=sc["factor"] if sc else 0.0, rs_low_freq=sc["low_freq_factor"] if sc else 0.0,
                rs_high_freq=sc["high_freq_factor"] if sc else 0.0,
                rs_orig_max_pos=sc["original_max_position_embeddings"] if sc else 0.0,
                tied=1 if d.get("tied", True) else 0, rot_dim=d.get("rot_dim", 0) or 0,
                hybrid=1 if d.get("hybrid") else 0, lin_nk=d.get("lin_nk", 0), lin_nv=d.get("lin_nv", 0),
                lin_dk=d.get("lin_dk", 0), lin_dv=d.get("lin_dv", 0), lin_conv=d.get("lin_conv", 0),
                mtp_vocab=d.get("mtp_vocab", 0) or 0)
    kinds = layer_kinds(d)
    if kinds is not None:
        arr = (C.c_uint8 * len(kinds))(*kinds)
        dims._kinds = arr   # kept alive with the struct; cc_create copies it
        dims.layer_kinds = C.cast(arr, C.POINTER(C.c_uint8))
    return dims


class Context:
    """One cc_ctx: a Runner's GPU half over positions [lo, hi)."""

    def __init__(self, d, n_max, t_max, slots, sessions=None, max_jobs=None, lo=0, hi=None, device=0):
        self.lib = load()
        self.d = dict(d)
        positions = d["n_layer"] + 2
        self.opts = Opts(lo=lo, hi=positions if hi is None else hi, n_max=n_max, t_max=t_max, slots=slots,
                         sessions=sessions or slots, page_tokens=64, max_jobs=max_jobs or (sessions or slots),
                         device=device)
        dims = make_dims(d)
        h = C.c_void_p()
        st = self.lib.cc_create(C.byref(dims), C.byref(self.opts), C.byref(h))
        self.h = h
        if st != CC_OK:
            msg = self.lib.cc_last_error(h).decode() if h else "cc_create failed"
            if h:
                self.lib.cc_destroy(h)
            self.h = None
            raise CCError(st, msg)

    def close(self):
        if self.h:
            self.lib.cc_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _chk(self, st):
        if st != CC_OK:
            raise CCError(st, self.lib.cc_last_error(self.h).decode())

    # --- weights ---------------------------------------------------------------
    def fill_random(self, seed):
        self._chk(self.lib.cc_fill_random(self.h, seed))

    def upload_q8(self, layer, tensor, codes, scales, group=32):
        """int8 codes [N, K] and scales [N, ceil(K/group)]: uint16 arrays are
        f16 bits, float32 arrays are f32 (rounded to f16 on the device side)."""
        codes = np.ascontiguousarray(codes, np.int8)
        if np.asarray(scales).dtype == np.float32:
            sc, kind = np.ascontiguousarray(scales, np.float32), 1
        else:
            sc, kind = np.ascontiguousarray(scales, np.uint16), 0
        self._chk(self.lib.cc_upload(self.h, layer, tensor, _p(codes), codes.size, _p(sc), sc.size, kind,
                                     int(group)))

    def upload_norm(self, layer, tensor, w):
        """An f32 tensor: a norm weight, or a hybrid block's q_norm, k_norm,
        conv1d_q/k/v ([channels, 4]), gate_params or gated_norm."""
        w = np.ascontiguousarray(w, np.float32)
        self._chk(self.lib.cc_upload(self.h, layer, tensor, _p(w), w.size, None, 0, 0, 32))

    # --- KV / pages --------------------------------------------------------------
    def fill_random_kv(self, slot, tokens, seed, key):
        self._chk(self.lib.cc_fill_random_kv(self.h, slot, tokens, seed, key))

    def read_kv(self, layer, which, slot, head, t0, t1):
        D = self.d["head_dim"]
        out = np.empty((t1 - t0, D // 4 + D // 32), np.uint32)
        self._chk(self.lib.cc_read_kv(self.h, layer, which, slot, head, t0, t1, _p(out)))
        return out

    def write_kv(self, layer, which, slot, head, t0, rows):
        rows = np.ascontiguousarray(rows, np.uint32)
        self._chk(self.lib.cc_write_kv(self.h, layer, which, slot, head, t0, t0 + rows.shape[0], _p(rows)))

    def pages(self, slot):
        n = self.lib.cc_slot_pages(self.h, slot)
        out = np.empty(max(n, 1), np.uint32)
        self._chk(self.lib.cc_read_pages(self.h, slot, _p(out), n))
        return out[:n]

    def read_logits(self, rows):
        out = np.empty((rows, self.d["vocab"]), np.float32)
        self._chk(self.lib.cc_read_logits(self.h, rows, _p(out)))
        return out

    def free_pages(self):
        return self.lib.cc_free_pages(self.h)

    def mtp_draft(self, slot, row, token, pos, k):
        """cc_mtp_draft: keep row `row` of the last pass (-1: the kept one) and
        chain `k` drafts after `token` at positions pos.. (uint32 [k])."""
        out = np.zeros(max(k, 1), np.uint32)
        self._chk(self.lib.cc_mtp_draft(self.h, slot, row, token, pos, k, _p(out)))
        return out[:k]

    def release(self, slot):
        self._chk(self.lib.cc_release(self.h, slot))

    def stats(self):
        s = Stats()
        self._chk(self.lib.cc_stats_get(self.h, C.byref(s)))
        return {k: getattr(s, k) for k, _ in Stats._fields_}

    KINDS = ("qkv", "o", "gate_up", "down", "head", "attn")

    def profile(self, enable=True):
        self._chk(self.lib.cc_profile(self.h, 1 if enable else 0))

    def profile_read(self):
        """{kind: (ms_total, launches, algorithmic_bytes)} since profile(True)."""
        out = {}
        for k, name in enumerate(self.KINDS):
            ms, n, b = C.c_double(), C.c_int64(), C.c_double()
            self._chk(self.lib.cc_profile_read(self.h, k, C.byref(ms), C.byref(n), C.byref(b)))
            out[name] = (ms.value, n.value, b.value)
        return out

    # --- the pass -----------------------------------------------------------------
    def step(self, jobs, at=0, to=None, topk=1):
        """jobs: dicts with slot, past, n, sampled and ids (or hidden f16 bits
        [n, H]), optionally snap (a verify) and keep (a rollback). Returns (vals [S, topk], ids [S, topk]) at the head, else the
        f16 bits of every row [T, H]. Raises CCError; `.statuses` holds the
        per-job statuses."""
        positions = self.d["n_layer"] + 2
        to = positions if to is None else to
        arr = (Job * len(jobs))()
        keep = []
        T = S = 0
        for i, j in enumerate(jobs):
            arr[i].slot, arr[i].past, arr[i].n = j["slot"], j["past"], j["n"]
            arr[i].sampled = j.get("sampled", 1 if to == positions else 0)
            if j.get("ids") is not None:
                a = np.ascontiguousarray(j["ids"], np.int32)
                keep.append(a)
                arr[i].ids = a.ctypes.data_as(C.POINTER(C.c_int32))
            if j.get("hidden") is not None:
                a = np.ascontiguousarray(j["hidden"], np.uint16)
                keep.append(a)
                arr[i].hidden = a.ctypes.data_as(C.POINTER(C.c_uint16))
            # speculation through linear_attention blocks: `snap` marks a
            # verify, `keep` (not None) rolls back to before the last verify
            arr[i].snap = 1 if j.get("snap") else 0
            arr[i].mtp = 1 if j.get("mtp") else 0
            if j.get("keep") is not None:
                arr[i].rollback, arr[i].keep = 1, int(j["keep"])
            T += j["n"]
            S += arr[i].sampled
        status = np.zeros(len(jobs), np.int32)
        if to == positions:
            vals = np.empty((max(S, 1), topk), np.float32)
            ids = np.empty((max(S, 1), topk), np.uint32)
            st = self.lib.cc_step(self.h, arr, len(jobs), at, to, topk, _p(vals), _p(ids), None, _p(status))
            if st != CC_OK:
                e = CCError(st, self.lib.cc_last_error(self.h).decode())
                e.statuses = status
                raise e
            return vals[:S], ids[:S]
        hid = np.empty((T, self.d["hidden"]), np.uint16)
        st = self.lib.cc_step(self.h, arr, len(jobs), at, to, 0, None, None, _p(hid), _p(status))
        if st != CC_OK:
            e = CCError(st, self.lib.cc_last_error(self.h).decode())
            e.statuses = status
            raise e
        return hid

    def decode_steps(self, slots, pasts, ids, steps, topk=1):
        """cc_decode_steps: `steps` greedy passes on the device for one-row
        jobs (slot, past, first id); returns (vals, ids) [steps, jobs, topk]."""
        n = len(slots)
        arr = (Job * n)()
        keep = []
        for i in range(n):
            a = np.array([int(ids[i])], np.int32)
            keep.append(a)
            arr[i].slot, arr[i].past, arr[i].n, arr[i].sampled = int(slots[i]), int(pasts[i]), 1, 1
            arr[i].ids = a.ctypes.data_as(C.POINTER(C.c_int32))
        vals = np.empty((steps, n, topk), np.float32)
        out = np.empty((steps, n, topk), np.uint32)
        self._chk(self.lib.cc_decode_steps(self.h, arr, n, steps, topk, _p(vals), _p(out)))
        return vals, out

    # --- kernel-level ops (parity tests) ---------------------------------------------
    def op_matmul_q8(self, X, W, scales_f16):
        X = np.ascontiguousarray(X, np.float32)
        W = np.ascontiguousarray(W, np.int8)
        S = np.ascontiguousarray(scales_f16, np.uint16)
        M, K = X.shape
        N = W.shape[0]
        Y = np.empty((M, N), np.float32)
        self._chk(self.lib.cc_op_matmul_q8(self.h, _p(X), M, K, _p(W), _p(S), N, _p(Y)))
        return Y

    def op_store_kv(self, layer, which, slot, src, past):
        src = np.ascontiguousarray(src, np.float32)
        self._chk(self.lib.cc_op_store_kv(self.h, layer, which, slot, _p(src), src.shape[0], past))

    def op_round_f16(self, a):
        a = np.array(a, dtype=np.float32, copy=True)
        self._chk(self.lib.cc_op_round_f16(self.h, _p(a), a.size))
        return a

    def op_topk(self, logits, M):
        logits = np.ascontiguousarray(logits, np.float32)
        rows, V = logits.shape
        vals = np.empty((rows, M), np.float32)
        ids = np.empty((rows, M), np.uint32)
        self._chk(self.lib.cc_op_topk(self.h, _p(logits), rows, V, M, _p(vals), _p(ids)))
        return vals, ids

    def op_rmsnorm(self, x, w):
        x = np.ascontiguousarray(x, np.float32)
        w = np.ascontiguousarray(w, np.float32)
        T, H = x.shape
        y = np.empty_like(x)
        self._chk(self.lib.cc_op_rmsnorm(self.h, _p(x), _p(w), T, H, _p(y)))
        return y

    def op_attend(self, layer, slot, q, past):
        q = np.ascontiguousarray(q, np.float32)
        out = np.empty_like(q)
        self._chk(self.lib.cc_op_attend(self.h, layer, slot, _p(q), q.shape[0], past, _p(out)))
        return out

    def sample_pass(self, rows, **wishes):
        """cc_sample_pass: a token of each of the last pass's `rows` sampled rows
        and its probability, drawn on the device. The wishes are Sampling's, in
        host memory (numpy arrays, lists)."""
        s = Sampling(rows, self.d["vocab"], **{n: a if a is None or n == "freq_cap" else _HostArray(n, a)
                                               for n, a in wishes.items()})
        ids, probs = np.empty(rows, np.int32), np.empty(rows, np.float32)
        self._chk(self.lib.cc_sample_pass(self.h, rows, s.ref, _p(ids), _p(probs)))
        return ids, probs

    # --- operators on the caller's device buffers --------------------------------------
    def _on(self, stream, held, t, out=None):
        """The stream of a call on `t`: the one given, else torch's current one, else the context's. (0 is
        torch's default stream where t is torch's.) held: the call's KVCache or Sampling, which is on the context's GPU as
        well."""
        if held.device is not None and held.device != self.opts.device:
            raise ValueError(f"buffers on GPU {held.device}, not on the context's ({self.opts.device})")
        for x in (t,) if out is None else (t, out):
            if _gpu_of(x) not in (None, self.opts.device):
                raise ValueError(f"an array on {x.device}, not on the context's GPU ({self.opts.device})")
            if _is_torch(x):
                _no_gradient(x)
        if not _is_torch(t):
            if stream is None and (held.torch or (out is not None and _is_torch(out))):
                # what torch has queued for them is on its stream, what was queued for the others on the context's
                raise ValueError("torch tensors beside arrays that are not torch's: the call's stream must be given")
            return stream
        if not _torch_first:
            raise RuntimeError("import torch before the library is loaded: they would hold two HIP runtimes")
        if stream is not None:
            return stream or 1
        torch = sys.modules["torch"]
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # a microsecond less than making a Stream
        of = raw(self.opts.device) if raw else torch.cuda.current_stream(self.opts.device).cuda_stream
        return of or 1   # 0: the legacy stream

    @staticmethod
    def _rows(t, name, rows, width):
        """Pointer and row stride of f32 rows [rows, width], whose elements lie beside each other."""
        shape = t.shape
        if len(shape) != 2 or shape[0] != rows or (width is not None and shape[1] != width) or _dtype(t) != "float32":
            raise ValueError(f"{name}: f32 [{rows}, {width}], not {t.dtype} {tuple(shape)}")
        if t.stride(1) != 1 and shape[1] > 1:
            raise ValueError(f"{name}: a row's values must lie beside each other")
        ld = t.stride(0)
        return t.data_ptr(), ld if rows > 1 else max(ld, shape[1])

    def _new(self, like, shape, dtype, given=None):
        """An array for a call on `like`. On a stream that was given, torch allocates for that stream: its memory goes to
        another tensor as soon as it is let go, which only the stream's own order makes safe."""
        if not _is_torch(like):
            return DeviceArray(shape, dtype, self.opts.device)
        torch = sys.modules["torch"]
        if given is None:
            if dtype == "float32" and shape == like.shape:   # half of torch.empty's 2 us; rows stay whole rows
                return torch.empty_like(like, memory_format=torch.contiguous_format)
            return like.new_empty(shape, dtype=getattr(torch, dtype))
        s = torch.cuda.ExternalStream(given, like.device) if given > 1 else torch.cuda.default_stream(like.device)
        with torch.cuda.stream(s):
            return like.new_empty(shape, dtype=getattr(torch, dtype))

    def kv_append(self, cache, jobs, k, v, stream=None):
        """cc_kv_append: the jobs' rows (slot, past, n) of k (before RoPE) and v,
        f32 [rows, kv heads * D], into the cache's pages, and the key bounds of
        the pages they complete."""
        stream = self._on(stream, cache, k, v)
        a, at, n, rows = _job_rows(jobs)
        kp, ldk = self._rows(k, "k", rows, cache.width)
        vp, ldv = self._rows(v, "v", rows, cache.width)
        st = self.lib.cc_kv_append(self.h, cache.ref, at, n, kp, ldk, vp, ldv, stream)
        if st:
            self._chk(st)

    def kv_bounds(self, cache, jobs, stream=None):
        """cc_kv_bounds: key bounds of the pages within the jobs' rows, from the cache."""
        stream = self._on(stream, cache, cache.kept[-1])
        a, at, n, _ = _job_rows(jobs)
        self._chk(self.lib.cc_kv_bounds(self.h, cache.ref, at, n, stream))

    def attend_pages(self, cache, jobs, q, budget, sink=1, recent=2, out=None, stream=None):
        """cc_attend_pages: attention of the jobs' rows, q f32 [rows, heads * D]
        before RoPE, over at most `budget` pages a row and kv head. Returns the
        rows' output (`out`, or a new array)."""
        given, stream = stream, self._on(stream, cache, q, out)
        a, at, n, rows = _job_rows(jobs)
        qp, ldq = self._rows(q, "q", rows, None)
        D, width = cache.c.head_dim, int(q.shape[1])
        heads = width // D
        if heads * D != width:
            raise ValueError(f"q: rows of {width} values are not whole heads of {D}")
        if out is None:
            out = self._new(q, (rows, width), "float32", given)
            op, ldo = out.data_ptr(), width
        else:
            op, ldo = self._rows(out, "out", rows, width)
        need = cache.workspace.get((rows, heads, budget))
        if need is None:
            need = self.lib.cc_attend_workspace(self.h, cache.ref, rows, heads, budget) if rows else 0
            if not need:
                raise CCError(CC_EARG, self.lib.cc_last_error(self.h).decode() if rows else "jobs: at least one")
            if len(cache.workspace) > 1000:
                cache.workspace.clear()
            cache.workspace[rows, heads, budget] = need
        ws = self._new(q, (need,), "uint8", given)
        st = self.lib.cc_attend_pages(self.h, cache.ref, at, n, heads, budget, sink, recent, qp, ldq, op, ldo,
                                      ws.data_ptr(), need, stream)
        if st:
            self._chk(st)
        return out

    def adjust_logits(self, logits, sampling, out=None, stream=None):
        """cc_logits_adjust: the rows with penalties, biases and masks, in `out`
        (logits itself, another array, or a new one)."""
        given, stream = stream, self._on(stream, sampling, logits, out)
        rows, V = sampling.rows, sampling.vocab
        lp, ld = self._rows(logits, "logits", rows, V)
        if out is None:
            out = self._new(logits, (rows, V), "float32", given)
            op, ldo = out.data_ptr(), V
        else:
            op, ldo = self._rows(out, "out", rows, V)
        st = self.lib.cc_logits_adjust(self.h, lp, ld, rows, V, sampling.ref, op, ldo, stream)
        if st:
            self._chk(st)
        return out

    def sample(self, logits, sampling, stream=None):
        """cc_sample: a token of each row of logits and the probability it was
        drawn with, int32 and f32 [rows]."""
        given, stream = stream, self._on(stream, sampling, logits)
        rows, V = sampling.rows, sampling.vocab
        lp, ld = self._rows(logits, "logits", rows, V)
        ids, probs = self._new(logits, (rows,), "int32", given), self._new(logits, (rows,), "float32", given)
        if sampling.workspace is None:
            sampling.workspace = self.lib.cc_sample_workspace(rows, V, sampling.ref)
        need = sampling.workspace
        ws = self._new(logits, (max(need, 16),), "uint8", given)
        st = self.lib.cc_sample(self.h, lp, ld, rows, V, sampling.ref, ids.data_ptr(), probs.data_ptr(), ws.data_ptr(),
                                need, stream)
        if st:
            self._chk(st)
        return ids, probs

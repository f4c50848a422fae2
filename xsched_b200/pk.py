"""ctypes face of libxpk.so (include/xsched_b200/pk.h): preemptible persistent kernels.

torch is used by callers for device memory and streams only; every kernel that runs is one of
the hand-written sm_100a kernels in xsched_b200/csrc/kernels.  If the shared library is missing
the import fails — there is no fallback path.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

from . import LIB_DIR

_LIB_PATH = LIB_DIR / "libxpk.so"
if not _LIB_PATH.exists():
    raise ImportError(f"{_LIB_PATH} not built; run `python -m xsched_b200.build` (needs nvcc)")
lib = C.CDLL(str(_LIB_PATH))

SUCCESS = 0
STATUS_IDLE, STATUS_RUNNING, STATUS_COMPLETED, STATUS_PREEMPTED, STATUS_ERROR = range(5)
KIND_TRIAD, KIND_VECADD, KIND_SORT, KIND_GEMM, KIND_ATTENTION, KIND_KV_COPY = 1, 2, 3, 4, 5, 6
DTYPE_BF16, DTYPE_F16 = 1, 2
KV_MAX_LIST, ATTENTION_MAX_SEQS = 2048, 1024
FLAG_NONE, FLAG_NON_PREEMPTIBLE, FLAG_ABORT_INFLIGHT, FLAG_GEMM_ONE_CTA, FLAG_GEMM_CTA_PAIR = 0, 1, 2, 4, 8

#: every symbol include/xsched_b200/pk.h declares
EXPORTS = [
    "xpkDeviceSmCount", "xpkResultString", "xpkFlagCreate", "xpkFlagDestroy", "xpkFlagSet",
    "xpkTaskCreateTriad", "xpkTaskCreateVecAdd", "xpkSortScratchBytes", "xpkTaskCreateSort",
    "xpkTaskCreateGemm", "xpkTaskLaunch", "xpkTaskQuery", "xpkTaskWait", "xpkTaskReset",
    "xpkTaskFlag", "xpkTaskKind", "xpkTaskDestroy", "xpkLaunchCount", "xpkSortNoAlloc", "xpkTaskTimes",
    "xpkFlagAttachRelay", "xpkFlagDetachRelay",
    "xpkKvCacheCreate", "xpkKvCacheDestroy", "xpkKvFree", "xpkKvFork", "xpkKvExtend", "xpkKvCompact", "xpkKvCopy",
    "xpkTaskCreateKvCopy", "xpkKvResult", "xpkKvAppend", "xpkAttentionScratchBytes", "xpkAttention", "xpkTaskCreateAttention",
]


class TaskInfo(C.Structure):
    _fields_ = [("status", C.c_uint32), ("error", C.c_uint32), ("tiles_done", C.c_uint64),
                ("tiles_total", C.c_uint64), ("launches", C.c_uint64), ("preemptions", C.c_uint64)]


_vp, _u32, _u64 = C.c_void_p, C.c_uint32, C.c_uint64


class KvCacheDesc(C.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("page_table", _vp), ("lens", _vp), ("refs", _vp), ("dtype", _u32), ("layers", _u32), ("pages", _u32),
                ("kv_heads", _u32), ("page_size", _u32), ("head_dim", _u32), ("seqs", _u32), ("table_width", _u32)]


class KvReport(C.Structure):
    _fields_ = [("copied", C.c_int32), ("missing", C.c_int32), ("refused", C.c_int32), ("live", C.c_int32)]


class KvAppendArgs(C.Structure):
    _fields_ = [("q", _vp), ("qkv", _vp), ("q_stride", _u64), ("qkv_stride", _u64), ("seqs", _vp), ("starts", _vp), ("q_weight", _vp), ("k_weight", _vp),
                ("inv_freq", _vp), ("eps", C.c_float), ("n", _u32), ("rows", _u32), ("q_heads", _u32), ("layer", _u32), ("rotary", _u32),
                ("interleaved", _u32)]


class AttentionArgs(C.Structure):
    _fields_ = [("out", _vp), ("q", _vp), ("out_stride", _u64), ("q_stride", _u64), ("seqs", _vp), ("starts", _vp), ("shared_len", _vp), ("scratch", _vp),
                ("scratch_bytes", _u64), ("scale", C.c_float), ("n", _u32), ("rows", _u32), ("q_heads", _u32), ("layer", _u32)]


lib.xpkResultString.restype = C.c_char_p
lib.xpkResultString.argtypes = [C.c_int]
lib.xpkDeviceSmCount.argtypes = [C.POINTER(C.c_int)]
lib.xpkFlagCreate.argtypes = [C.POINTER(_vp)]
lib.xpkFlagDestroy.argtypes = [_vp]
lib.xpkFlagSet.argtypes = [_vp, _u32, _vp]
lib.xpkFlagAttachRelay.argtypes = [_vp, C.POINTER(_vp)]
lib.xpkFlagDetachRelay.argtypes = [_vp, _vp]
lib.xpkTaskCreateTriad.argtypes = [C.POINTER(_vp), _vp, _vp, _vp, C.c_float, _u64, _u32, _u32, _vp]
lib.xpkTaskCreateVecAdd.argtypes = [C.POINTER(_vp), _vp, _vp, _vp, _u64, _u32, _u32, _vp]
lib.xpkSortScratchBytes.restype = C.c_size_t
lib.xpkSortScratchBytes.argtypes = [_u64]
lib.xpkTaskCreateSort.argtypes = [C.POINTER(_vp), _vp, _vp, _vp, _u64, _u32, _vp]
lib.xpkTaskCreateGemm.argtypes = [C.POINTER(_vp), _vp, _vp, _vp, _u32, _u32, _u32, _u32, _vp]
lib.xpkTaskLaunch.argtypes = [_vp, _vp, C.c_int]
lib.xpkTaskQuery.argtypes = [_vp, C.POINTER(TaskInfo)]
lib.xpkTaskWait.argtypes = [_vp, _u64, C.POINTER(TaskInfo)]
lib.xpkTaskReset.argtypes = [_vp, _vp]
lib.xpkTaskTimes.argtypes = [_vp, C.POINTER(_u64), C.POINTER(_u64)]
lib.xpkTaskFlag.argtypes = [_vp, C.POINTER(_vp)]
lib.xpkTaskKind.argtypes = [_vp, C.POINTER(_u32)]
lib.xpkTaskDestroy.argtypes = [_vp]
lib.xpkLaunchCount.restype = _u64
lib.xpkSortNoAlloc.argtypes = [_vp, _vp, _u64, _vp]
SORT_NOALLOC_MAX_KEYS = 4 << 20
lib.xpkKvCacheCreate.argtypes = [C.POINTER(_vp), C.POINTER(KvCacheDesc)]
lib.xpkKvCacheDestroy.argtypes = [_vp]
lib.xpkKvFree.argtypes = [_vp, _vp, _u32, _vp]
lib.xpkKvFork.argtypes = [_vp, _vp, _vp, _u32, _vp]
lib.xpkKvExtend.argtypes = [_vp, _vp, _vp, _u32, _vp]
lib.xpkKvCompact.argtypes = [_vp, _vp]
lib.xpkKvCopy.argtypes = [_vp, _vp, _vp, _u32, _vp]
lib.xpkTaskCreateKvCopy.argtypes = [C.POINTER(_vp), _vp, _vp, _vp, _u32, _u32, _vp]
lib.xpkKvResult.argtypes = [_vp, C.POINTER(KvReport), _vp]
lib.xpkKvAppend.argtypes = [_vp, C.POINTER(KvAppendArgs), _vp]
lib.xpkAttentionScratchBytes.restype = C.c_size_t
lib.xpkAttentionScratchBytes.argtypes = [_vp, _u32, _u32, _u32]
lib.xpkAttention.argtypes = [_vp, C.POINTER(AttentionArgs), _vp]
lib.xpkTaskCreateAttention.argtypes = [C.POINTER(_vp), _vp, C.POINTER(AttentionArgs), _u32, _vp]


class XpkError(RuntimeError):
    def __init__(self, code: int, what: str):
        super().__init__(f"{what}: {lib.xpkResultString(code).decode()} ({code})")
        self.code = code


def _check(code: int, what: str) -> None:
    if code != SUCCESS:
        raise XpkError(code, what)


def sm_count() -> int:
    n = C.c_int(0)
    _check(lib.xpkDeviceSmCount(C.byref(n)), "xpkDeviceSmCount")
    return n.value


def launch_count() -> int:
    return int(lib.xpkLaunchCount())


def sort_scratch_bytes(n: int) -> int:
    return int(lib.xpkSortScratchBytes(n))


def sort_no_alloc(keys, tmp, stream: int) -> None:
    """In-place ascending sort of the int32 tensor `keys` through xpkSortNoAlloc (no allocation at all;
    at most SORT_NOALLOC_MAX_KEYS keys; calls on one device must not overlap on the GPU)."""
    _check(lib.xpkSortNoAlloc(keys.data_ptr(), tmp.data_ptr(), keys.numel(), stream), "xpkSortNoAlloc")


class Flag:
    """One 32-bit preempt flag in device memory, shareable between tasks."""

    def __init__(self):
        p = _vp()
        _check(lib.xpkFlagCreate(C.byref(p)), "xpkFlagCreate")
        self.ptr = p.value

    def set(self, value: int, ctrl_stream: int = 0) -> None:
        _check(lib.xpkFlagSet(self.ptr, value, ctrl_stream), "xpkFlagSet")

    def attach_relay(self):
        """Give the flag an early-warning word in mapped host memory; returns it as a ctypes c_uint32 the caller
        stores to (non-zero just before raising the flag, zero before lowering it)."""
        p = _vp()
        _check(lib.xpkFlagAttachRelay(self.ptr, C.byref(p)), "xpkFlagAttachRelay")
        self.relay = p.value
        return C.c_uint32.from_address(p.value)

    def destroy(self) -> None:
        if self.ptr:
            if getattr(self, "relay", None):
                lib.xpkFlagDetachRelay(self.ptr, self.relay)
                self.relay = None
            lib.xpkFlagDestroy(self.ptr)
            self.ptr = None


@dataclass
class Info:
    status: int
    error: int
    tiles_done: int
    tiles_total: int
    launches: int
    preemptions: int


class Task:
    """Handle of one preemptible task.  Keep the tensors whose pointers were passed alive."""

    def __init__(self, handle: int, keepalive=()):
        self.handle = handle
        self._keep = keepalive

    # -- constructors -------------------------------------------------------------------
    @staticmethod
    def triad(a, b, c, s: float, tile_elems: int = 0, flags: int = 0, flag: Flag | None = None) -> "Task":
        h = _vp()
        _check(lib.xpkTaskCreateTriad(C.byref(h), a.data_ptr(), b.data_ptr(), c.data_ptr(), s, a.numel(),
                                      tile_elems, flags, flag.ptr if flag else None), "xpkTaskCreateTriad")
        return Task(h.value, (a, b, c, flag))

    @staticmethod
    def vecadd(c, a, b, tile_elems: int = 0, flags: int = 0, flag: Flag | None = None) -> "Task":
        h = _vp()
        _check(lib.xpkTaskCreateVecAdd(C.byref(h), c.data_ptr(), a.data_ptr(), b.data_ptr(), c.numel(),
                                       tile_elems, flags, flag.ptr if flag else None), "xpkTaskCreateVecAdd")
        return Task(h.value, (a, b, c, flag))

    @staticmethod
    def sort(keys, tmp, scratch, flags: int = 0, flag: Flag | None = None) -> "Task":
        h = _vp()
        _check(lib.xpkTaskCreateSort(C.byref(h), keys.data_ptr(), tmp.data_ptr(), scratch.data_ptr(), keys.numel(),
                                     flags, flag.ptr if flag else None), "xpkTaskCreateSort")
        return Task(h.value, (keys, tmp, scratch, flag))

    @staticmethod
    def gemm(c, a, b, flags: int = 0, flag: Flag | None = None) -> "Task":
        """c[M,N] = a[M,K] @ b[N,K].T, all bf16 row-major contiguous."""
        M, K = a.shape
        N, K2 = b.shape
        assert K == K2 and tuple(c.shape) == (M, N)
        h = _vp()
        _check(lib.xpkTaskCreateGemm(C.byref(h), c.data_ptr(), a.data_ptr(), b.data_ptr(), M, N, K, flags,
                                     flag.ptr if flag else None), "xpkTaskCreateGemm")
        return Task(h.value, (a, b, c, flag))

    @staticmethod
    def attention(cache: "KvCache", out, q, seqs, *, scratch, starts=None, shared_len=None, layer: int = 0, scale: float | None = None,
                  flags: int = 0, flag: Flag | None = None) -> "Task":
        """KvCache.attention as a task; `scratch` is the task's own.  Its tiles are counted when a launch has read the lengths."""
        a = cache._attention_args(out, q, seqs, starts, shared_len, scratch, layer, scale)
        h = _vp()
        _check(lib.xpkTaskCreateAttention(C.byref(h), cache.handle, C.byref(a), flags, flag.ptr if flag else None), "xpkTaskCreateAttention")
        return Task(h.value, (cache, out, q, seqs, starts, shared_len, scratch, flag))

    @staticmethod
    def kv_copy(cache: "KvCache", src, dst, flags: int = 0, flag: Flag | None = None) -> "Task":
        """KvCache.copy as a task."""
        n = cache._list("kv_copy", src, dst)
        h = _vp()
        _check(lib.xpkTaskCreateKvCopy(C.byref(h), cache.handle, src.data_ptr(), dst.data_ptr(), n, flags, flag.ptr if flag else None),
               "xpkTaskCreateKvCopy")
        return Task(h.value, (cache, src, dst, flag))

    # -- control ------------------------------------------------------------------------
    def launch(self, stream: int, sm_limit: int = 0) -> None:
        _check(lib.xpkTaskLaunch(self.handle, stream, sm_limit), "xpkTaskLaunch")

    def query(self) -> Info:
        ti = TaskInfo()
        _check(lib.xpkTaskQuery(self.handle, C.byref(ti)), "xpkTaskQuery")
        return Info(ti.status, ti.error, ti.tiles_done, ti.tiles_total, ti.launches, ti.preemptions)

    def wait(self, timeout_us: int = 30_000_000) -> Info:
        ti = TaskInfo()
        _check(lib.xpkTaskWait(self.handle, timeout_us, C.byref(ti)), "xpkTaskWait")
        return Info(ti.status, ti.error, ti.tiles_done, ti.tiles_total, ti.launches, ti.preemptions)

    def reset(self, stream: int) -> None:
        _check(lib.xpkTaskReset(self.handle, stream), "xpkTaskReset")

    def flag_ptr(self) -> int:
        p = _vp()
        _check(lib.xpkTaskFlag(self.handle, C.byref(p)), "xpkTaskFlag")
        return p.value

    def set_flag(self, value: int, ctrl_stream: int = 0) -> None:
        _check(lib.xpkFlagSet(self.flag_ptr(), value, ctrl_stream), "xpkFlagSet")

    def destroy(self) -> None:
        if self.handle:
            lib.xpkTaskDestroy(self.handle)
            self.handle = None
            self._keep = ()


def _no_gradient(what: str, x) -> None:
    """The cache's kernels have no backward pass: what autograd would follow through them is refused, not lost."""
    if x.requires_grad:
        import torch
        if torch.is_grad_enabled():
            raise ValueError(f"{what} requires a gradient, and this call has none to give: call it under torch.no_grad()")


def _rows(what: str, x, width: int):
    """(rows, elements between rows) of a tensor whose trailing dimensions, `width` elements in all, are dense."""
    shape = x.shape
    rows = shape[0]
    if x.numel() != rows * width:
        raise ValueError(f"{what}: {tuple(shape)} is not [rows] of {width} elements")
    if x.is_contiguous():
        return rows, 0
    inner = 1
    for size, stride in zip(reversed(x.shape[1:]), reversed(x.stride()[1:])):
        if size != 1 and stride != inner:
            raise ValueError(f"{what}: a row's elements lie apart (strides {x.stride()})")
        inner *= size
    if rows > 1 and x.stride(0) < width:                  # an expanded tensor has a step of 0, which would mean dense
        raise ValueError(f"{what}: rows overlap (strides {x.stride()})")
    return rows, x.stride(0) if rows > 1 else 0


class KvCache:
    """A paged key/value cache and the operators of a decode loop around it (see pk.h for what each does exactly).

    k, v [layers, pages, kv_heads, page_size, head_dim] (bf16 or fp16), page_table [seqs, width], lens [seqs] and refs [pages]
    (int32) are the caller's tensors on one device and stay where they are.  Calls take the stream they run on; lists and
    lengths are read on the device when the kernels run.  destroy() gives the handle back.

    For inference: nothing is recorded for autograd, and tensors that require a gradient are refused unless under torch.no_grad()."""

    def __init__(self, k, v, page_table, lens, refs):
        dtype = {"torch.bfloat16": DTYPE_BF16, "torch.float16": DTYPE_F16}.get(str(k.dtype))
        if dtype is None or k.dtype != v.dtype:
            raise ValueError(f"k and v are both bfloat16 or both float16, got {k.dtype} and {v.dtype}")
        if k.dim() != 5 or k.shape != v.shape:
            raise ValueError(f"k and v are [layers, pages, kv_heads, page_size, head_dim] alike, got {tuple(k.shape)} and {tuple(v.shape)}")
        layers, pages, heads, page, dim = k.shape
        if page_table.dim() != 2 or lens.shape != page_table.shape[:1] or refs.shape != (pages,):
            raise ValueError("page_table is [seqs, width], lens [seqs], refs [pages]")
        for name, x in (("page_table", page_table), ("lens", lens), ("refs", refs)):
            if str(x.dtype) != "torch.int32":
                raise ValueError(f"{name} is int32, got {x.dtype}")
        for name, x in (("k", k), ("v", v), ("page_table", page_table), ("lens", lens), ("refs", refs)):
            if not x.is_contiguous() or x.device != k.device or not x.is_cuda:
                raise ValueError(f"{name} is contiguous and on the same CUDA device as k")
            _no_gradient(name, x)
        self.k, self.v, self.page_table, self.lens, self.refs = k, v, page_table, lens, refs
        self.device, self.dtype, self.heads, self.dim, self.seqs = k.device, k.dtype, heads, dim, lens.numel()
        self._int32 = lens.dtype
        self.handle = None
        d = KvCacheDesc(k.data_ptr(), v.data_ptr(), page_table.data_ptr(), lens.data_ptr(), refs.data_ptr(), dtype, layers, pages, heads, page, dim,
                        page_table.shape[0], page_table.shape[1])
        h = _vp()
        import torch
        with torch.cuda.device(k.device):                     # the handle belongs to the device that is current here
            _check(lib.xpkKvCacheCreate(C.byref(h), C.byref(d)), "xpkKvCacheCreate")
        self.handle = h.value

    def destroy(self) -> None:
        if self.handle:
            lib.xpkKvCacheDestroy(self.handle)
            self.handle = None

    # -- checks -------------------------------------------------------------------------
    def _ints(self, what: str, x):
        if x is None:
            return None
        if x.dtype is not self._int32 or not x.is_contiguous() or x.device != self.device:
            raise ValueError(f"{what} is a contiguous int32 tensor on {self.device}")
        return x.data_ptr()

    def _list(self, what: str, a, b) -> int:
        if self._ints(what, a) is None or self._ints(what, b) is None or a.numel() != b.numel():
            raise ValueError(f"{what}: two int32 lists of the same length")
        return a.numel()

    def _data(self, what: str, x):
        if x is None:
            return None
        if x.dtype is not self.dtype or x.device != self.device:
            raise ValueError(f"{what} is {self.dtype} on {self.device}, got {x.dtype} on {x.device}")
        _no_gradient(what, x)
        return x.data_ptr()

    def _entries(self, seqs, starts, rows: int) -> int:
        n = seqs.numel() if seqs is not None else starts.numel() - 1 if starts is not None else rows
        if starts is not None and starts.numel() != n + 1:
            raise ValueError(f"starts has {starts.numel()} entries for {n} sequences: one more is wanted")
        if starts is None and n != rows:
            raise ValueError(f"{rows} rows for {n} sequences: without `starts` each has one")
        if seqs is None and n > self.seqs:
            raise ValueError(f"{n} sequences, the cache has {self.seqs}")
        return n

    # -- pages --------------------------------------------------------------------------
    def free(self, seqs, stream: int) -> None:
        n = self._list("free", seqs, seqs)
        _check(lib.xpkKvFree(self.handle, seqs.data_ptr(), n, stream), "xpkKvFree")

    def fork(self, parents, children, stream: int) -> None:
        n = self._list("fork", parents, children)
        _check(lib.xpkKvFork(self.handle, parents.data_ptr(), children.data_ptr(), n, stream), "xpkKvFork")

    def extend(self, seqs, tokens, stream: int) -> None:
        n = self._list("extend", seqs, tokens)
        _check(lib.xpkKvExtend(self.handle, seqs.data_ptr(), tokens.data_ptr(), n, stream), "xpkKvExtend")

    def compact(self, stream: int) -> None:
        _check(lib.xpkKvCompact(self.handle, stream), "xpkKvCompact")

    def copy(self, src, dst, stream: int) -> None:
        n = self._list("copy", src, dst)
        _check(lib.xpkKvCopy(self.handle, src.data_ptr(), dst.data_ptr(), n, stream), "xpkKvCopy")

    def result(self, stream: int) -> KvReport:
        """What the last extend or compact on the cache found (waits for the stream)."""
        r = KvReport()
        _check(lib.xpkKvResult(self.handle, C.byref(r), stream), "xpkKvResult")
        return r

    # -- new tokens ---------------------------------------------------------------------
    def append(self, q, qkv, seqs, stream: int, *, starts=None, q_weight=None, k_weight=None, eps: float = 1e-6, inv_freq=None,
               interleaved: bool = False, layer: int = 0) -> None:
        """Norms, rotation and write of the rows of qkv [rows, (q_heads + 2 kv_heads) head_dim]; queries go to q [rows, q_heads, head_dim]."""
        heads = q.numel() // max(1, q.shape[0] * self.dim)
        rows, q_stride = _rows("q", q, heads * self.dim)
        qkv_rows, qkv_stride = _rows("qkv", qkv, (heads + 2 * self.heads) * self.dim)
        if rows != qkv_rows:
            raise ValueError(f"{rows} rows of q, {qkv_rows} of qkv")
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if w is not None and (w.numel() != self.dim or not w.is_contiguous()):
                raise ValueError(f"{name} has {self.dim} elements")
        if inv_freq is not None and (inv_freq.element_size() != 8 or not inv_freq.is_floating_point() or not inv_freq.is_contiguous() or inv_freq.device != self.device):
            raise ValueError("inv_freq is a contiguous float64 tensor on the cache's device")
        if inv_freq is not None:
            _no_gradient("inv_freq", inv_freq)
        a = KvAppendArgs(self._data("q", q), self._data("qkv", qkv), q_stride, qkv_stride, self._ints("seqs", seqs), self._ints("starts", starts),
                         self._data("q_weight", q_weight), self._data("k_weight", k_weight), None if inv_freq is None else inv_freq.data_ptr(), eps,
                         self._entries(seqs, starts, rows), rows, heads, layer, 0 if inv_freq is None else 2 * inv_freq.numel(), interleaved)
        _check(lib.xpkKvAppend(self.handle, C.byref(a), stream), "xpkKvAppend")

    # -- attention ----------------------------------------------------------------------
    def attention_scratch_bytes(self, rows: int, n: int, q_heads: int) -> int:
        return int(lib.xpkAttentionScratchBytes(self.handle, rows, n, q_heads))

    def _attention_args(self, out, q, seqs, starts, shared_len, scratch, layer, scale) -> AttentionArgs:
        heads = q.numel() // max(1, q.shape[0] * self.dim)
        rows, q_stride = _rows("q", q, heads * self.dim)
        out_rows, out_stride = _rows("out", out, heads * self.dim)
        if rows != out_rows:
            raise ValueError(f"{rows} rows of q, {out_rows} of out")
        if scratch.device != self.device or not scratch.is_contiguous():
            raise ValueError("scratch is contiguous and on the cache's device")
        return AttentionArgs(self._data("out", out), self._data("q", q), out_stride, q_stride, self._ints("seqs", seqs), self._ints("starts", starts),
                             self._ints("shared_len", shared_len), scratch.data_ptr(), scratch.numel() * scratch.element_size(),
                             self.dim ** -0.5 if scale is None else scale, self._entries(seqs, starts, rows), rows, heads, layer)

    def attention(self, out, q, seqs, stream: int, *, scratch, starts=None, shared_len=None, layer: int = 0, scale: float | None = None) -> None:
        """out = attention of q [rows, q_heads, head_dim] to the positions of its sequences; scale None: head_dim ** -0.5."""
        a = self._attention_args(out, q, seqs, starts, shared_len, scratch, layer, scale)
        _check(lib.xpkAttention(self.handle, C.byref(a), stream), "xpkAttention")

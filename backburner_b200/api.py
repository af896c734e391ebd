"""ctypes binding of libpacuda.so (include/pa_cuda.h) and the Python host API over it.

Tensors passed in are torch CUDA tensors (device memory, streams); nothing here computes attention itself.
"""
from __future__ import annotations

import ctypes
import os
from dataclasses import dataclass
from typing import Sequence

F16, Q8_0, Q4_0 = 0, 1, 2          # config_req.is_q8 (phone-attn/phone-attn.h:15)
QK_F16, QK_INT8 = 0, 1             # QK arithmetic: f16(d*q) K, or the int8-domain QK (scripts/sme/sme_attn.c:465-508)
_HERE = os.path.dirname(os.path.abspath(__file__))
lib_path = os.path.join(_HERE, "libpacuda.so")

OK, EINVAL, ECUDA, ENOMEM, ETIMEOUT, EUNSUPPORTED, ENCCL = 0, -1, -2, -3, -4, -5, -6


class PaCudaError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"pa_cuda error {code}: {msg}")
        self.code = code


class LibraryMissing(PaCudaError):
    def __init__(self, why: str):
        super().__init__(ECUDA, f"libpacuda.so not loadable ({why}); build it with `python -m backburner_b200.build`")


class _Shape(ctypes.Structure):
    _fields_ = [("hd", ctypes.c_uint32), ("nkv", ctypes.c_uint32), ("rows", ctypes.c_uint32),
                ("quant", ctypes.c_uint32), ("rs", ctypes.c_uint64), ("hb", ctypes.c_uint64)]


class _Seg(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("nk", ctypes.c_uint32), ("set", ctypes.c_uint32)]


class _Page(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("hk", ctypes.c_void_p), ("hv", ctypes.c_void_p)]


class _Cache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("n_layers", ctypes.c_uint32),
                ("n_pages", ctypes.c_uint32), ("page_keys", ctypes.c_uint32)]


class _Mask(ctypes.Structure):
    _fields_ = [("n_tok", ctypes.c_uint32), ("window", ctypes.c_uint32), ("sinks", ctypes.c_uint32),
                ("tree", ctypes.c_uint32)]


class _Append(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("q_set", ctypes.c_int64), ("q_tok", ctypes.c_int64), ("k_set", ctypes.c_int64),
                ("k_tok", ctypes.c_int64), ("v_set", ctypes.c_int64), ("v_tok", ctypes.c_int64),
                ("wq", ctypes.c_void_p), ("wk", ctypes.c_void_p), ("freqs", ctypes.c_void_p), ("pos", ctypes.c_void_p),
                ("dtype", ctypes.c_uint32), ("w_dtype", ctypes.c_uint32), ("rot", ctypes.c_uint32),
                ("interleaved", ctypes.c_uint32), ("eps", ctypes.c_float), ("scale", ctypes.c_float)]


_P = ctypes.c_void_p
_U = ctypes.c_uint32
_SIGS = {
    "pa_cuda_available": (ctypes.c_int, []),
    "pa_cuda_abi_version": (ctypes.c_int, []),
    "pa_cuda_create": (ctypes.c_int, [ctypes.c_int, ctypes.POINTER(_P)]),
    "pa_cuda_destroy": (None, [_P]),
    "pa_cuda_last_error": (ctypes.c_char_p, [_P]),
    "pa_cuda_status": (ctypes.c_int, [_P, _P]),
    "pa_cuda_set_timeout_ns": (None, [_P, ctypes.c_uint64]),
    "pa_cuda_launch_count": (ctypes.c_uint64, [_P]),
    "pa_cuda_set_stall_test": (None, [_P, ctypes.c_int]),
    "pa_cuda_set_kernel": (None, [_P, ctypes.c_int]),
    "pa_cuda_set_qk_domain": (None, [_P, ctypes.c_int]),
    "pa_cuda_plan_create": (ctypes.c_int, [_P, ctypes.POINTER(_Shape), ctypes.c_uint32, ctypes.POINTER(_Seg),
                                           ctypes.c_uint32, ctypes.c_uint32, ctypes.POINTER(_P)]),
    "pa_cuda_plan_scratch_bytes": (ctypes.c_size_t, [_P]),
    "pa_cuda_plan_jobs": (ctypes.c_uint32, [_P]),
    "pa_cuda_plan_launches": (ctypes.c_uint32, [_P]),
    "pa_cuda_plan_kernel": (ctypes.c_char_p, [_P]),
    "pa_cuda_plan_run": (ctypes.c_int, [_P, _P, _P, _P, _P, _P]),
    "pa_cuda_plan_run_host": (ctypes.c_int, [_P, _P, _P, _P, _P, _P]),
    "pa_cuda_plan_destroy": (None, [_P]),
    "pa_cuda_plan_profile": (ctypes.c_int, [_P, ctypes.c_uint32]),
    "pa_cuda_plan_kernel_ms": (ctypes.c_int, [_P, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_uint32)]),
    "pa_cuda_attn": (ctypes.c_int, [_P, ctypes.POINTER(_Shape), _P, ctypes.c_uint32, ctypes.POINTER(_Seg),
                                    ctypes.c_uint32, _P, _P, _P, _P]),
    "pa_cuda_attn_partial": (ctypes.c_int, [_P, ctypes.POINTER(_Shape), _P, ctypes.c_float, _P, _P, ctypes.c_uint32,
                                            _P, _P, _P, _P]),
    "pa_cuda_merge": (ctypes.c_int, [_P, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_uint32, _P, _P, _P, _P, _P, _P,
                                     ctypes.c_int, _P]),
    "pa_cuda_merge_gathered": (ctypes.c_int, [_P, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_uint32, _P, _P, _P, _P,
                                              ctypes.c_int, _P]),
    "pa_cuda_normalize": (ctypes.c_int, [_P, ctypes.c_uint32, ctypes.c_uint64, _P, _P, _P, _P, _P, _P]),
    "pa_cuda_scale_q": (ctypes.c_int, [_P, _P, ctypes.c_float, ctypes.c_uint64, _P, _P]),
    "pa_cuda_fold_reply": (ctypes.c_int, [_P, ctypes.c_uint32, ctypes.c_uint64, _P, _P, _P, _P, _P, _P]),
    "pa_cuda_nccl_unique_id": (ctypes.c_int, [_P, ctypes.c_size_t]),
    "pa_cuda_nccl_comm_create": (ctypes.c_int, [_P, _P, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_void_p)]),
    "pa_cuda_nccl_comm_destroy": (None, [_P]),
    "pa_cuda_shard_attn_allgather_merge": (ctypes.c_int, [_P, _P, _P, _P, _P, _P, _P]),
    "pa_cuda_set_shard_exchange": (None, [_P, ctypes.c_int]),
    "pa_cuda_shard_last": (None, [_P, ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_int)]),
    "pa_cuda_set_shard_groups": (None, [_P, ctypes.c_int]),
    "pa_cuda_set_shard_timeout_ms": (None, [_P, ctypes.c_uint32]),
    "pa_cuda_nccl_wait": (ctypes.c_int, [_P, _P, _P, ctypes.c_uint32]),
    "pa_cuda_alloc_page": (ctypes.c_int, [_P, ctypes.c_size_t, ctypes.POINTER(_Page)]),
    "pa_cuda_free_page": (None, [_P, ctypes.POINTER(_Page)]),
    "pa_cuda_begin": (ctypes.c_int, [_P, ctypes.POINTER(_Page), ctypes.POINTER(ctypes.c_uint32), ctypes.c_int, _P,
                                     ctypes.POINTER(_Shape), ctypes.c_int, ctypes.c_int]),
    "pa_cuda_end": (ctypes.c_double, [_P, _P, _P, _P]),
    "pa_cuda_exec_ms": (ctypes.c_double, [_P]),
    "pa_cuda_arm": (ctypes.c_int, [_P, _P, ctypes.POINTER(ctypes.c_uint32), ctypes.c_int, ctypes.POINTER(_Shape),
                                   ctypes.c_int]),
    "pa_cuda_graph_calls": (ctypes.c_uint64, [_P]),
    "pa_cuda_attn_noalloc": (ctypes.c_int, [ctypes.POINTER(_Shape), _P, _P, _P, ctypes.c_uint32, _P, _P, _P, _P,
                                            ctypes.POINTER(ctypes.c_char_p)]),
    "pa_cuda_cache_plan_create": (ctypes.c_int, [_P, ctypes.POINTER(_Shape), ctypes.POINTER(_Cache), _U, _U,
                                                 ctypes.POINTER(_Mask), ctypes.POINTER(_P)]),
    "pa_cuda_cache_plan_kernel": (ctypes.c_char_p, [_P]),
    "pa_cuda_cache_plan_destroy": (None, [_P]),
    "pa_cuda_cache_attn": (ctypes.c_int, [_P, _U, _P, _P, _P, _P, _P, _P, _P, _P, _P]),
    "pa_cuda_cache_attn_reply": (ctypes.c_int, [_P, _U, _P, _P, _P, _P, _P, _P, _P, _P]),
    "pa_cuda_cache_append": (ctypes.c_int, [_P, ctypes.POINTER(_Shape), ctypes.POINTER(_Cache), _U,
                                            ctypes.POINTER(_Append), _U, _U, _P, _U, _P, _P, _P]),
    "pa_cuda_cache_rows": (ctypes.c_int, [_P, ctypes.POINTER(_Shape), ctypes.POINTER(_Cache), _U, _U, _U, _P, _U, _P,
                                          _P, _P, _P]),
    "pa_cuda_cache_copy_pages": (ctypes.c_int, [_P, ctypes.POINTER(_Shape), ctypes.POINTER(_Cache), _P, _P, _U, _P]),
    "pa_cuda_cache_compact": (ctypes.c_int, [_P, ctypes.POINTER(_Shape), ctypes.POINTER(_Cache), _U, _U, _P, _U, _P, _P,
                                             _P, _P, _P]),
}

_lib = None


def lib() -> ctypes.CDLL:
    """The loaded libpacuda.so (raises LibraryMissing if it is not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(lib_path):
            raise LibraryMissing("not built")
        try:
            L = ctypes.CDLL(lib_path)
        except OSError as e:  # pragma: no cover - depends on the machine
            raise LibraryMissing(str(e)) from e
        for name, (res, args) in _SIGS.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def available() -> bool:
    """True when libpacuda.so loads and a compute-capability-10 GPU is visible (pa_cuda_available)."""
    try:
        return bool(lib().pa_cuda_available())
    except LibraryMissing:
        return False


def head_bytes(quant: int, hd: int) -> int:
    return hd // 32 * (34 if quant == Q8_0 else 18) if quant in (Q8_0, Q4_0) else hd * 2


@dataclass(frozen=True)
class Shape:
    """Geometry of a call: head dim, KV heads, query rows per KV head, quantisation, row stride and head bytes."""
    hd: int
    nkv: int
    rows: int
    quant: int
    rs: int
    hb: int

    def c(self) -> _Shape:
        return _Shape(self.hd, self.nkv, self.rows, self.quant, self.rs, self.hb)


def shape_for(hd: int, nkv: int, rows: int, quant: int = Q8_0, rs: int | None = None) -> Shape:
    hb = head_bytes(quant, hd)
    return Shape(hd, nkv, rows, quant, rs if rs is not None else nkv * hb, hb)


@dataclass
class Seg:
    """nk consecutive key positions at device pointers k, v, folded into output set `set`."""
    k: int
    v: int
    nk: int
    set: int = 0


def _ptr(t) -> int:
    return 0 if t is None else int(t.data_ptr())


def _stream_ptr(stream) -> int:
    """cudaStream_t handle for a torch stream (None: torch's current stream). torch's default stream has handle 0,
    which the C ABI reads as "the context's own stream", so it is passed as cudaStreamLegacy (1) instead."""
    if stream is None:
        import torch
        stream = torch.cuda.current_stream()
    h = int(getattr(stream, "cuda_stream", stream))
    return h if h != 0 else 1


class Context:
    """A libpacuda context on one device (pa_cuda_create)."""

    def __init__(self, device: int = 0):
        self._h = _P()
        rc = lib().pa_cuda_create(device, ctypes.byref(self._h))
        if rc != OK:
            raise PaCudaError(rc, f"pa_cuda_create(device={device}) failed")
        self.device = device

    @property
    def handle(self):
        return self._h

    def check(self, rc: int, what: str = ""):
        if rc != OK:
            msg = lib().pa_cuda_last_error(self._h).decode(errors="replace")
            raise PaCudaError(rc, f"{what}: {msg}" if what else msg)

    def status(self, stream=None):
        """Synchronise the stream and raise if a kernel gave up a bounded wait (ETIMEOUT) or a cache call met an argument out
        of range on the device (EINVAL); after both, the next call raises the second (pa_cuda_status)."""
        self.check(lib().pa_cuda_status(self._h, _stream_ptr(stream)), "status")

    def set_timeout_ns(self, ns: int):
        lib().pa_cuda_set_timeout_ns(self._h, int(ns))

    def set_kernel(self, which: int):
        """0: by shape; 1: split-K mma.sync kernel; 2: tcgen05 kernel on single CTAs; 3: tcgen05 kernel on CTA pairs
        (2 and 3: hd 128, quantised rows) — for plans created afterwards."""
        lib().pa_cuda_set_kernel(self._h, int(which))

    def set_qk_domain(self, domain: int):
        """QK_F16 (default) or QK_INT8: the reference's int8-domain QK (Q quantised per 32-block by the Q8_0 rule,
        int32 block dot products with the Q8_0 K bytes, scores in fp32), Q8_0 rows on the split-K kernel only — for
        plans created afterwards."""
        lib().pa_cuda_set_qk_domain(self._h, int(domain))

    def set_stall_test(self, on: bool):
        """Failure-detection hook: the next decode kernels wait on a barrier nothing completes (bounded)."""
        lib().pa_cuda_set_stall_test(self._h, 1 if on else 0)

    @property
    def launches(self) -> int:
        return int(lib().pa_cuda_launch_count(self._h))

    # exchange of the position-shard call (shard_attn_allgather_merge) for calls made afterwards
    EXCHANGE_AUTO, EXCHANGE_ALLGATHER, EXCHANGE_ALLREDUCE, EXCHANGE_PEER = 0, 1, 2, 3

    def set_shard_exchange(self, mode: int):
        """0: by size; 1: all-gather of every rank's packed (O, m, l) and the fold; 2: max / sum all-reduces; 3: peer
        stores over NVLink."""
        lib().pa_cuda_set_shard_exchange(self._h, int(mode))

    def shard_last(self):
        """(exchange, set groups) the last shard call of this context used."""
        e, g = ctypes.c_int(), ctypes.c_int()
        lib().pa_cuda_shard_last(self._h, ctypes.byref(e), ctypes.byref(g))
        return int(e.value), int(g.value)

    def set_shard_groups(self, groups: int):
        """Output-set groups whose exchange overlaps the next group's kernels (0: by size, 1: none)."""
        lib().pa_cuda_set_shard_groups(self._h, int(groups))

    def set_shard_timeout_ms(self, ms: int):
        """> 0: the shard call waits for its exchange and aborts the communicator past ms (raises ETIMEOUT)."""
        lib().pa_cuda_set_shard_timeout_ms(self._h, int(ms))

    def close(self):
        if self._h:
            lib().pa_cuda_destroy(self._h)
            self._h = _P()

    def __del__(self):  # pragma: no cover
        try:
            self.close()
        except Exception:
            pass


class Plan:
    """The split of a call (output sets x key segments) into chunk jobs, built once, run many times
    (pa_cuda_plan_create / pa_cuda_plan_run)."""

    def __init__(self, ctx: Context, shape: Shape, n_sets: int, segs: Sequence[Seg], chunk_keys: int = 0):
        self.ctx, self.shape, self.n_sets = ctx, shape, n_sets
        arr = (_Seg * max(1, len(segs)))(*[_Seg(s.k, s.v, s.nk, s.set) for s in segs])
        self._h = _P()
        self._sh = shape.c()
        ctx.check(lib().pa_cuda_plan_create(ctx.handle, ctypes.byref(self._sh), n_sets, arr, len(segs), chunk_keys,
                                            ctypes.byref(self._h)), "plan_create")

    @property
    def scratch_bytes(self) -> int:
        return int(lib().pa_cuda_plan_scratch_bytes(self._h))

    @property
    def jobs(self) -> int:
        return int(lib().pa_cuda_plan_jobs(self._h))

    @property
    def launches(self) -> int:
        return int(lib().pa_cuda_plan_launches(self._h))

    @property
    def kernel(self) -> str:
        """Name of the attention-kernel instance the plan launches."""
        return lib().pa_cuda_plan_kernel(self._h).decode()

    def run(self, Qs, O, m, l, stream=None):
        self.ctx.check(lib().pa_cuda_plan_run(self._h, _ptr(Qs), _ptr(O), _ptr(m), _ptr(l), _stream_ptr(stream)),
                       "plan_run")

    def run_host(self, Qs_host, O_host, m_host, l_host, stream=None):
        """Host buffers in, host buffers out (copies inside; returns when they have landed)."""
        self.ctx.check(lib().pa_cuda_plan_run_host(self._h, _ptr(Qs_host), _ptr(O_host), _ptr(m_host), _ptr(l_host),
                                                   _stream_ptr(stream)), "plan_run_host")

    def profile(self, max_runs: int):
        """Record CUDA events around the decode kernel of the next max_runs runs (0: off)."""
        self.ctx.check(lib().pa_cuda_plan_profile(self._h, max_runs), "plan_profile")

    def kernel_ms(self):
        """(summed decode-kernel milliseconds, runs) since profile() / the last call."""
        t = ctypes.c_double()
        n = ctypes.c_uint32()
        self.ctx.check(lib().pa_cuda_plan_kernel_ms(self._h, ctypes.byref(t), ctypes.byref(n)), "plan_kernel_ms")
        return float(t.value), int(n.value)

    def close(self):
        if self._h:
            lib().pa_cuda_plan_destroy(self._h)
            self._h = _P()

    def __del__(self):  # pragma: no cover
        try:
            self.close()
        except Exception:
            pass


def _outputs(shape: Shape, n_sets: int, device):
    import torch
    rows = n_sets * shape.nkv * shape.rows
    O = torch.empty((n_sets, shape.nkv, shape.rows, shape.hd), dtype=torch.float32, device=device)
    m = torch.empty((n_sets, shape.nkv, shape.rows), dtype=torch.float32, device=device)
    l = torch.empty_like(m)
    assert O.numel() == rows * shape.hd
    return O, m, l


def attn(ctx: Context, shape: Shape, Qs, segs: Sequence[Seg], n_sets: int = 1, out=None, stream=None):
    """Partial attention of n_sets output sets over key segments (pa_cuda_attn). Qs: f16 (as int16/float16 tensor)
    [n_sets][nkv][rows][hd] = f16(q*scale). Returns (O, m, l) fp32."""
    O, m, l = out if out is not None else _outputs(shape, n_sets, Qs.device)
    arr = (_Seg * max(1, len(segs)))(*[_Seg(s.k, s.v, s.nk, s.set) for s in segs])
    sh = shape.c()
    ctx.check(lib().pa_cuda_attn(ctx.handle, ctypes.byref(sh), _ptr(Qs), n_sets, arr, len(segs), _ptr(O), _ptr(m),
                                 _ptr(l), _stream_ptr(stream)), "attn")
    return O, m, l


def attn_partial(ctx: Context, shape: Shape, Q, scale: float, K, V, nk: int, stream=None):
    """sme_attn_partial over all heads of one segment: Q fp32 [nkv][rows][hd] unscaled, K/V uint8 rows."""
    O, m, l = _outputs(shape, 1, Q.device)
    sh = shape.c()
    ctx.check(lib().pa_cuda_attn_partial(ctx.handle, ctypes.byref(sh), _ptr(Q), float(scale), _ptr(K), _ptr(V), nk,
                                         _ptr(O), _ptr(m), _ptr(l), _stream_ptr(stream)), "attn_partial")
    return O[0], m[0], l[0]


def merge(ctx: Context, hd: int, Op, mp, lp, out=None, fold: bool = False, stream=None):
    """LSE merge of n partials Op [n][rows][hd], mp/lp [n][rows] -> (O [rows][hd], m, l) (pa_cuda_merge)."""
    import torch
    n = Op.shape[0]
    rows = mp[0].numel() if n else (out[1].numel() if out is not None else 0)
    if out is None:
        O = torch.empty((rows, hd), dtype=torch.float32, device=Op.device)
        m = torch.empty((rows,), dtype=torch.float32, device=Op.device)
        l = torch.empty_like(m)
    else:
        O, m, l = out
    ctx.check(lib().pa_cuda_merge(ctx.handle, hd, rows, n, _ptr(Op), _ptr(mp), _ptr(lp), _ptr(O), _ptr(m), _ptr(l),
                                  1 if fold else 0, _stream_ptr(stream)), "merge")
    return O, m, l


def merge_gathered(ctx: Context, hd: int, rows: int, packed, n_parts: int, out=None, fold: bool = False, stream=None):
    """Merge n_parts partials packed as [n_parts][rows*hd + 2*rows] (O, then m, then l, per part), as one all-gather
    of each rank's packed partial delivers them (pa_cuda_merge_gathered). Returns (O [rows][hd], m, l)."""
    import torch
    if out is None:
        O = torch.empty((rows, hd), dtype=torch.float32, device=packed.device)
        m = torch.empty((rows,), dtype=torch.float32, device=packed.device)
        l = torch.empty_like(m)
    else:
        O, m, l = out
    ctx.check(lib().pa_cuda_merge_gathered(ctx.handle, hd, rows, n_parts, _ptr(packed), _ptr(O), _ptr(m), _ptr(l),
                                           1 if fold else 0, _stream_ptr(stream)), "merge_gathered")
    return O, m, l


def packed_views(buf, rows: int, hd: int):
    """(O, m, l) views into one packed partial buffer of rows*(hd+2) floats."""
    return buf[:rows * hd].view(rows, hd), buf[rows * hd:rows * hd + rows], buf[rows * hd + rows:rows * (hd + 2)]


def normalize(ctx: Context, hd: int, O, m, l, stream=None):
    """O/l -> f16, lse = m + log l (pa_cuda_normalize). Returns (Oh float16, lse fp32)."""
    import torch
    rows = m.numel()
    Oh = torch.empty((rows, hd), dtype=torch.float16, device=O.device)
    lse = torch.empty((rows,), dtype=torch.float32, device=O.device)
    ctx.check(lib().pa_cuda_normalize(ctx.handle, hd, rows, _ptr(O), _ptr(m), _ptr(l), _ptr(Oh), _ptr(lse),
                                      _stream_ptr(stream)), "normalize")
    return Oh, lse


def fold_reply(ctx: Context, hd: int, Oh, lse, O, m, l, stream=None):
    """Fold a normalised reply (f16 Oh [rows][hd], lse [rows]) into the unnormalised partial (O, m, l) in place, as
    the co-attention slot O_unnorm = Oh, l = 1, m = lse (pa_cuda_fold_reply)."""
    rows = lse.numel()
    ctx.check(lib().pa_cuda_fold_reply(ctx.handle, hd, rows, _ptr(Oh), _ptr(lse), _ptr(O), _ptr(m), _ptr(l),
                                       _stream_ptr(stream)), "fold_reply")
    return O, m, l


def nccl_unique_id() -> bytes:
    """The NCCL unique id (128 bytes) one rank creates and every rank passes to NcclComm (pa_cuda_nccl_unique_id)."""
    buf = ctypes.create_string_buffer(128)
    rc = lib().pa_cuda_nccl_unique_id(buf, 128)
    if rc != OK:
        raise PaCudaError(rc, "pa_cuda_nccl_unique_id: NCCL could not be opened or failed")
    return buf.raw


class NcclComm:
    """A communicator of the position-shard ranks over the context's device (pa_cuda_nccl_comm_create)."""

    def __init__(self, ctx: Context, uid: bytes, rank: int, world: int):
        self.ctx = ctx
        h = ctypes.c_void_p()
        idbuf = ctypes.create_string_buffer(bytes(uid), 128)
        ctx.check(lib().pa_cuda_nccl_comm_create(ctx.handle, idbuf, int(rank), int(world), ctypes.byref(h)),
                  "nccl_comm_create")
        self._h = h

    @property
    def handle(self):
        return self._h

    def close(self):
        if self._h:
            lib().pa_cuda_nccl_comm_destroy(self._h)
            self._h = None


def nccl_wait(ctx: Context, comm: NcclComm, stream=None, timeout_ms: int = 0):
    """Wait for the stream's work, aborting the communicator on an NCCL error or after timeout_ms (pa_cuda_nccl_wait)."""
    ctx.check(lib().pa_cuda_nccl_wait(ctx.handle, comm.handle, _stream_ptr(stream), int(timeout_ms)), "nccl_wait")


def shard_attn_allgather_merge(plan: Plan, Qs, comm: NcclComm, O, m, l, stream=None):
    """This rank's plan, one NCCL all-gather of every rank's packed (O, m, l), and their log-sum-exp fold into O, m, l
    (the same on every rank); pa_cuda_shard_attn_allgather_merge."""
    plan.ctx.check(lib().pa_cuda_shard_attn_allgather_merge(plan._h, _ptr(Qs), comm.handle, _ptr(O), _ptr(m), _ptr(l),
                                                            _stream_ptr(stream)), "shard_attn_allgather_merge")
    return O, m, l


def scale_q(ctx: Context, Q, scale: float, stream=None):
    """f16(Q * scale) on the device (pa_cuda_scale_q)."""
    import torch
    Qs = torch.empty(Q.shape, dtype=torch.float16, device=Q.device)
    ctx.check(lib().pa_cuda_scale_q(ctx.handle, _ptr(Q), float(scale), Q.numel(), _ptr(Qs), _stream_ptr(stream)),
              "scale_q")
    return Qs


class Engine:
    """pa::engine over libpacuda (phone-attn/phone-attn.h:166-183): engine-owned pages (host-writable, device-
    resident managed memory), begin() with host f16 Q [ng][nkv][48][hd], end() with host O/m/l."""

    NR = 48

    def __init__(self, ctx: Context):
        self.ctx = ctx
        self._pages = []

    def alloc_page(self, nbytes: int) -> _Page:
        p = _Page()
        self.ctx.check(lib().pa_cuda_alloc_page(self.ctx.handle, nbytes, ctypes.byref(p)), "alloc_page")
        self._pages.append(p)
        return p

    def free_page(self, p: _Page):
        lib().pa_cuda_free_page(self.ctx.handle, ctypes.byref(p))

    @staticmethod
    def page_view(p: _Page, nbytes: int, which: str = "k"):
        """A writable host view (numpy uint8) of a page's K or V memory."""
        import numpy as np
        addr = p.k if which == "k" else p.v
        return np.ctypeslib.as_array((ctypes.c_uint8 * nbytes).from_address(addr))

    def begin(self, pages: Sequence[_Page], nkeys: Sequence[int], Qs_host, shape: Shape, ng: int = 1, ntok: int = 8):
        arr = (_Page * max(1, len(pages)))(*pages)
        nk = (ctypes.c_uint32 * max(1, len(nkeys)))(*nkeys)
        sh = shape.c()
        self.ctx.check(lib().pa_cuda_begin(self.ctx.handle, arr, nk, len(pages), Qs_host.ctypes.data, ctypes.byref(sh),
                                           ng, ntok), "begin")

    def end(self, O, m, l) -> float:
        ms = lib().pa_cuda_end(self.ctx.handle, O.ctypes.data, m.ctypes.data, l.ctypes.data)
        if ms < 0:
            msg = lib().pa_cuda_last_error(self.ctx.handle).decode(errors="replace")
            raise PaCudaError(ETIMEOUT, f"end: {msg}")
        return ms

    def arm(self, pages: Sequence[_Page], nkeys: Sequence[int], shape: Shape, ntok: int = 8):
        """engine::arm: prepare the likely next one-group call (its plan and a CUDA graph of the whole call)."""
        arr = (_Page * max(1, len(pages)))(*pages)
        nk = (ctypes.c_uint32 * max(1, len(nkeys)))(*nkeys)
        sh = shape.c()
        self.ctx.check(lib().pa_cuda_arm(self.ctx.handle, arr, nk, len(pages), ctypes.byref(sh), ntok), "arm")

    @property
    def graph_calls(self) -> int:
        """begin calls served by an armed graph"""
        return int(lib().pa_cuda_graph_calls(self.ctx.handle))

    @property
    def exec_ms(self) -> float:
        return float(lib().pa_cuda_exec_ms(self.ctx.handle))


# ---------------------------------------------------------------- paged cache
def _want(ctx: Context, t, name: str, dtype, shape):
    """Pointer of a contiguous tensor of this type and shape on the context's device; anything else is an error."""
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous() or t.get_device() != ctx.device:
        raise PaCudaError(EINVAL, f"{name}: needs a contiguous {dtype} tensor {shape} on cuda:{ctx.device}, got "
                                  f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _layer(cache, layer: int) -> int:
    if not 0 <= layer < cache.n_layers:   # (ctypes would take it modulo 2^32)
        raise PaCudaError(EINVAL, f"layer {layer} of a cache of {cache.n_layers}")
    return layer


def _stream_on(ctx: Context, stream):
    """_stream_ptr for the context's device, whatever the current one is; and the torch stream where it is another than the
    device's current one (else None)."""
    import torch
    here = torch._C._cuda_getCurrentRawStream(ctx.device) or 1   # (current_stream's handle, without its Stream object)
    if stream is None:
        return here, None
    if isinstance(stream, torch.cuda.Stream) and stream.device_index != ctx.device:
        raise PaCudaError(EINVAL, f"the stream is on cuda:{stream.device_index}, the context on cuda:{ctx.device}")
    h = int(getattr(stream, "cuda_stream", stream)) or 1     # (1: cudaStreamLegacy, torch's default stream)
    if h == here:
        return h, None
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.default_stream(ctx.device) if h == 1 else torch.cuda.ExternalStream(h, device=ctx.device)
    return h, stream


def _there(side, like, *kinds):
    """Outputs (shape, type) on like's device, for a call on a stream of its own: allocated on that stream, since memory of the
    current one may still be read by work that is queued on it, and held for the current stream's use too."""
    import torch
    with torch.cuda.stream(side):
        out = tuple(like.new_empty(shape, dtype=dtype) for shape, dtype in kinds)
    for t in out:
        t.record_stream(torch.cuda.current_stream(t.device))
    return out


def _keep(side, *tensors):
    """What a call on a stream of its own reads and writes is not given out again before that stream is done with it. Only for
    streams that torch owns: the allocator uses the stream when the tensor is freed (a cache's rows perhaps long after), and
    another's may have been destroyed by then."""
    import torch
    if not isinstance(side, torch.cuda.ExternalStream):
        for t in tensors:
            if t is not None:
                t.record_stream(side)


class Cache:
    """A paged device cache (pa_cuda_cache): K and V uint8 [n_layers][n_pages][page_keys][row bytes] on one device, rows of
    nkv heads in the F16, Q8_0 or Q4_0 format. Tables, lengths and positions stay with the caller.

    The calls on a cache run on torch's current stream or on `stream`, whose order with other streams is the caller's. With a
    torch stream the tensors may be dropped as soon as a call returns; with another's stream (a handle, an ExternalStream)
    the caller keeps them until the call has run."""

    def __init__(self, hd: int, nkv: int, quant: int = Q8_0, n_layers: int = 1, n_pages: int = 1, page_keys: int = 256,
                 device: int = 0, rs: int | None = None):
        import torch
        hb = head_bytes(quant, hd)
        rs = rs if rs is not None else (nkv * hb + 15) // 16 * 16
        K = torch.zeros((n_layers, n_pages, page_keys, rs), dtype=torch.uint8, device=f"cuda:{device}")
        self._set(K, torch.zeros_like(K), hd, nkv, quant)

    @classmethod
    def of(cls, K, V, hd: int, nkv: int, quant: int) -> "Cache":
        """The same over tensors the caller holds."""
        c = cls.__new__(cls)
        c._set(K, V, hd, nkv, quant)
        return c

    def _set(self, K, V, hd, nkv, quant):
        import torch
        for name, t in (("K", K), ("V", V)):
            if t.dtype is not torch.uint8 or t.dim() != 4 or not t.is_contiguous() or not t.is_cuda:
                raise PaCudaError(EINVAL, f"cache {name}: needs a contiguous CUDA uint8 tensor [layers][pages][page_keys]"
                                          f"[row bytes], got {t.dtype} {tuple(t.shape)}")
        if K.shape != V.shape or K.device != V.device:
            raise PaCudaError(EINVAL, "cache K and V differ in shape or device")
        self.K, self.V, self.hd, self.nkv, self.quant = K, V, hd, nkv, quant
        self.n_layers, self.n_pages, self.page_keys, self.rs = K.shape
        self.hb = head_bytes(quant, hd)
        self.device = K.get_device()
        self._c = ctypes.byref(_Cache(K.data_ptr(), V.data_ptr(), self.n_layers, self.n_pages, self.page_keys))

    def shape(self, rows: int):
        """A reference to the C geometry with this many query rows per KV head."""
        return ctypes.byref(_Shape(self.hd, self.nkv, rows, self.quant, self.rs, self.hb))

    def on(self, ctx: Context):
        if self.device != ctx.device:
            raise PaCudaError(EINVAL, f"the cache is on cuda:{self.device}, the context on cuda:{ctx.device}")
        return self._c


class CachePlan:
    """Attention of n_sets sequences x n_tok query tokens over a paged cache (pa_cuda_cache_plan_create): causal, with a
    sliding window and sinks (window > 0), or for drafted tokens that form a tree (tree=True). One call at a time."""

    def __init__(self, ctx: Context, cache: Cache, n_sets: int, n_tok: int, gqa: int, max_pages: int, window: int = 0,
                 sinks: int = 0, tree: bool = False):
        self.ctx, self.cache, self.n_sets, self.n_tok, self.gqa = ctx, cache, n_sets, n_tok, gqa
        self.max_pages, self.tree = max_pages, bool(tree)
        self._h = _P()
        for name, x in dict(n_sets=n_sets, n_tok=n_tok, gqa=gqa, max_pages=max_pages, window=window, sinks=sinks,
                            rows=gqa * n_tok).items():
            if not 0 <= x < 1 << 32:   # (ctypes would take it modulo 2^32)
                raise PaCudaError(EINVAL, f"CachePlan: {name} = {x}")
        mask = _Mask(n_tok, window, sinks, 1 if tree else 0)
        ctx.check(lib().pa_cuda_cache_plan_create(ctx.handle, cache.shape(gqa * n_tok), cache.on(ctx), n_sets, max_pages,
                                                  ctypes.byref(mask), ctypes.byref(self._h)), "cache_plan_create")
        self._rows = (n_sets, cache.nkv, gqa * n_tok)
        self._full = self._rows + (cache.hd,)

    @property
    def kernel(self) -> str:
        """Name of the attention kernel the plan launches."""
        return lib().pa_cuda_cache_plan_kernel(self._h).decode()

    def _args(self, layer, Qs, table, n_keys, q_pos, tree):
        import torch
        ctx, i32, per = self.ctx, torch.int32, (self.n_sets,)
        if (tree is not None) != self.tree:
            raise PaCudaError(EINVAL, "a tree plan takes the tree's masks, another plan none")
        return (self._h, _layer(self.cache, layer), _want(ctx, Qs, "Qs", torch.float16, self._full),
                _want(ctx, table, "table", i32, (self.n_sets, self.max_pages)), _want(ctx, n_keys, "n_keys", i32, per),
                None if q_pos is None else _want(ctx, q_pos, "q_pos", i32, per),
                None if tree is None else _want(ctx, tree, "tree", torch.int64, (self.n_sets, self.n_tok)))

    def run(self, layer: int, Qs, table, n_keys, q_pos=None, tree=None, out=None, stream=None):
        """The unnormalised partial (O, m, l) (pa_cuda_cache_attn). Qs: f16(q * scale) [n_sets][nkv][gqa * n_tok][hd],
        row g * n_tok + t; table int32 [n_sets][max_pages]; n_keys, q_pos int32 [n_sets]; tree int64 [n_sets][n_tok]."""
        import torch
        ctx, f32 = self.ctx, torch.float32
        args = self._args(layer, Qs, table, n_keys, q_pos, tree)
        st, side = _stream_on(ctx, stream)
        if out is None and side is None:
            m = Qs.new_empty(self._rows, dtype=f32)
            out = Qs.new_empty(self._full, dtype=f32), m, torch.empty_like(m)
        elif out is None:
            out = _there(side, Qs, (self._full, f32), (self._rows, f32), (self._rows, f32))
        else:
            for t, name, shape in zip(out, ("O", "m", "l"), (self._full, self._rows, self._rows)):
                _want(ctx, t, name, f32, shape)
        O, m, l = out
        ctx.check(lib().pa_cuda_cache_attn(*args, O.data_ptr(), m.data_ptr(), l.data_ptr(), st), "cache_attn")
        if side is not None:
            _keep(side, Qs, table, n_keys, q_pos, tree, *out, self.cache.K, self.cache.V)
        return O, m, l

    def reply(self, layer: int, Qs, table, n_keys, q_pos=None, tree=None, out=None, stream=None):
        """The same, normalised: (f16 O / l, lse) (pa_cuda_cache_attn_reply)."""
        import torch
        ctx = self.ctx
        args = self._args(layer, Qs, table, n_keys, q_pos, tree)
        st, side = _stream_on(ctx, stream)
        if out is None and side is None:
            out = torch.empty_like(Qs), Qs.new_empty(self._rows, dtype=torch.float32)
        elif out is None:
            out = _there(side, Qs, (self._full, torch.float16), (self._rows, torch.float32))
        else:
            _want(ctx, out[0], "Oh", torch.float16, self._full)
            _want(ctx, out[1], "lse", torch.float32, self._rows)
        Oh, lse = out
        ctx.check(lib().pa_cuda_cache_attn_reply(*args, Oh.data_ptr(), lse.data_ptr(), st), "cache_attn_reply")
        if side is not None:
            _keep(side, Qs, table, n_keys, q_pos, tree, *out, self.cache.K, self.cache.V)
        return Oh, lse

    def close(self):
        if self._h:
            lib().pa_cuda_cache_plan_destroy(self._h)
            self._h = _P()

    def __del__(self):  # pragma: no cover
        try:
            self.close()
        except Exception:
            pass


_kinds = {}


def _kinds_of(torch):
    """PA_CUDA_T_* of the types cache_append takes."""
    _kinds.update({torch.float16: 0, torch.bfloat16: 1, torch.float32: 2})
    return _kinds


def cache_append(ctx: Context, cache: Cache, layer: int, q, k, v, table, start, pos=None, wq=None, wk=None, freqs=None,
                 eps: float = 1e-6, scale: float = 1.0, interleaved: bool = False, out=None, stream=None):
    """Head norm and rotation of new queries and keys, and the append of their rows (pa_cuda_cache_append). q
    [n_sets][n_tok][nkv * gqa][hd], k, v [n_sets][n_tok][nkv][hd]: f16, bf16 or f32, any strides over sets and tokens; wq, wk
    [hd]; freqs float64 [rot / 2]; table int32 [n_sets][max_pages]; start int32 [n_sets]: key index of token 0; pos int32
    [n_sets][n_tok] (< 0: padding). Returns Qs f16 [n_sets][nkv][gqa * n_tok][hd], what CachePlan takes."""
    import torch
    kinds = _kinds or _kinds_of(torch)
    S, T, nq, hd = q.shape
    kv, dt, dev = (S, T, cache.nkv, cache.hd), q.dtype, ctx.device
    if hd != cache.hd or nq == 0 or nq % cache.nkv or k.shape != kv or v.shape != kv or dt not in kinds:
        raise PaCudaError(EINVAL, f"cache_append: q {tuple(q.shape)} {dt}, k {tuple(k.shape)}, v {tuple(v.shape)} do not fit "
                                  f"nkv {cache.nkv}, hd {cache.hd} (f16, bf16 or f32)")
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if (qs[3] != 1 or ks[3] != 1 or vs[3] != 1 or (qs[2] != hd and nq > 1) or ((ks[2] != hd or vs[2] != hd) and kv[2] > 1) or
            k.dtype is not dt or v.dtype is not dt or q.get_device() != dev or k.get_device() != dev or v.get_device() != dev):
        raise PaCudaError(EINVAL, f"cache_append: q, k and v need one type and heads of hd consecutive elements, hd apart, on "
                                  f"cuda:{dev}")
    w_dtype = kinds[dt]
    if wq is not None or wk is not None:
        w = wk if wq is None else wq
        w_dtype = kinds.get(w.dtype, 3)
        if wq is not None:
            _want(ctx, wq, "wq", w.dtype, (hd,))
        if wk is not None:
            _want(ctx, wk, "wk", w.dtype, (hd,))
    rot = 0 if freqs is None else 2 * freqs.shape[0]
    a = _Append(q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1],
                None if wq is None else wq.data_ptr(), None if wk is None else wk.data_ptr(),
                None if freqs is None else _want(ctx, freqs, "freqs", torch.float64, (rot // 2,)),
                None if pos is None else _want(ctx, pos, "pos", torch.int32, (S, T)),
                kinds[dt], w_dtype, rot, 1 if interleaved else 0, eps, scale)
    n_rows = nq // cache.nkv * T
    rows = (S, cache.nkv, n_rows, hd)
    st, side = _stream_on(ctx, stream)
    if out is None:
        out = q.new_empty(rows, dtype=torch.float16) if side is None else _there(side, q, (rows, torch.float16))[0]
    else:
        _want(ctx, out, "out", torch.float16, rows)
    pages = table.shape[-1]
    ctx.check(lib().pa_cuda_cache_append(ctx.handle, cache.shape(n_rows or 1), cache.on(ctx), _layer(cache, layer),
                                         ctypes.byref(a), S, T,
                                         _want(ctx, table, "table", torch.int32, (S, pages)), pages,
                                         _want(ctx, start, "start", torch.int32, (S,)),
                                         out.data_ptr(), st), "cache_append")
    if side is not None:
        _keep(side, q, k, v, table, start, pos, wq, wk, freqs, out, cache.K, cache.V)
    return out


def cache_rows(ctx: Context, cache: Cache, layer: int, table, first, n: int, out=None, stream=None):
    """Keys first[s] .. first[s] + n - 1 of every sequence as the f16 values their rows stand for: (K, V)
    [n_sets][n][nkv][hd] (pa_cuda_cache_rows)."""
    import torch
    S = table.shape[0]
    shape = (S, n, cache.nkv, cache.hd)
    st, side = _stream_on(ctx, stream)
    if out is None and side is None:
        K = table.new_empty(shape, dtype=torch.float16)
        out = (K, torch.empty_like(K))
    elif out is None:
        out = _there(side, table, (shape, torch.float16), (shape, torch.float16))
    else:
        _want(ctx, out[0], "K", torch.float16, shape)
        _want(ctx, out[1], "V", torch.float16, shape)
    ctx.check(lib().pa_cuda_cache_rows(ctx.handle, cache.shape(1), cache.on(ctx), _layer(cache, layer), S, n,
                                       _want(ctx, table, "table", torch.int32, (S, table.shape[1])), table.shape[1],
                                       _want(ctx, first, "first", torch.int32, (S,)),
                                       out[0].data_ptr(), out[1].data_ptr(), st), "cache_rows")
    if side is not None:
        _keep(side, table, first, *out, cache.K, cache.V)
    return out


def cache_copy_pages(ctx: Context, cache: Cache, src, dst, stream=None):
    """Pages src[i] -> dst[i] (int32 [n]) of every layer, K and V (pa_cuda_cache_copy_pages): a sequence forked off a shared
    prefix copies the page it will write to. No page is both read and written in one call."""
    import torch
    n = src.numel()
    st, side = _stream_on(ctx, stream)
    ctx.check(lib().pa_cuda_cache_copy_pages(ctx.handle, cache.shape(1), cache.on(ctx),
                                             _want(ctx, src, "src", torch.int32, (n,)),
                                             _want(ctx, dst, "dst", torch.int32, (n,)), n, st),
              "cache_copy_pages")
    if side is not None:
        _keep(side, src, dst, cache.K, cache.V)


def cache_compact(ctx: Context, cache: Cache, table, start, path, count, out=None, stream=None):
    """Keeps the accepted rows of a verified draft (pa_cuda_cache_compact): rows start[s] + path[s][i] move to start[s] + i,
    i < count[s], in every layer. start, count int32 [n_sets], path int32 [n_sets][n_tok], rising. Returns the new n_keys,
    start + count."""
    import torch
    S, T = path.shape
    st, side = _stream_on(ctx, stream)
    if out is None:
        out = torch.empty_like(start) if side is None else _there(side, start, (start.shape, start.dtype))[0]
    ctx.check(lib().pa_cuda_cache_compact(ctx.handle, cache.shape(1), cache.on(ctx), S, T,
                                          _want(ctx, table, "table", torch.int32, (S, table.shape[1])), table.shape[1],
                                          _want(ctx, start, "start", torch.int32, (S,)),
                                          _want(ctx, path, "path", torch.int32, (S, T)),
                                          _want(ctx, count, "count", torch.int32, (S,)),
                                          _want(ctx, out, "out", torch.int32, (S,)), st),
              "cache_compact")
    if side is not None:
        _keep(side, table, start, path, count, out, cache.K, cache.V)
    return out

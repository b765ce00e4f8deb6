"""ctypes binding of libq3cu.so (the C ABI in include/q3cu.h) over torch tensors.

torch is used only for device memory and streams; every op runs the library's
own sm_100a kernels.  There is no fallback: if the shared library is missing or
no sm_100 GPU is present, the calls raise.
"""
from __future__ import annotations

import ctypes as C
import os
import re
import threading

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libq3cu.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "q3cu.h")

F32, BF16, Q8_0 = 0, 1, 8
GS = 64
DEV_BAD_INDEX, DEV_TIMEOUT = 0x1, 0x2
STATUS = {0: "OK", 1: "ERR_INVALID", 2: "ERR_ALIGN", 3: "ERR_GROUP", 4: "ERR_CUDA", 5: "ERR_INDEX",
          6: "ERR_TIMEOUT", 7: "ERR_NOT_INIT", 8: "ERR_OOM", 9: "ERR_DEVICE", 10: "ERR_FORMAT"}

_lib = None
_lock = threading.Lock()


class Q3Error(RuntimeError):
    def __init__(self, status: int, op: str, msg: str):
        super().__init__(f"{op}: {STATUS.get(status, status)}: {msg}")
        self.status = status


class _KVCache(C.Structure):             # q3cu_kv_cache
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("page_stride", C.c_int64), ("n_pages", C.c_int32),
                ("n_kv", C.c_int32), ("page_size", C.c_int32), ("head_dim", C.c_int32), ("dtype", C.c_int32)]


class _KVCacheQ8(_KVCache):              # q3cu_kv_cache_q8: behind its first member
    _fields_ = [("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("scale_stride", C.c_int64)]


class _Rope(C.Structure):                # q3cu_rope
    _fields_ = [("theta", C.c_float), ("dim", C.c_int32), ("layout", C.c_int32), ("scaling", C.c_int32),
                ("factor", C.c_float), ("original", C.c_float), ("beta_fast", C.c_float), ("beta_slow", C.c_float),
                ("gain", C.c_float), ("freq", C.POINTER(C.c_double))]


class _KVBatch(C.Structure):             # q3cu_kv_batch
    _fields_ = [("row_off", C.c_void_p), ("kv_len", C.c_void_p), ("pages", C.c_void_p), ("n_seqs", C.c_int32),
                ("max_pages", C.c_int32)]


class _KVPrefix(C.Structure):            # q3cu_kv_prefix
    _fields_ = [("seq_off", C.c_void_p), ("len", C.c_void_p), ("n_groups", C.c_int32)]


def header_functions(path: str = HEADER) -> list[str]:
    """Names of the entry points declared in include/q3cu.h."""
    text = open(path).read()
    return sorted(set(re.findall(r"\b(q3cu_[a-z0-9_]+)\s*\(", text)))


def load_library(path: str = LIB_PATH) -> C.CDLL:
    global _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(path):
                raise ImportError(f"{path} is missing: run __graft_entry__.build() (make -C metalqwen3_b200/csrc)")
            lib = C.CDLL(path)
            vp, i32, i64, f32 = C.c_void_p, C.c_int, C.c_int64, C.c_float
            st = C.c_int
            sigs = {
                "q3cu_init": (st, [i32, C.POINTER(vp)]),
                "q3cu_destroy": (st, [vp]),
                "q3cu_is_initialized": (i32, [vp]),
                "q3cu_last_error_string": (C.c_char_p, []),
                "q3cu_status_string": (C.c_char_p, [st]),
                "q3cu_version": (i32, []),
                "q3cu_device_status": (st, [vp, vp, C.POINTER(C.c_uint32)]),
                "q3cu_selftest_wait_timeout": (st, [vp, vp]),
                "q3cu_check_header": (st, [vp, C.c_size_t, vp]),
                "q3cu_rmsnorm": (st, [vp, vp, i32, vp, i64, i32, f32, vp, vp]),
                "q3cu_rmsnorm_q8": (st, [vp, vp, i32, vp, i64, i32, f32, vp, vp, vp]),
                "q3cu_qk_norm_rope": (st, [vp, vp, vp, i32, vp, i64, i32, i32, i32, vp, vp, f32, f32, vp]),
                "q3cu_swiglu": (st, [vp, vp, vp, i32, i64, i32, vp]),
                "q3cu_swiglu_q8": (st, [vp, vp, vp, i32, i64, i32, vp, vp, vp]),
                "q3cu_softmax_rows": (st, [vp, vp, vp, vp, i64, vp]),
                "q3cu_quantize_q8": (st, [vp, vp, i32, i64, i32, vp, vp, vp]),
                "q3cu_dequantize_q8": (st, [vp, vp, vp, i64, vp, vp]),
                "q3cu_embed_gather": (st, [vp, vp, vp, i32, i32, vp, i64, vp, vp, vp, vp]),
                "q3cu_matmul_q8": (st, [vp, vp, vp, i32, vp, vp, i32, i32, vp, vp]),
                "q3cu_execute_quantized_matmul": (st, [vp, vp, vp, vp, vp, vp, i32, i32, i32]),
                "q3cu_attention": (st, [vp, vp, vp, vp, i32, i32, i32, i32, vp, i32, vp, vp, vp]),
                "q3cu_kv_append": (st, [vp, C.POINTER(_KVCache), C.POINTER(_KVBatch), i64, vp, vp, vp, i32, i64, i64,
                                        i32, vp, vp, f32, f32, vp, i32, vp]),
                "q3cu_kv_append_rope": (st, [vp, C.POINTER(_KVCache), C.POINTER(_KVBatch), i64, vp, vp, vp, i32, i64, i64,
                                             i32, vp, vp, C.POINTER(_Rope), f32, vp, i32, vp]),
                "q3cu_kv_read": (st, [vp, C.POINTER(_KVCache), C.POINTER(_KVBatch), i64, vp, vp, i32, i64, vp]),
                "q3cu_attention_paged": (st, [vp, C.POINTER(_KVCache), C.POINTER(_KVBatch), vp, i32, i64, i32, vp,
                                              C.c_size_t, vp, vp]),
                "q3cu_attention_paged_workspace": (st, [vp, i32, i32, C.POINTER(C.c_size_t)]),
                "q3cu_attention_shared": (st, [vp, C.POINTER(_KVCache), C.POINTER(_KVBatch), C.POINTER(_KVPrefix), vp, i32,
                                               i64, i32, vp, C.c_size_t, vp, vp]),
                "q3cu_attention_shared_workspace": (st, [vp, i32, i32, i32, C.POINTER(C.c_size_t)]),
                "q3cu_attention_prompt": (st, [vp, C.POINTER(_KVCache), C.POINTER(_KVBatch), i64, vp, i32, i64, i32,
                                               vp, vp]),
                "q3cu_execute_attention": (st, [vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, i32, C.c_uint64,
                                                i32]),
                "q3cu_model_load": (st, [vp, vp, C.c_size_t, i32, C.POINTER(vp)]),
                "q3cu_model_config": (st, [vp, vp]),
                "q3cu_model_forward": (st, [vp, i32, i32, vp, vp]),
                "q3cu_model_logits": (vp, [vp]),
                "q3cu_model_destroy": (st, [vp]),
                "q3cu_execute_rmsnorm": (st, [vp, vp, vp, vp, i32]),
                "q3cu_execute_softmax": (st, [vp, vp, i32]),
                "q3cu_execute_swiglu": (st, [vp, vp, vp, i32]),
                "q3cu_execute_rope": (st, [vp, vp, vp, i32, i32, i32, i32, vp, vp]),
                "q3cu_execute_quantize": (st, [vp, vp, vp, vp, i32]),
                "q3cu_execute_embedding": (st, [vp, vp, vp, vp, i32, i32]),
            }
            for name, (res, args) in sigs.items():
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            _lib = lib
    return _lib


def _ptr(t):
    if t is None:
        return None
    if hasattr(t, "data_ptr"):
        return C.c_void_p(t.data_ptr())
    return C.c_void_p(t.ctypes.data)      # numpy (host-pointer wrappers)


def _dtype(t):
    import torch
    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.bfloat16:
        return BF16
    raise TypeError(f"unsupported dtype {t.dtype}")


def _tensor(t, what, dtype=None, shape=None, device=None):
    """Checks a device tensor's type and shape (None: any)."""
    if not t.is_cuda or (device is not None and t.get_device() != device):
        raise ValueError(f"{what} must be on the context's GPU, it is on {t.device}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, it is {t.dtype}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{what} must be {list(shape)}, it is {list(t.shape)}")
    return t


def _rows(t, what, dtype, heads, rows, device):
    """Checks t [rows][heads][128] (heads or rows None: any) with dense heads; returns (row stride in elements, rows,
    heads, pointer)."""
    shape = t.shape
    if len(shape) == 3 and t.get_device() == device and (dtype is None or t.dtype is dtype):
        n, h, d = shape
        row, head, element = t.stride()
        if d == 128 and (heads is None or h == heads) and (rows is None or n == rows) and (
                element == 1 and (head == 128 or h < 2) or n * h == 0):
            return row if n > 1 or row > h * 128 else h * 128, n, h, t.data_ptr()
    if len(shape) != 3 or shape[2] != 128 or (heads is not None and shape[1] != heads) or (
            rows is not None and shape[0] != rows):
        raise ValueError(f"{what} must be [{'rows' if rows is None else rows}][{'heads' if heads is None else heads}]"
                         f"[128], it is {list(shape)}")
    if t.get_device() != device:                    # -1 on the CPU
        raise ValueError(f"{what} must be on the context's GPU, it is on {t.device}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, it is {t.dtype}")
    raise ValueError(f"{what}: the heads of a row must be contiguous, strides are {t.stride()}")


class KVCache:
    """One layer's paged key-value cache: k and v [n_pages][n_kv][page_size][128] of one type: f32, bf16 or, with the
    scales k_scale and v_scale [n_pages][n_kv][page_size][2] in f32, int8 codes (Q8_0).
    A page is dense; pages may lie further apart (the same stride in k and v, and in their scales)."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("k and v must be [n_pages][n_kv][page_size][128] of one type on one GPU")
        n_pages, n_kv, size, hd = k.shape
        if k.stride()[1:] != (size * hd, hd, 1) or v.stride()[1:] != k.stride()[1:] or (
                n_pages > 1 and k.stride(0) != v.stride(0)):
            raise ValueError("a page must be contiguous, and k and v have one page stride")
        _tensor(k, "k"), _tensor(v, "v")
        self.k, self.v, self.n_kv, self.device = k, v, n_kv, k.get_device()
        self.k_scale, self.v_scale = k_scale, v_scale
        pages = (k.data_ptr(), v.data_ptr(), k.stride(0) if n_pages > 1 else n_kv * size * hd, n_pages, n_kv, size, hd)
        self.quantised = str(k.dtype) == "torch.int8"
        if self.quantised:
            if k_scale is None or v_scale is None:
                raise ValueError("a Q8_0 cache needs k_scale and v_scale")
            shape = (n_pages, n_kv, size, hd // GS)
            for t, what in ((k_scale, "k_scale"), (v_scale, "v_scale")):
                if str(_tensor(t, what, None, shape, self.device).dtype) != "torch.float32":
                    raise TypeError(f"{what} must be torch.float32, it is {t.dtype}")
                if t.stride()[1:] != (size * shape[3], shape[3], 1) or (n_pages > 1 and t.stride(0) != k_scale.stride(0)):
                    raise ValueError("a page's scales must be contiguous, and k_scale and v_scale have one page stride")
            self.c = _KVCacheQ8(*pages, Q8_0, k_scale.data_ptr(), v_scale.data_ptr(),
                                k_scale.stride(0) if n_pages > 1 else n_kv * size * shape[3])
        else:
            if k_scale is not None or v_scale is not None:
                raise ValueError("scales belong to int8 codes")
            self.c = _KVCache(*pages, _dtype(k))
        self.ref = C.byref(self.c)


class Rope:
    """How kv_append rotates heads (q3cu_rope in include/q3cu.h): the first `dim` elements, by halves or interleaved
    (neighbouring pairs); `scaling` None, "linear" or "yarn" with its `factor` (and the `original` length); `gain` of
    cosines and sines (None: the scaling's own); or `freq`, dim / 2 radians a position, in place of theta and scaling."""

    SCALINGS = {None: 0, "linear": 1, "yarn": 2}

    def __init__(self, theta=1e6, dim=128, interleaved=False, scaling=None, factor=1.0, original=0, beta_fast=32.0,
                 beta_slow=1.0, gain=None, freq=None):
        if scaling not in self.SCALINGS:
            raise ValueError(f"scaling must be one of {list(self.SCALINGS)}, it is {scaling!r}")
        if gain is not None and not gain > 0:
            raise ValueError(f"gain must be positive, it is {gain}")
        if freq is not None:
            freq = [float(f) for f in freq]
            if 2 * len(freq) != dim:
                raise ValueError(f"freq must have dim / 2 = {dim // 2} values, it has {len(freq)}")
        self.freq = None if freq is None else (C.c_double * len(freq))(*freq)
        self.c = _Rope(theta, dim, int(bool(interleaved)), self.SCALINGS[scaling], factor, original, beta_fast, beta_slow,
                       0.0 if gain is None else gain, self.freq)
        self.ref = C.byref(self.c)


class KVBatch:
    """The sequences of a call: kv_len [n_seqs], pages [n_seqs][max_pages] and, for packed rows, row_off
    [n_seqs + 1], all int32 on the GPU (the meaning of each: q3cu_kv_batch in include/q3cu.h)."""

    def __init__(self, kv_len, pages, row_off=None):
        n = kv_len.numel()
        i32 = kv_len.new_empty(0).int().dtype
        if pages.dim() != 2:
            raise ValueError(f"pages must be [n_seqs][max_pages], it is {list(pages.shape)}")
        self.device = kv_len.get_device()
        for t, what, shape in ((kv_len, "kv_len", (n,)), (pages, "pages", (n, pages.shape[1])), (row_off, "row_off", (n + 1,))):
            if t is not None and not _tensor(t, what, i32, shape, self.device).is_contiguous():
                raise ValueError(f"{what} must be contiguous")
        self.kv_len, self.pages, self.row_off = kv_len, pages, row_off
        self.c = _KVBatch(None if row_off is None else row_off.data_ptr(), kv_len.data_ptr(), pages.data_ptr(), n,
                          pages.shape[1])
        self.ref = C.byref(self.c)


class KVPrefix:
    """Groups of sequences that begin alike: seq_off [n_groups + 1] and length [n_groups], int32 on the GPU (the meaning
    of each: q3cu_kv_prefix in include/q3cu.h)."""

    def __init__(self, seq_off, length):
        n = length.numel()
        i32 = length.new_empty(0).int().dtype
        self.device = length.get_device()
        for t, what, shape in ((seq_off, "seq_off", (n + 1,)), (length, "length", (n,))):
            if not _tensor(t, what, i32, shape, self.device).is_contiguous():
                raise ValueError(f"{what} must be contiguous")
        self.seq_off, self.length = seq_off, length
        self.c = _KVPrefix(seq_off.data_ptr(), length.data_ptr(), n)
        self.ref = C.byref(self.c)


class Q3CU:
    """One library context on one device (not thread-safe)."""

    def __init__(self, device: int = 0):
        import torch
        self.torch = torch
        self.lib = load_library()
        self.device = device
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        torch.cuda.set_device(device)
        h = C.c_void_p()
        self._check(self.lib.q3cu_init(device, C.byref(h)), "q3cu_init")
        self.ctx = h

    # -- plumbing ------------------------------------------------------------
    def _check(self, status, op):
        if status != 0:
            raise Q3Error(status, op, (self.lib.q3cu_last_error_string() or b"").decode())

    def _stream(self, stream=None):
        if stream is not None:
            return stream.cuda_stream
        raw = self._raw_stream                  # the handle alone: a Stream object takes a microsecond to make
        return raw(self.device) if raw else self.torch.cuda.current_stream(self.device).cuda_stream

    def _make(self, stream, make, *args, **kwargs):
        """What a call makes for itself, by torch's function `make`.  Where a stream is given the memory is
        that stream's own: what lies free in the current stream's may still be in use by work that is pending there."""
        if stream is None:
            return make(*args, **kwargs)
        cuda = self.torch.cuda
        if not isinstance(stream, cuda.Stream):      # anything with a stream's handle
            stream = cuda.ExternalStream(stream.cuda_stream, self.device)
        with cuda.stream(stream):
            t = make(*args, **kwargs)
        t.record_stream(cuda.current_stream(self.device))       # where the caller may read it
        return t

    def close(self):
        if getattr(self, "ctx", None):
            self.lib.q3cu_destroy(self.ctx)
            self.ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def selftest_wait_timeout(self, stream=None) -> None:
        """Enqueue the failure-path self-test: a kernel whose bounded wait gives
        up (about 2 s) and sets the timeout bit; read it with device_status()."""
        self._check(self.lib.q3cu_selftest_wait_timeout(self.ctx, self._stream(stream)), "q3cu_selftest_wait_timeout")

    def device_status(self, stream=None) -> int:
        flags = C.c_uint32(0)
        st = self.lib.q3cu_device_status(self.ctx, self._stream(stream), C.byref(flags))
        if st not in (0, 5, 6):
            self._check(st, "q3cu_device_status")
        return flags.value

    # -- device-pointer ops ----------------------------------------------------
    def rmsnorm(self, x, w, eps=1e-6, out=None, stream=None):
        rows, dim = x.shape
        out = self._make(stream, self.torch.empty_like, x) if out is None else out
        self._check(self.lib.q3cu_rmsnorm(self.ctx, _ptr(x), _dtype(x), _ptr(w), rows, dim, eps, _ptr(out),
                                          self._stream(stream)), "q3cu_rmsnorm")
        return out

    def rmsnorm_q8(self, x, w, eps=1e-6, q=None, s=None, stream=None):
        rows, dim = x.shape
        if q is None:
            q = self._make(stream, self.torch.empty, (rows, dim), dtype=self.torch.int8, device=x.device)
        if s is None:
            s = self._make(stream, self.torch.empty, (rows, dim // GS), dtype=self.torch.float32, device=x.device)
        self._check(self.lib.q3cu_rmsnorm_q8(self.ctx, _ptr(x), _dtype(x), _ptr(w), rows, dim, eps, _ptr(q),
                                             _ptr(s), self._stream(stream)), "q3cu_rmsnorm_q8")
        return q, s

    def qk_norm_rope(self, q, k, pos, q_norm, k_norm, theta=1e6, eps=1e-6, stream=None):
        """In place.  q: [rows, n_heads, hd], k: [rows, n_kv, hd]."""
        rows, nh, hd = q.shape
        nkv = k.shape[1]
        self._check(self.lib.q3cu_qk_norm_rope(self.ctx, _ptr(q), _ptr(k), _dtype(q), _ptr(pos), rows, nh, nkv, hd,
                                               _ptr(q_norm), _ptr(k_norm), theta, eps, self._stream(stream)),
                    "q3cu_qk_norm_rope")
        return q, k

    def swiglu(self, hb, hb2, stream=None):
        rows, hidden = hb.shape
        self._check(self.lib.q3cu_swiglu(self.ctx, _ptr(hb), _ptr(hb2), _dtype(hb), rows, hidden,
                                         self._stream(stream)), "q3cu_swiglu")
        return hb

    def swiglu_q8(self, hb, hb2, q=None, s=None, stream=None):
        rows, hidden = hb.shape
        if q is None:
            q = self._make(stream, self.torch.empty, (rows, hidden), dtype=self.torch.int8, device=hb.device)
        if s is None:
            s = self._make(stream, self.torch.empty, (rows, hidden // GS), dtype=self.torch.float32, device=hb.device)
        self._check(self.lib.q3cu_swiglu_q8(self.ctx, _ptr(hb), _ptr(hb2), _dtype(hb), rows, hidden, _ptr(q), _ptr(s),
                                            self._stream(stream)), "q3cu_swiglu_q8")
        return q, s

    def softmax_rows(self, x, off, lens, stream=None):
        self._check(self.lib.q3cu_softmax_rows(self.ctx, _ptr(x), _ptr(off), _ptr(lens), off.numel(),
                                               self._stream(stream)), "q3cu_softmax_rows")
        return x

    def quantize_q8(self, x, q=None, s=None, stream=None):
        rows, n = x.shape
        q = self._make(stream, self.torch.empty, (rows, n), dtype=self.torch.int8, device=x.device) if q is None else q
        if s is None:
            s = self._make(stream, self.torch.empty, (rows, n // GS), dtype=self.torch.float32, device=x.device)
        self._check(self.lib.q3cu_quantize_q8(self.ctx, _ptr(x), _dtype(x), rows, n, _ptr(q), _ptr(s),
                                              self._stream(stream)), "q3cu_quantize_q8")
        return q, s

    def dequantize_q8(self, q, s, out=None, stream=None):
        n = q.numel()
        if out is None:
            out = self._make(stream, self.torch.empty, q.shape, dtype=self.torch.float32, device=q.device)
        self._check(self.lib.q3cu_dequantize_q8(self.ctx, _ptr(q), _ptr(s), n, _ptr(out), self._stream(stream)),
                    "q3cu_dequantize_q8")
        return out

    def embed_gather(self, tq, ts, ids, want_f32=True, want_q8=True, out=None, oq=None, os_=None, stream=None):
        vocab, dim = tq.shape
        n = ids.numel()
        T = self.torch
        if want_f32 and out is None:
            out = self._make(stream, T.empty, (n, dim), dtype=T.float32, device=tq.device)
        if want_q8 and oq is None:
            oq = self._make(stream, T.empty, (n, dim), dtype=T.int8, device=tq.device)
            os_ = self._make(stream, T.empty, (n, dim // GS), dtype=T.float32, device=tq.device)
        self._check(self.lib.q3cu_embed_gather(self.ctx, _ptr(tq), _ptr(ts), vocab, dim, _ptr(ids), n,
                                               _ptr(out if want_f32 else None), _ptr(oq if want_q8 else None),
                                               _ptr(os_ if want_q8 else None), self._stream(stream)),
                    "q3cu_embed_gather")
        return out, oq, os_

    def matmul_q8(self, xq, xs, wq, ws, out=None, stream=None):
        """out[b] = W @ x[b] for Q8_0 x (xq [B][n], xs [B][n/64]) and W (wq [d][n], ws [d][n/64])."""
        B, n = xq.shape
        d = wq.shape[0]
        if wq.shape[1] != n:
            raise ValueError(f"W is {tuple(wq.shape)}, x rows have {n} elements")
        if out is None:
            out = self._make(stream, self.torch.empty, (B, d), dtype=self.torch.float32, device=xq.device)
        self._check(self.lib.q3cu_matmul_q8(self.ctx, _ptr(xq), _ptr(xs), B, _ptr(wq), _ptr(ws), n, d, _ptr(out),
                                            self._stream(stream)), "q3cu_matmul_q8")
        return out

    def attention(self, q, key_cache, value_cache, pos, kv_mul, att=None, probs=None, xb=None, stream=None):
        """One token's attention over cache rows 0..pos: q [n_heads][128];
        key_cache / value_cache [rows][kv_dim]; att: scratch for the scores;
        returns (xb [n_heads][128], probs [n_heads][att_stride] with the
        probabilities in columns 0..pos)."""
        T = self.torch
        n_heads = q.numel() // 128
        kv_dim = key_cache.shape[-1]
        att = self._make(stream, T.zeros, (n_heads, pos + 1), dtype=T.float32, device=q.device) if att is None else att
        probs = self._make(stream, T.zeros_like, att) if probs is None else probs
        xb = self._make(stream, T.empty, (n_heads, 128), dtype=T.float32, device=q.device) if xb is None else xb
        self._check(self.lib.q3cu_attention(self.ctx, _ptr(q), _ptr(key_cache), _ptr(value_cache), pos, n_heads,
                                            kv_dim, kv_mul, _ptr(att), att.shape[-1], _ptr(probs), _ptr(xb),
                                            self._stream(stream)), "q3cu_attention")
        return xb, probs

    # -- the paged key-value cache -----------------------------------------------
    def _elsewhere(self, cache, batch, work=None, prefix=None):
        """Refuses what lies on another device than the context's, which its kernels could not reach."""
        for what, t in (("cache", cache), ("batch", batch), ("prefix", prefix)):
            if t is not None and t.device != self.device:
                raise ValueError(f"the {what} must be on the context's GPU, it is on cuda:{t.device}")
        raise ValueError(f"work must be contiguous memory on the context's GPU, it is on {work.device}")

    def kv_append(self, cache, batch, q, k, v, q_norm=None, k_norm=None, theta=1e6, eps=1e-6, q_out=None,
                  out_dtype=None, stream=None, rope=None):
        """QK-norm (where weights are given) and rotation (by `theta`, or as a Rope says) of the packed rows
        q [rows][n_heads][128] and k [rows][n_kv][128] (q may be None); keys and values into the cache; returns the
        rotated queries (q_out, or of out_dtype: by default the cache's type, bf16 for a Q8_0 cache).  q, k, v may be
        slices of one projection's rows."""
        dev, dtype = self.device, k.dtype
        if cache.device != dev or batch.device != dev:
            self._elsewhere(cache, batch)
        kv_stride, rows, _, kp = _rows(k, "k", None, cache.n_kv, None, dev)
        v_stride, _, _, vp = _rows(v, "v", dtype, cache.n_kv, rows, dev)
        if v_stride != kv_stride:
            raise ValueError("k and v must have one row stride")
        for w, what in ((q_norm, "q_norm"), (k_norm, "k_norm")):
            if w is not None and (w.dtype != self.torch.float32 or w.shape != (128,) or w.stride() != (1,)
                                  or w.get_device() != dev):
                raise ValueError(f"{what} must be 128 contiguous float32 on the context's GPU")
        q_stride, heads, qp, op, ot = 0, 0, None, None, F32
        if q is not None:
            q_stride, _, heads, qp = _rows(q, "q", dtype, None, rows, dev)
            if q_out is None:
                q_out = self._make(stream, self.torch.empty, (rows, heads, 128), device=q.device, dtype=out_dtype or (
                    self.torch.bfloat16 if cache.quantised else cache.k.dtype))
            _, _, _, op = _rows(q_out, "q_out", out_dtype, heads, rows, dev)
            if not q_out.is_contiguous():
                raise ValueError("q_out must be contiguous")
            ot = _dtype(q_out)
        call = self.lib.q3cu_kv_append if rope is None else self.lib.q3cu_kv_append_rope
        status = call(self.ctx, cache.ref, batch.ref, rows, qp, kp, vp, _dtype(k), q_stride, kv_stride,
                      heads, None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(),
                      theta if rope is None else rope.ref, eps, op, ot, self._stream(stream))
        if status:
            self._check(status, "q3cu_kv_append")
        return q_out

    def kv_read(self, cache, batch, rows=None, dtype=None, k_out=None, v_out=None, stream=None):
        """The packed rows' keys and values as the cache holds them: (k, v) [rows][n_kv][128], into k_out and v_out
        (f32 or bf16, rows may lie further apart) or new ones of `dtype` (the cache's type by default, bf16 for Q8_0; give
        `rows` then)."""
        dev = self.device
        if cache.device != dev or batch.device != dev:
            self._elsewhere(cache, batch)
        if (k_out is None) != (v_out is None) or (k_out is None and rows is None):
            raise ValueError("give k_out and v_out, or the number of rows")
        if k_out is None:
            dtype = dtype or (self.torch.bfloat16 if cache.quantised else cache.k.dtype)
            k_out, v_out = (self._make(stream, self.torch.empty, (rows, cache.n_kv, 128), dtype=dtype, device=cache.k.device)
                            for _ in range(2))
        stride, rows, _, kp = _rows(k_out, "k_out", dtype, cache.n_kv, rows, dev)
        v_stride, _, _, vp = _rows(v_out, "v_out", k_out.dtype, cache.n_kv, rows, dev)
        if v_stride != stride:
            raise ValueError("k_out and v_out must have one row stride")
        status = self.lib.q3cu_kv_read(self.ctx, cache.ref, batch.ref, rows, kp, vp, _dtype(k_out), stride,
                                       self._stream(stream))
        if status:
            self._check(status, "q3cu_kv_read")
        return k_out, v_out

    def attention_paged_workspace(self, cache, n_heads, stream=None):
        """A workspace for attention_paged with these head counts, for any batch; calls that may run at
        the same time (other streams, captured graphs replayed side by side) need one each.  `stream`: where it is
        used, if not on the current one."""
        n = C.c_size_t(0)
        self._check(self.lib.q3cu_attention_paged_workspace(self.ctx, n_heads, cache.n_kv, C.byref(n)),
                    "q3cu_attention_paged_workspace")
        return self._make(stream, self.torch.empty, n.value, dtype=self.torch.uint8, device=cache.k.device)

    def attention_paged(self, cache, batch, q, out=None, work=None, stream=None):
        """One new token per sequence: q [n_seqs][n_heads][128] over each sequence's kv_len positions."""
        if cache.device != self.device or batch.device != self.device or (
                work is not None and (work.get_device() != self.device or not work.is_contiguous())):
            self._elsewhere(cache, batch, work)
        stride, rows, heads, qp = _rows(q, "q", None, None, batch.c.n_seqs, self.device)
        if out is None:
            out = self._make(stream, self.torch.empty, (rows, heads, 128), dtype=q.dtype, device=q.device)
        elif not out.is_contiguous():
            raise ValueError("out must be contiguous")
        op = _rows(out, "out", q.dtype, heads, rows, self.device)[3]
        if work is None:
            work = self.attention_paged_workspace(cache, heads, stream)
        status = self.lib.q3cu_attention_paged(self.ctx, cache.ref, batch.ref, qp, _dtype(q), stride, heads,
                                               work.data_ptr(), work.nbytes, op, self._stream(stream))
        if status:
            self._check(status, "q3cu_attention_paged")
        return out

    def attention_shared_workspace(self, cache, n_seqs, n_heads, stream=None):
        """A workspace for attention_shared with these head counts and at most n_seqs sequences; calls that may run at
        the same time need one each.  `stream`: where it is used, if not on the current one."""
        n = C.c_size_t(0)
        self._check(self.lib.q3cu_attention_shared_workspace(self.ctx, n_seqs, n_heads, cache.n_kv, C.byref(n)),
                    "q3cu_attention_shared_workspace")
        return self._make(stream, self.torch.empty, n.value, dtype=self.torch.uint8, device=cache.k.device)

    def attention_shared(self, cache, batch, prefix, q, out=None, work=None, stream=None):
        """attention_paged where groups of sequences share their first positions (a KVPrefix), which are attended to once
        for the whole group; q and out bf16, the cache bf16 or Q8_0."""
        if cache.device != self.device or batch.device != self.device or prefix.device != self.device or (
                work is not None and (work.get_device() != self.device or not work.is_contiguous())):
            self._elsewhere(cache, batch, work, prefix)
        stride, rows, heads, qp = _rows(q, "q", None, None, batch.c.n_seqs, self.device)
        if out is None:
            out = self._make(stream, self.torch.empty, (rows, heads, 128), dtype=q.dtype, device=q.device)
        elif not out.is_contiguous():
            raise ValueError("out must be contiguous")
        op = _rows(out, "out", q.dtype, heads, rows, self.device)[3]
        if work is None:
            work = self.attention_shared_workspace(cache, rows, heads, stream)
        status = self.lib.q3cu_attention_shared(self.ctx, cache.ref, batch.ref, prefix.ref, qp, _dtype(q), stride, heads,
                                                work.data_ptr(), work.nbytes, op, self._stream(stream))
        if status:
            self._check(status, "q3cu_attention_shared")
        return out

    def attention_prompt(self, cache, batch, q, out=None, stream=None):
        """Causal attention of the packed rows q [rows][n_heads][128] (the cache's type, bf16 over a Q8_0 cache) over the
        cache, which holds their keys and values; rows behind the last sequence are not written."""
        if cache.device != self.device or batch.device != self.device:
            self._elsewhere(cache, batch)
        stride, rows, heads, qp = _rows(q, "q", None, None, None, self.device)
        if out is None:
            out = self._make(stream, self.torch.empty, (rows, heads, 128), dtype=q.dtype, device=q.device)
        elif not out.is_contiguous():
            raise ValueError("out must be contiguous")
        op = _rows(out, "out", q.dtype, heads, rows, self.device)[3]
        status = self.lib.q3cu_attention_prompt(self.ctx, cache.ref, batch.ref, rows, qp, _dtype(q), stride, heads, op,
                                                self._stream(stream))
        if status:
            self._check(status, "q3cu_attention_prompt")
        return out

    # -- host-pointer drop-in (numpy arrays, synchronous) -----------------------
    def execute_attention(self, xb, q, att, key_cache, value_cache, pos, head_dim, n_heads, n_kv_heads, seq_len,
                          kv_dim, loff, kv_mul):
        self._check(self.lib.q3cu_execute_attention(self.ctx, _ptr(xb), _ptr(q), _ptr(att), _ptr(key_cache),
                                                    _ptr(value_cache), pos, head_dim, n_heads, n_kv_heads, seq_len,
                                                    kv_dim, loff, kv_mul), "executeAttention")

    def execute_rmsnorm(self, out, inp, w):
        self._check(self.lib.q3cu_execute_rmsnorm(self.ctx, _ptr(out), _ptr(inp), _ptr(w), inp.size), "executeRMSNorm")

    def execute_softmax(self, x):
        self._check(self.lib.q3cu_execute_softmax(self.ctx, _ptr(x), x.size), "executeSoftmax")

    def execute_swiglu(self, hb, hb2):
        self._check(self.lib.q3cu_execute_swiglu(self.ctx, _ptr(hb), _ptr(hb2), hb.size), "executeSwiGLU")

    def execute_rope(self, q, k, head_dim, pos, n_heads, n_kv, qn, kn):
        self._check(self.lib.q3cu_execute_rope(self.ctx, _ptr(q), _ptr(k), head_dim, pos, n_heads, n_kv, _ptr(qn),
                                               _ptr(kn)), "executeRoPE")

    def execute_quantize(self, q, s, x):
        self._check(self.lib.q3cu_execute_quantize(self.ctx, _ptr(q), _ptr(s), _ptr(x), x.size), "executeQuantize")

    def execute_quantized_matmul(self, out, xq, xs, wq, ws, n, d, group_size=GS):
        self._check(self.lib.q3cu_execute_quantized_matmul(self.ctx, _ptr(out), _ptr(xq), _ptr(xs), _ptr(wq), _ptr(ws),
                                                           n, d, group_size), "executeQuantizedMatMul")

    def execute_embedding(self, out, tq, ts, token, dim):
        self._check(self.lib.q3cu_execute_embedding(self.ctx, _ptr(out), _ptr(tq), _ptr(ts), token, dim),
                    "executeEmbedding")


class Q3Model:
    """A checkpoint image (numpy uint8 array or bytes: the reference's file
    format) resident on the device of `q3` (a Q3CU context), with its KV cache;
    forward(token, pos) returns the logits as a numpy array."""

    def __init__(self, q3, image, ctx_length=0):
        import numpy as np
        self.q3, self.lib = q3, q3.lib
        self._img = np.ascontiguousarray(np.frombuffer(image, np.uint8) if isinstance(image, (bytes, bytearray))
                                         else image, np.uint8)
        self.m = C.c_void_p()
        q3._check(self.lib.q3cu_model_load(q3.ctx, self._img.ctypes.data, self._img.nbytes, ctx_length,
                                           C.byref(self.m)), "q3cu_model_load")
        cfg = (C.c_int32 * 12)()
        q3._check(self.lib.q3cu_model_config(self.m, cfg), "q3cu_model_config")
        keys = ("magic", "version", "dim", "hidden_dim", "n_layers", "n_heads", "n_kv_heads", "vocab_size",
                "seq_len", "head_dim", "shared_classifier", "group_size")
        self.config = dict(zip(keys, list(cfg)))
        self._img = None                      # the weights live on the device now

    def forward(self, token, pos, stream=None, to_host=True, out=None):
        """Logits of `token` at `pos` as a new float32 array, or into `out` (a
        C-contiguous float32 array of vocab_size, e.g. over pinned memory), or
        left on the device (to_host=False; see logits_ptr)."""
        import numpy as np
        if to_host and out is None:
            out = np.empty(self.config["vocab_size"], np.float32)
        if to_host and (out.dtype != np.float32 or out.size != self.config["vocab_size"]
                        or not out.flags["C_CONTIGUOUS"]):
            raise ValueError("out must be a C-contiguous float32 array of vocab_size elements")
        self.q3._check(self.lib.q3cu_model_forward(self.m, int(token), int(pos),
                                                   out.ctypes.data if to_host else None, self.q3._stream(stream)),
                       "q3cu_model_forward")
        return out if to_host else None

    def logits_ptr(self):
        return self.lib.q3cu_model_logits(self.m)

    def close(self):
        if self.m:
            self.lib.q3cu_model_destroy(self.m)
            self.m = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

"""tier_b200 -- B200-native (sm_100a) frozen-weight linear path of tierlm.

The product is the C ABI in include/tierk.h, implemented by libtierk.so (built
in-tree by ``python -m tier_b200.build``).  This module is its host-side mirror:
a ctypes binding of every entry point plus thin helpers that take torch
tensors for device memory and streams.  The operation names follow the
reference's C++ hot path (tier/tier.cpp): ``dequant`` = dq_launch (294-298),
``gemv`` = gemv_q / gemv<T> (300-306, 2261-2268), ``linear`` / ``linear_dx`` /
``linear_dx_acc`` = the linear operators (1202-1238), ``lmhead_*`` = the
chunked LM-head loops (3184-3266).

There is no CPU fallback: if libtierk.so is missing or fails to load, importing
the binding raises.
"""
from __future__ import annotations

import ctypes
import os
from pathlib import Path

_PKG = Path(__file__).resolve().parent
LIB_PATH = _PKG / "libtierk.so"

# status codes (tk_status)
TK_OK, TK_ERR_INVALID, TK_ERR_UNSUPPORTED, TK_ERR_CUDA, TK_ERR_NOMEM, TK_ERR_TIMEOUT, TK_ERR_DEVICE = range(7)
# block types = the reference's QT_* codes (tier/quant.h:20-23)
F32, F16, Q4_0, Q4_1, Q5_0, Q5_1, Q8_0 = 0, 1, 2, 3, 6, 7, 8
Q2_K, Q3_K, Q4_K, Q5_K, Q6_K, BF16, F16X2 = 10, 11, 12, 13, 14, 30, 100
IQ4_NL, IQ4_XS, TQ1_0, TQ2_0, MXFP4, NF4, FP4 = 20, 23, 34, 35, 39, 200, 201
# lattice types: decode after Context.set_iq_grids
IQ2_XXS, IQ2_XS, IQ3_XXS, IQ1_S, IQ3_S, IQ2_S, IQ1_M = 16, 17, 18, 19, 21, 22, 29
QTYPES = {"F32": F32, "F16": F16, "BF16": BF16, "Q4_0": Q4_0, "Q4_1": Q4_1, "Q5_0": Q5_0, "Q5_1": Q5_1,
          "Q8_0": Q8_0, "Q2_K": Q2_K, "Q3_K": Q3_K, "Q4_K": Q4_K, "Q5_K": Q5_K, "Q6_K": Q6_K,
          "IQ4_NL": IQ4_NL, "IQ4_XS": IQ4_XS, "TQ1_0": TQ1_0, "TQ2_0": TQ2_0, "MXFP4": MXFP4, "NF4": NF4, "FP4": FP4,
          "IQ2_XXS": IQ2_XXS, "IQ2_XS": IQ2_XS, "IQ2_S": IQ2_S, "IQ3_XXS": IQ3_XXS, "IQ3_S": IQ3_S, "IQ1_S": IQ1_S,
          "IQ1_M": IQ1_M}
BLOCK = {F32: (1, 4), F16: (1, 2), BF16: (1, 2), Q4_0: (32, 18), Q4_1: (32, 20), Q5_0: (32, 22), Q5_1: (32, 24),
         Q8_0: (32, 34), Q2_K: (256, 84), Q3_K: (256, 110), Q4_K: (256, 144), Q5_K: (256, 176), Q6_K: (256, 210),
         IQ4_NL: (32, 18), IQ4_XS: (256, 136), TQ1_0: (256, 54), TQ2_0: (256, 66), MXFP4: (32, 17),
         NF4: (64, 36), FP4: (64, 36),
         IQ2_XXS: (256, 66), IQ2_XS: (256, 74), IQ2_S: (256, 82), IQ3_XXS: (256, 98), IQ3_S: (256, 110),
         IQ1_S: (256, 50), IQ1_M: (256, 56)}
# activation dtypes
DT_F32, DT_F16, DT_BF16 = 0, 1, 2
# product sets
X3_AUTO, X3_REF, X3_HHL, X2, X1 = 0, 1, 2, 3, 4
QFUSED = 0x100   # OR into `products`: decode a quantized W inside the GEMM
IPC_HANDLE_BYTES = 64   # TK_IPC_HANDLE_BYTES
WFROZEN = 0x200  # OR into tk_gemv's qtype: W is never written by earlier kernels (early weight fetch)
WREUSE = 0x400   # OR into linear products: reuse the previous call's fp16 expansion of the same (unchanged) W
# kernel families for profiling
PROF_GEMM, PROF_DEQUANT, PROF_SPLIT, PROF_GEMV, PROF_LMHEAD, PROF_COMM, PROF_SERVE = range(7)


class TierkError(RuntimeError):
    def __init__(self, status: int, msg: str):
        super().__init__(f"tierk status {status}: {msg}")
        self.status = status


class Weight(ctypes.Structure):
    """tk_weight: a frozen W[rows, cols] resident on the device."""
    _fields_ = [("qtype", ctypes.c_int), ("rows", ctypes.c_int), ("cols", ctypes.c_int),
                ("scale_log2", ctypes.c_int), ("row_bytes", ctypes.c_size_t), ("data", ctypes.c_void_p)]


class IqGrids(ctypes.Structure):
    """tk_iq_grids: host pointers to the six lattice tables (int8)."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("iq2xxs", "iq2xs", "iq2s", "iq3xxs", "iq3s", "iq1s")]


class KvCache(ctypes.Structure):
    """tk_kvcache: one layer's 4-bit key/value cache on the device."""
    _device = None         # where make_kvcache's tensors are
    _fields_ = [("n_pages", ctypes.c_int), ("page_tokens", ctypes.c_int), ("n_kv_heads", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("k_q", ctypes.c_void_p), ("k_s", ctypes.c_void_p),
                ("v_q", ctypes.c_void_p), ("v_s", ctypes.c_void_p)]


class Seqs(ctypes.Structure):
    """tk_seqs: a batch of sequences with packed new tokens."""
    _device = None         # where make_seqs' tensors are
    _fields_ = [("n_seqs", ctypes.c_int), ("n_tokens", ctypes.c_int), ("max_new", ctypes.c_int),
                ("max_pages", ctypes.c_int), ("q_start", ctypes.c_void_p), ("kv_len", ctypes.c_void_p),
                ("pages", ctypes.c_void_p)]


# (name, rows, cols) of each table, in tk_iq_grids order
IQ_GRID_SHAPES = [("iq2xxs", 256, 8), ("iq2xs", 512, 8), ("iq2s", 1024, 8), ("iq3xxs", 256, 4), ("iq3s", 512, 4),
                  ("iq1s", 2048, 8)]


def iq_grids_from_gguf() -> dict:
    """The lattice tables as int8 arrays, taken from gguf-py's IQ*.grid (the
    numbers of tier/quant_tables.h).  Needs the gguf package."""
    import numpy as np
    from gguf import quants
    out = {}
    for (name, rows, cols), cls in zip(IQ_GRID_SHAPES, ("IQ2_XXS", "IQ2_XS", "IQ2_S", "IQ3_XXS", "IQ3_S", "IQ1_S")):
        q = getattr(quants, cls)
        q.init_grid()
        g = np.asarray(q.grid, dtype=np.float64).reshape(rows, cols)
        out[name] = np.ascontiguousarray(g.astype(np.int8))
    return out


_P = ctypes.c_void_p
_I = ctypes.c_int
_SZ = ctypes.c_size_t
_F = ctypes.c_float
_L = ctypes.c_long

# (name, restype, argtypes) -- mirrors include/tierk.h
SIGNATURES = [
    ("tk_init", _I, [_I, ctypes.POINTER(_P)]),
    ("tk_destroy", None, [_P]),
    ("tk_last_error_string", ctypes.c_char_p, []),
    ("tk_reserve", _I, [_P, _SZ]),
    ("tk_workspace_bytes", _SZ, [_P]),
    ("tk_sync_status", _I, [_P, _P]),
    ("tk_launch_count", ctypes.c_uint64, [_P]),
    ("tk_profile", _I, [_P, _I]),
    ("tk_profile_read", _I, [_P, _I, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_uint64)]),
    ("tk_row_bytes", _SZ, [_I, _I]),
    ("tk_set_iq_grids", _I, [_P, ctypes.POINTER(IqGrids)]),
    ("tk_lmhead_chunk", _I, [_SZ, _I, _I, _I]),
    ("tk_dequant", _I, [_P, _I, _P, _SZ, _I, _I, _I, _I, _P, _P]),
    ("tk_gemv", _I, [_P, _I, _P, _SZ, _I, _I, _P, _I, _I, _P, _I, _P]),
    ("tk_gemv_multi", _I, [_P, _I, _I, _P, _P, _P, _P, _SZ, _I, _P, _I, _I, _P]),
    ("tk_kv_append", _I, [_P, ctypes.POINTER(KvCache), ctypes.POINTER(Seqs), _P, _P, _I, _I, _I, _P]),
    ("tk_kv_read", _I, [_P, ctypes.POINTER(KvCache), ctypes.POINTER(Seqs), _P, _P, _I, _I, _I, _P]),
    ("tk_kv_attend", _I, [_P, ctypes.POINTER(KvCache), ctypes.POINTER(Seqs), _P, _I, _I, _I, _F, _I, _P, _I, _P]),
    ("tk_draft_verify", _I, [_P, _I, _P, _I, _I, _P, _L, _P, _L, _P, _P, _P, _F, _P, _P, _P, _P]),
    ("tk_logprobs", _I, [_P, _I, _I, _P, _I, _L, _P, _F, _P, _P, _P, _P, _I, _P, _P, _P]),
    ("tk_logprobs_grad", _I, [_P, _I, _I, _P, _I, _L, _P, _F, _P, _P, _P, _P, _P, _P, _I, _L, _P]),
    ("tk_distill", _I, [_P, _I, _I, _P, _I, _L, _I, _P, _P, _F, _P, _P, _P, _P, _P, _I, _L, _P]),
    ("tk_distill_grad", _I, [_P, _I, _I, _P, _I, _L, _I, _P, _P, _F, _P, _P, _P, _P, _I, _L, _P]),
    ("tk_linear_fwd", _I, [_P, ctypes.POINTER(Weight), _P, _I, _I, _I, _P, _I, _F, _I, _P]),
    ("tk_linear_dx", _I, [_P, ctypes.POINTER(Weight), _P, _I, _I, _I, _P, _I, _F, _I, _P]),
    ("tk_linear_fwd_noalloc", _I, [_P, ctypes.POINTER(Weight), _P, _I, _I, _I, _P, _I, _F, _I, _P]),
    ("tk_weight_split_f32", _I, [_P, _P, _I, _I, _P, ctypes.POINTER(_I), _P]),
    ("tk_split3", _I, [_P, _P, _SZ, _P, _P, _P, _P]),
    ("tk_quantize", _I, [_P, _I, _P, _I, _I, _I, _I, _P, _SZ, _P]),
    ("tk_tq_open", _I, [ctypes.c_char_p, ctypes.POINTER(_P)]),
    ("tk_tq_close", None, [_P]),
    ("tk_tq_count", _I, [_P]),
    ("tk_tq_find", _I, [_P, ctypes.c_char_p]),
    ("tk_tq_entry", _I, [_P, _I, ctypes.POINTER(ctypes.c_char_p), ctypes.POINTER(_I), ctypes.POINTER(_I),
                         ctypes.POINTER(_I), ctypes.POINTER(ctypes.c_uint64), ctypes.POINTER(ctypes.c_uint64),
                         ctypes.POINTER(ctypes.c_double)]),
    ("tk_tq_read", _I, [_P, _I, _P, _I, _P]),
    ("tk_tq_write", _I, [ctypes.c_char_p, _I, ctypes.POINTER(ctypes.c_char_p), ctypes.POINTER(_I),
                         ctypes.POINTER(_I), ctypes.POINTER(_I), ctypes.POINTER(_P), ctypes.POINTER(ctypes.c_double),
                         ctypes.c_char_p]),
    ("tk_qtype_from_name", _I, [ctypes.c_char_p]),
    ("tk_qtype_name", ctypes.c_char_p, [_I]),
    ("tk_comm_init", _I, [_P, _I, _I, _SZ, _P]),
    ("tk_comm_connect", _I, [_P, _P]),
    ("tk_linear_dx_rs", _I, [_P, ctypes.POINTER(Weight), _P, _I, _I, _I, _P, _I, _I, _P]),
    ("tk_linear_fwd_dx", _I, [_P, ctypes.POINTER(Weight), _P, _I, _I, _I, _P, _I, _P, _I, _I, _I, _P, _I, _I, _P]),
    ("tk_linear_fwd_dx_rs", _I, [_P, ctypes.POINTER(Weight), _P, _I, _I, _I, _P, _I, _P, _I, _I, _I, _P, _I, _I,
                                 _P]),
    ("tk_allgather", _I, [_P, _P, _SZ, _P, _P]),
    ("tk_allreduce_f32", _I, [_P, _P, _SZ, _P]),
    ("tk_reshard_cols", _I, [_P, _P, _I, _I, _SZ, _I, _P, _SZ, _P]),
    ("tk_reshard_cols_send", _I, [_P, _P, _I, _I, _SZ, _I, _P]),
    ("tk_reshard_cols_recv", _I, [_P, _P, _SZ, _I, _P]),
    ("tk_lmhead_merge", _I, [_P, _I, _P, _P, _P, _P, _P, _I, _P]),
    ("tk_lmhead_stats", _I, [_P, _P, _I, _I, _I, _P, _I, _P, _P, _F, _I, _I, _P, _P, _P, _P, _P]),
    ("tk_lmhead_grad", _I, [_P, _P, _I, _I, _I, _P, _I, _P, _P, _I, _F, _I, _I, _P, _P, _P, _P]),
    ("tk_lmhead_loss", _I, [_P, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P]),
    ("tk_lmhead_rescale", _I, [_P, _I, _P, _P, _P, _P, _I, _P]),
    ("tk_lmhead_fused", _I, [_P, _P, _I, _I, _I, _P, _I, _P, _P, _F, _I, _I, _P, _P, _P, _P, _P, _P]),
    ("tk_lmhead_finish", _I, [_P, _P, _I, _I, _I, _I, _P, _P, _I, _F, _P, _P, _P, _P]),
]

_lib = None


def load(path: str | os.PathLike | None = None) -> ctypes.CDLL:
    """Load libtierk.so (raises if absent -- there is no fallback)."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path else LIB_PATH
    if not p.exists():
        raise RuntimeError(f"libtierk.so not built ({p}); run `python -m tier_b200.build`")
    lib = ctypes.CDLL(str(p))
    for name, res, args in SIGNATURES:
        f = getattr(lib, name)
        f.restype = res
        f.argtypes = args
    if path is None:
        _lib = lib
    return lib


def row_bytes(qtype: int, cols: int) -> int:
    be, bb = BLOCK[qtype]
    return cols // be * bb


def lmhead_chunk(device_bytes: int, hidden: int, seq: int, vocab: int) -> int:
    """tk_lmhead_chunk: the reference's lm_chunk rule (tier/tier.cpp:2015-2017)
    with chunks in multiples of 256; device_bytes is the GPU's total memory."""
    return int(load().tk_lmhead_chunk(device_bytes, hidden, seq, vocab))


def _check(st: int):
    if st != TK_OK:
        raise TierkError(st, load().tk_last_error_string().decode())


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _current_stream() -> int:
    """The current stream's handle, without the Stream object (3 us a call) where torch offers that."""
    global _raw_stream
    if _raw_stream is None:
        import torch
        raw, device = (getattr(torch._C, n, None) for n in ("_cuda_getCurrentRawStream", "_cuda_getDevice"))
        torch.cuda.init()
        _raw_stream = (lambda: raw(device())) if raw and device else (lambda: torch.cuda.current_stream().cuda_stream)
    return _raw_stream()


_raw_stream = None


def _stream(stream) -> int | None:
    if stream is None:
        return _current_stream()
    return getattr(stream, "cuda_stream", stream)


def _reachable(t, device) -> bool:
    return t.get_device() == device or (t.get_device() < 0 and t.is_pinned())


def _row_stride(fn, name, t, code, n, width, ld, device):
    """The stride in elements of n rows of `width` elements of DT_* code `code` (ld, or None: the tensor's own), which must
    lie in t: the library sees an address and cannot tell where its memory ends.  What the library itself refuses (null
    pointers, unknown codes, strides below the width, alignment) is left to it."""
    if t is None:
        return ld or 0
    strides = t.stride()                                   # (each look at a tensor is 50 to 200 ns: as few as there may be)
    if len(strides) == 2 and strides[1] == 1 and (not ld or ld == strides[0]) and t.dtype is _DTYPES.get(code):
        rows, cols = t.shape
        if rows >= n and cols >= width and t.get_device() == device:
            return strides[0]
    return _other_row_stride(fn, name, t, code, n, width, ld, device)


def _other_row_stride(fn, name, t, code, n, width, ld, device):
    """_row_stride of what is not a plain matrix of those rows."""
    if not _DTYPES:
        import torch
        _DTYPES.update({DT_F32: torch.float32, DT_F16: torch.float16, DT_BF16: torch.bfloat16, _I32: torch.int32})
    shaped, ld, want, bad = not ld, ld or t.stride(0), _DTYPES.get(code), None
    if want is None:
        return ld
    if t.element_size() != want.itemsize or (t.dtype.is_floating_point and t.dtype is not want):   # (raw bits may pass)
        bad = f"holds {t.dtype}, given as {want}"
    elif not _reachable(t, device):
        bad = f"is not on device {device}"
    elif ld >= width > 0 and n > 0:
        if t.dim() > 1 and t.size(0) > 0 and not t[0].is_contiguous():
            bad = "has rows that are not contiguous"
        elif (shaped and (t.size(0) < n or t[0].numel() < width)
              or (n - 1) * ld + width > t.untyped_storage().nbytes() // want.itemsize - t.storage_offset()):
            bad = f"holds no {n} rows of {width}, {ld} apart"
    if bad:
        raise TierkError(TK_ERR_INVALID, f"{fn}: {name} {bad}")
    return ld


def _check_vector(fn, name, t, n, code, device):
    """n contiguous elements: fp32 (DT_F32) or 32-bit whole numbers (_I32)."""
    if t is None or (t.dtype is _DTYPES.get(code) and t.numel() >= n and t.is_contiguous() and t.get_device() == device):
        return
    if not (t.numel() >= n and t.element_size() == 4 and t.is_floating_point() == (code == DT_F32) and t.is_contiguous()):
        raise TierkError(TK_ERR_INVALID, f"{fn}: {name} must be {n} contiguous {'float32' if code == DT_F32 else 'int32'} elements")
    if not _reachable(t, device):
        raise TierkError(TK_ERR_INVALID, f"{fn}: {name} is not on device {device}")


def _vector(fn, name, t, n, code, device):
    """_check_vector, and the address."""
    if t is None:
        return None
    if not (t.dtype is _DTYPES.get(code) and t.get_device() == device and t.numel() >= n and t.is_contiguous()):
        _check_vector(fn, name, t, n, code, device)
    return t.data_ptr()


def _width(fn, name, t, n):
    """The columns of a contiguous matrix of n rows (None: 0)."""
    if t is None:
        return 0
    shape = t.shape
    if len(shape) != 2 or shape[0] != n:
        raise TierkError(TK_ERR_INVALID, f"{fn}: {name} must be a matrix of {n} rows")
    return shape[1]


def _beside(fn, name, t, ids, shape, code, device):
    """The address of what belongs to the places in ids, entry by entry: of their very shape (the library goes by the
    places' columns alone, and would take a wider or turned matrix's numbers for other rows')."""
    if t is None:
        return None
    if not (t.shape == shape and t.dtype is _DTYPES.get(code) and t.get_device() == device and t.is_contiguous()):
        if ids is not None and t.shape != shape:
            raise TierkError(TK_ERR_INVALID, f"{fn}: {name} must be a matrix of {shape[0]} rows of {shape[1]}, as the places")
        _check_vector(fn, name, t, shape[0] * shape[1], code, device)
    return t.data_ptr()


_I32 = -1
_DTYPES: dict = {}         # the torch type of each DT_* code, once a tensor has been looked at; _I32's


class Context:
    """A tk_ctx bound to one CUDA device."""

    def __init__(self, device: int = 0):
        self.lib = load()
        h = _P()
        _check(self.lib.tk_init(device, ctypes.byref(h)))
        self.h = h
        self.device = device
        self.peers = None        # (rank, world) once host.connect_peers has set up the peer buffers

    def close(self):
        if self.h:
            self.lib.tk_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- diagnostics ----
    def launches(self) -> int:
        return int(self.lib.tk_launch_count(self.h))

    def sync_status(self, stream=None):
        _check(self.lib.tk_sync_status(self.h, _stream(stream)))

    def profile(self, enable: bool, resume: bool = False):
        """Start a new per-launch timing record (enable), resume the current
        one (enable and resume), or pause it (not enable; the record is kept)."""
        _check(self.lib.tk_profile(self.h, (2 if resume else 1) if enable else 0))

    def profile_read(self, kind: int) -> tuple[float, int]:
        t = ctypes.c_double(0)
        n = ctypes.c_uint64(0)
        _check(self.lib.tk_profile_read(self.h, kind, ctypes.byref(t), ctypes.byref(n)))
        return t.value, int(n.value)

    def reserve(self, nbytes: int):
        _check(self.lib.tk_reserve(self.h, nbytes))

    # ---- operations (torch tensors in, device pointers to the C ABI) ----
    def set_iq_grids(self, grids: dict | None = None):
        """Register the IQ1/IQ2/IQ3 lattice tables (tk_set_iq_grids): a dict of
        int8 arrays keyed as IQ_GRID_SHAPES, or None for iq_grids_from_gguf()."""
        import numpy as np
        grids = iq_grids_from_gguf() if grids is None else grids
        keep = []
        s = IqGrids()
        for name, rows, cols in IQ_GRID_SHAPES:
            a = np.ascontiguousarray(grids[name], dtype=np.int8)
            if a.shape != (rows, cols):
                raise ValueError(f"{name}: expected shape {(rows, cols)}, got {a.shape}")
            keep.append(a)
            setattr(s, name, a.ctypes.data)
        _check(self.lib.tk_set_iq_grids(self.h, ctypes.byref(s)))

    def dequant(self, qtype, blocks, rows, cols, out, r0=0, out_dtype=DT_F32, row_bytes_=None, stream=None):
        rb = row_bytes_ if row_bytes_ is not None else row_bytes(qtype, cols)
        _check(self.lib.tk_dequant(self.h, qtype, _ptr(blocks), rb, r0, rows, cols, out_dtype, _ptr(out),
                                   _stream(stream)))
        return out

    def gemv(self, qtype, W, N, K, x, y, M=1, ldx=None, ldy=None, row_bytes_=None, stream=None):
        rb = row_bytes_ if row_bytes_ is not None else row_bytes(qtype & ~WFROZEN, K)
        _check(self.lib.tk_gemv(self.h, qtype, _ptr(W), rb, N, K, _ptr(x), ldx or K, M, _ptr(y), ldy or N,
                                _stream(stream)))
        return y

    def gemv_multi(self, qtype, Ws, rows, ys, K, x, M=1, ldx=None, row_bytes_=None, stream=None):
        """ys[i][:M, :rows[i]] = x . Ws[i]^T for weights that share x (tk_gemv_multi):
        one launch for a layer's q/k/v or gate/up."""
        n = len(Ws)
        rb = row_bytes_ if row_bytes_ is not None else row_bytes(qtype & ~WFROZEN, K)
        wp = (ctypes.c_void_p * n)(*[w.data_ptr() for w in Ws])
        rp = (ctypes.c_int * n)(*rows)
        yp = (ctypes.c_void_p * n)(*[y.data_ptr() for y in ys])
        lp = (ctypes.c_int * n)(*[y.stride(0) for y in ys])
        _check(self.lib.tk_gemv_multi(self.h, qtype, n, wp, rp, yp, lp, rb, K, _ptr(x), ldx or K, M,
                                      _stream(stream)))
        return ys

    def linear(self, W: Weight, X, M, Y, x_dtype=DT_F32, ldx=None, ldy=None, beta=0.0, products=X3_AUTO,
               stream=None):
        _check(self.lib.tk_linear_fwd(self.h, ctypes.byref(W), _ptr(X), x_dtype, M, ldx or W.cols, _ptr(Y),
                                      ldy or W.rows, beta, products, _stream(stream)))
        return Y

    def linear_dx(self, W: Weight, dY, M, dX, dy_dtype=DT_F32, lddy=None, lddx=None, beta=0.0, products=X3_AUTO,
                  stream=None):
        _check(self.lib.tk_linear_dx(self.h, ctypes.byref(W), _ptr(dY), dy_dtype, M, lddy or W.rows, _ptr(dX),
                                     lddx or W.cols, beta, products, _stream(stream)))
        return dX

    def linear_dx_acc(self, W: Weight, dY, M, dX, **kw):
        return self.linear_dx(W, dY, M, dX, beta=1.0, **kw)

    def linear_fwd_dx(self, W: Weight, X, Mx, Y, dY, Md, dX, x_dtype=DT_F32, dy_dtype=None, ldx=None, ldy=None,
                      lddy=None, lddx=None, products=X3_AUTO, stream=None):
        """Y = X . W^T and dX = dY . W in one launch (tk_linear_fwd_dx)."""
        dy_dtype = x_dtype if dy_dtype is None else dy_dtype
        _check(self.lib.tk_linear_fwd_dx(self.h, ctypes.byref(W), _ptr(X), x_dtype, Mx, ldx or W.cols, _ptr(Y),
                                         ldy or W.rows, _ptr(dY), dy_dtype, Md, lddy or W.rows, _ptr(dX),
                                         lddx or W.cols, products, _stream(stream)))
        return Y, dX

    def quantize(self, qtype, x, rows, cols, out, x_dtype=DT_F32, ldx=None, row_bytes_=None, stream=None):
        """out (uint8 [rows, row_bytes]) = x quantized to qtype, byte-exact with the reference's q_row."""
        rb = row_bytes_ if row_bytes_ is not None else row_bytes(qtype, cols)
        _check(self.lib.tk_quantize(self.h, qtype, _ptr(x), x_dtype, rows, cols, ldx or cols, _ptr(out), rb,
                                    _stream(stream)))
        return out

    # ---- 4-bit key/value cache, attention over it, drafted tokens ----
    def _kv_strides(self, fn, cache, seqs, heads, code, names, a, lda, b, ldb):
        """Row strides of a call's two packed arrays, which must lie in their tensors."""
        device, width = self.device, heads * cache.head_dim
        if cache._device not in (None, device) or seqs._device not in (None, device):
            raise TierkError(TK_ERR_INVALID, f"{fn}: cache and batch must be on device {device}")
        n = seqs.n_tokens if seqs.n_seqs > 0 and seqs.max_new > 0 else 0
        return (_row_stride(fn, names[0], a, code, n, width, lda, device),
                _row_stride(fn, names[1], b, code, n, width, ldb, device))

    def kv_append(self, cache: KvCache, seqs: Seqs, k, v, x_dtype=DT_F32, ldk=None, ldv=None, stream=None):
        """Round the batch's new keys and values to 4 bits into the cache (tk_kv_append)."""
        ldk, ldv = self._kv_strides("tk_kv_append", cache, seqs, cache.n_kv_heads, x_dtype, "kv", k, ldk, v, ldv)
        _check(self.lib.tk_kv_append(self.h, ctypes.byref(cache), ctypes.byref(seqs), _ptr(k), _ptr(v), x_dtype,
                                     ldk, ldv, _stream(stream)))

    def kv_read(self, cache: KvCache, seqs: Seqs, k, v, out_dtype=DT_F32, ldk=None, ldv=None, stream=None):
        """k, v = the values that the cache holds for the batch's new tokens (tk_kv_read)."""
        ldk, ldv = self._kv_strides("tk_kv_read", cache, seqs, cache.n_kv_heads, out_dtype, "kv", k, ldk, v, ldv)
        _check(self.lib.tk_kv_read(self.h, ctypes.byref(cache), ctypes.byref(seqs), _ptr(k), _ptr(v), out_dtype,
                                   ldk, ldv, _stream(stream)))
        return k, v

    def kv_attend(self, cache: KvCache, seqs: Seqs, q, n_heads, out, x_dtype=DT_F32, scale=None, window=0, ldq=None,
                  ldo=None, stream=None):
        """out = attention of the batch's new tokens over the cache (tk_kv_attend);
        scale defaults to 1 / sqrt(head_dim)."""
        scale = cache.head_dim ** -0.5 if scale is None else scale
        ldq, ldo = self._kv_strides("tk_kv_attend", cache, seqs, n_heads, x_dtype, ("q", "out"), q, ldq, out, ldo)
        _check(self.lib.tk_kv_attend(self.h, ctypes.byref(cache), ctypes.byref(seqs), _ptr(q), x_dtype,
                                     ldq, n_heads, scale, window, _ptr(out), ldo, _stream(stream)))
        return out

    def draft_verify(self, target, tokens, row_start, u_accept, u_sample, n_accept, next_token, logp=None, draft=None,
                     temperature=1.0, stream=None):
        """Accept drafted tokens against the target's logits and draw each
        sequence's next token (tk_draft_verify)."""
        fn, dev, B, (n, V) = "tk_draft_verify", self.device, n_accept.numel(), target.shape
        ldt = _row_stride(fn, "target", target, DT_F32, n, V, None, dev)
        ldd = _row_stride(fn, "draft", draft, DT_F32, n, V, None, dev)
        _check_vector(fn, "row_start", row_start, B + 1, _I32, dev)
        _check_vector(fn, "tokens", tokens, n, _I32, dev)
        if temperature:
            _check_vector(fn, "u_accept", u_accept, n - 1, DT_F32, dev)     # (the last row judges no draft)
            _check_vector(fn, "u_sample", u_sample, B, DT_F32, dev)
        _check_vector(fn, "n_accept", n_accept, B, _I32, dev)
        _check_vector(fn, "next_token", next_token, B, _I32, dev)
        _check_vector(fn, "logp", logp, n, DT_F32, dev)
        _check(self.lib.tk_draft_verify(self.h, B, _ptr(row_start), n, V, _ptr(target), ldt, _ptr(draft), ldd, _ptr(tokens),
                                        _ptr(u_accept), _ptr(u_sample), temperature, _ptr(n_accept), _ptr(next_token),
                                        _ptr(logp), _stream(stream)))
        return n_accept, next_token

    # ---- rows of logits ----
    def logprobs(self, logits, tokens=None, logp=None, entropy=None, rmax=None, rsum=None, top_ids=None, top_logp=None,
                 temperature=1.0, x_dtype=DT_F32, stream=None):
        """Log-probabilities of given tokens, entropy and the likeliest tokens of
        each row of logits [n, vocab] (tk_logprobs); top_ids, top_logp [n, k]."""
        fn, dev, (n, V) = "tk_logprobs", self.device, logits.shape
        k = _width(fn, "top_ids", top_ids, n)
        ldx = _row_stride(fn, "logits", logits, x_dtype, n, V, None, dev)
        _check(self.lib.tk_logprobs(self.h, n, V, _ptr(logits), x_dtype, ldx, _vector(fn, "tokens", tokens, n, _I32, dev),
                                    temperature, _vector(fn, "logp", logp, n, DT_F32, dev),
                                    _vector(fn, "entropy", entropy, n, DT_F32, dev), _vector(fn, "rmax", rmax, n, DT_F32, dev),
                                    _vector(fn, "rsum", rsum, n, DT_F32, dev), k,
                                    _vector(fn, "top_ids", top_ids, n * k, _I32, dev),
                                    _beside(fn, "top_logp", top_logp, top_ids, (n, k), DT_F32, dev), _stream(stream)))
        return logp

    def logprobs_grad(self, logits, tokens, rmax, rsum, dlogits, d_logp=None, entropy=None, d_entropy=None, temperature=1.0,
                      x_dtype=DT_F32, d_dtype=None, stream=None):
        """dlogits [n, vocab] of d_logp . logp + d_entropy . entropy
        (tk_logprobs_grad); dlogits may be logits."""
        fn, dev, (n, V) = "tk_logprobs_grad", self.device, logits.shape
        d_dtype = x_dtype if d_dtype is None else d_dtype
        ldx = _row_stride(fn, "logits", logits, x_dtype, n, V, None, dev)
        ldd = _row_stride(fn, "dlogits", dlogits, d_dtype, n, V, None, dev)
        _check(self.lib.tk_logprobs_grad(self.h, n, V, _ptr(logits), x_dtype, ldx, _vector(fn, "tokens", tokens, n, _I32, dev),
                                         temperature, _vector(fn, "rmax", rmax, n, DT_F32, dev),
                                         _vector(fn, "rsum", rsum, n, DT_F32, dev),
                                         _vector(fn, "d_logp", d_logp, n, DT_F32, dev),
                                         _vector(fn, "entropy", entropy, n, DT_F32, dev),
                                         _vector(fn, "d_entropy", d_entropy, n, DT_F32, dev), _ptr(dlogits), d_dtype, ldd,
                                         _stream(stream)))
        return dlogits

    def distill(self, logits, ids, teacher, loss=None, weight=None, dlogits=None, rmax=None, rsum=None, temperature=1.0,
                x_dtype=DT_F32, d_dtype=None, stream=None):
        """Loss of each row of logits [n, vocab] against a teacher's top logits
        ids, teacher [n, k], and its gradient (tk_distill); dlogits may be logits."""
        fn, dev, (n, V) = "tk_distill", self.device, logits.shape
        d_dtype, k = x_dtype if d_dtype is None else d_dtype, _width(fn, "ids", ids, n)
        ldx = _row_stride(fn, "logits", logits, x_dtype, n, V, None, dev)
        ldd = _row_stride(fn, "dlogits", dlogits, d_dtype, n, V, None, dev)
        _check(self.lib.tk_distill(self.h, n, V, _ptr(logits), x_dtype, ldx, k, _vector(fn, "ids", ids, n * k, _I32, dev),
                                   _beside(fn, "teacher", teacher, ids, (n, k), DT_F32, dev), temperature,
                                   _vector(fn, "weight", weight, n, DT_F32, dev), _vector(fn, "loss", loss, n, DT_F32, dev),
                                   _vector(fn, "rmax", rmax, n, DT_F32, dev), _vector(fn, "rsum", rsum, n, DT_F32, dev),
                                   _ptr(dlogits), d_dtype, ldd, _stream(stream)))
        return loss

    def distill_grad(self, logits, ids, teacher, rmax, rsum, dlogits, weight=None, temperature=1.0, x_dtype=DT_F32, d_dtype=None,
                     stream=None):
        """The gradient alone, from distill's rmax and rsum (tk_distill_grad)."""
        fn, dev, (n, V) = "tk_distill_grad", self.device, logits.shape
        d_dtype, k = x_dtype if d_dtype is None else d_dtype, _width(fn, "ids", ids, n)
        ldx = _row_stride(fn, "logits", logits, x_dtype, n, V, None, dev)
        ldd = _row_stride(fn, "dlogits", dlogits, d_dtype, n, V, None, dev)
        _check(self.lib.tk_distill_grad(self.h, n, V, _ptr(logits), x_dtype, ldx, k, _vector(fn, "ids", ids, n * k, _I32, dev),
                                        _beside(fn, "teacher", teacher, ids, (n, k), DT_F32, dev), temperature,
                                        _vector(fn, "rmax", rmax, n, DT_F32, dev), _vector(fn, "rsum", rsum, n, DT_F32, dev),
                                        _vector(fn, "weight", weight, n, DT_F32, dev), _ptr(dlogits), d_dtype, ldd,
                                        _stream(stream)))
        return dlogits

    # ---- reduce-scatter over peer memory (multi-GPU) ----
    def comm_init(self, rank: int, world: int, recv_bytes: int) -> bytes:
        """Allocate this rank's receive buffer; returns its IPC handle (64 bytes)."""
        buf = ctypes.create_string_buffer(IPC_HANDLE_BYTES)
        _check(self.lib.tk_comm_init(self.h, rank, world, recv_bytes, buf))
        return buf.raw

    def comm_connect(self, handles: bytes):
        """Open the peers' buffers: `handles` = every rank's handle, in rank order."""
        buf = ctypes.create_string_buffer(handles, len(handles))
        _check(self.lib.tk_comm_connect(self.h, buf))

    def linear_dx_rs(self, W: Weight, dY, M, dX_rows, dy_dtype=DT_F32, lddy=None, ldd=None, products=X3_AUTO,
                     stream=None):
        """This rank's token rows of sum over ranks of dY . W (tk_linear_dx_rs)."""
        _check(self.lib.tk_linear_dx_rs(self.h, ctypes.byref(W), _ptr(dY), dy_dtype, M, lddy or W.rows, _ptr(dX_rows),
                                        ldd or W.cols, products, _stream(stream)))
        return dX_rows

    def linear_fwd_dx_rs(self, W: Weight, X, Mx, Y, dY, Md, dX_rows, x_dtype=DT_F32, dy_dtype=None, ldx=None,
                         ldy=None, lddy=None, ldd=None, products=X3_AUTO, stream=None):
        """Y = X . W^T (this rank's columns) and this rank's token rows of the
        summed dY . W, in one launch (tk_linear_fwd_dx_rs)."""
        dy_dtype = x_dtype if dy_dtype is None else dy_dtype
        _check(self.lib.tk_linear_fwd_dx_rs(self.h, ctypes.byref(W), _ptr(X), x_dtype, Mx, ldx or W.cols, _ptr(Y),
                                            ldy or W.rows, _ptr(dY), dy_dtype, Md, lddy or W.rows, _ptr(dX_rows),
                                            ldd or W.cols, products, _stream(stream)))
        return Y, dX_rows

    def allgather(self, src, dst, nbytes=None, stream=None):
        """dst = every rank's src in rank order (tk_allgather)."""
        nb = nbytes if nbytes is not None else src.numel() * src.element_size()
        _check(self.lib.tk_allgather(self.h, _ptr(src), nb, _ptr(dst), _stream(stream)))
        return dst

    def reshard_cols(self, src, dst, stream=None):
        """Column shards src [M, n] -> row shard dst [M/world, world*n] (tk_reshard_cols)."""
        M, n = src.shape
        _check(self.lib.tk_reshard_cols(self.h, _ptr(src), M, n, src.stride(0), src.element_size(), _ptr(dst),
                                        dst.stride(0), _stream(stream)))
        return dst

    def reshard_cols_send(self, src, stream=None):
        M, n = src.shape
        _check(self.lib.tk_reshard_cols_send(self.h, _ptr(src), M, n, src.stride(0), src.element_size(),
                                             _stream(stream)))

    def reshard_cols_recv(self, dst, stream=None):
        _check(self.lib.tk_reshard_cols_recv(self.h, _ptr(dst), dst.stride(0), dst.element_size(), _stream(stream)))
        return dst

    def allreduce_f32(self, buf, stream=None):
        """buf = sum over ranks, in rank order (tk_allreduce_f32)."""
        _check(self.lib.tk_allreduce_f32(self.h, _ptr(buf), buf.numel(), _stream(stream)))
        return buf

    def lmhead_merge(self, n, rmax, rsum, amax, tgt, dX=None, H=0, stream=None):
        """Merge the vocabulary shards' running LM-head state (tk_lmhead_merge)."""
        _check(self.lib.tk_lmhead_merge(self.h, n, _ptr(rmax), _ptr(rsum), _ptr(amax), _ptr(tgt), _ptr(dX), H,
                                        _stream(stream)))

    def weight_split_f32(self, W32, rows, cols, planes, stream=None) -> int:
        sc = _I(0)
        _check(self.lib.tk_weight_split_f32(self.h, _ptr(W32), rows, cols, _ptr(planes), ctypes.byref(sc),
                                            _stream(stream)))
        return sc.value

    def split3(self, x, h, m, l, stream=None):
        _check(self.lib.tk_split3(self.h, _ptr(x), x.numel(), _ptr(h), _ptr(m), _ptr(l), _stream(stream)))

    def lmhead_stats(self, W, v0, V_shard, H, X, T, labels, mask, softcap, chunk, rmax, rsum, amax, tgt,
                     products=X3_REF, stream=None):
        _check(self.lib.tk_lmhead_stats(self.h, _ptr(W), v0, V_shard, H, _ptr(X), T, _ptr(labels), _ptr(mask),
                                        softcap, chunk, products, _ptr(rmax), _ptr(rsum), _ptr(amax), _ptr(tgt),
                                        _stream(stream)))

    def lmhead_grad(self, W, v0, V_shard, H, X, T, labels, mask, n_loss, softcap, chunk, rmax, rsum, dX,
                    products=X3_REF, stream=None):
        _check(self.lib.tk_lmhead_grad(self.h, _ptr(W), v0, V_shard, H, _ptr(X), T, _ptr(labels), _ptr(mask),
                                       n_loss, softcap, chunk, products, _ptr(rmax), _ptr(rsum), _ptr(dX),
                                       _stream(stream)))

    def lmhead_loss(self, T, labels, mask, rmax, rsum, amax, tgt, loss, hits, stream=None):
        _check(self.lib.tk_lmhead_loss(self.h, T, _ptr(labels), _ptr(mask), _ptr(rmax), _ptr(rsum), _ptr(amax),
                                       _ptr(tgt), _ptr(loss), _ptr(hits), _stream(stream)))

    def lmhead_rescale(self, n, rmax_local, rsum_local, rmax_global, dX=None, H=0, stream=None):
        _check(self.lib.tk_lmhead_rescale(self.h, n, _ptr(rmax_local), _ptr(rsum_local), _ptr(rmax_global),
                                          _ptr(dX) if dX is not None else None, H, _stream(stream)))

    def lmhead_fused(self, W, v0, V_shard, H, X, T, labels, mask, softcap, chunk, rmax, rsum, amax, tgt, dX,
                     products=X3_REF, stream=None):
        _check(self.lib.tk_lmhead_fused(self.h, _ptr(W), v0, V_shard, H, _ptr(X), T, _ptr(labels), _ptr(mask),
                                        softcap, chunk, products, _ptr(rmax), _ptr(rsum), _ptr(amax), _ptr(tgt),
                                        _ptr(dX), _stream(stream)))

    def lmhead_finish(self, W, v0, V_shard, H, T, labels, mask, n_loss, softcap, rsum, tgt, dX, stream=None):
        _check(self.lib.tk_lmhead_finish(self.h, _ptr(W), v0, V_shard, H, T, _ptr(labels), _ptr(mask), n_loss,
                                         softcap, _ptr(rsum), _ptr(tgt), _ptr(dX), _stream(stream)))


def make_weight(qtype: int, rows: int, cols: int, data, scale_log2: int = 0) -> Weight:
    """Describe a device weight tensor (uint8 blocks or fp16 planes) for the C ABI."""
    rb = cols * 2 if qtype in (F16, F16X2) else row_bytes(qtype, cols)
    w = Weight(qtype, rows, cols, scale_log2, rb, data.data_ptr())
    w._owner = data   # the descriptor keeps its device memory alive
    return w


def _one_device(what, tensors) -> int | None:
    """The CUDA device of all tensors (None: pinned host memory, which every device reaches)."""
    at = {None if t.get_device() < 0 and t.is_pinned() else t.get_device() for t in tensors}
    if -1 in at or len(at - {None}) > 1:
        raise ValueError(f"{what} must be on one CUDA device")
    return next(iter(at - {None}), None)


def make_kvcache(k_q, k_s, v_q, v_s) -> KvCache:
    """Describe a cache's four device tensors (layout: tk_kvcache in tierk.h):
    k_q, v_q uint8 [pages, kv_heads, page_tokens, head_dim / 2], k_s, v_s
    float16 [pages, kv_heads, page_tokens, head_dim / 32]."""
    n, h, p, half = k_q.shape
    for t, shape, size in ((k_q, (n, h, p, half), 1), (v_q, (n, h, p, half), 1), (k_s, (n, h, p, half // 16), 2),
                           (v_s, (n, h, p, half // 16), 2)):
        if tuple(t.shape) != shape or t.element_size() != size or not t.is_contiguous():
            raise ValueError(f"cache tensor {tuple(t.shape)}: expected contiguous {shape} of {size}-byte elements")
    c = KvCache(n, p, h, 2 * half, k_q.data_ptr(), k_s.data_ptr(), v_q.data_ptr(), v_s.data_ptr())
    c._owner = (k_q, k_s, v_q, v_s)   # the descriptor keeps its device memory alive
    c._device = _one_device("cache tensors", c._owner)
    return c


def alloc_kvcache(n_pages: int, page_tokens: int, n_kv_heads: int, head_dim: int, device="cuda") -> KvCache:
    """A zeroed cache of n_pages pages."""
    import torch
    shape = (n_pages, n_kv_heads, page_tokens)
    q = [torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device=device) for _ in "kv"]
    s = [torch.zeros(*shape, head_dim // 32, dtype=torch.float16, device=device) for _ in "kv"]
    return make_kvcache(q[0], s[0], q[1], s[1])


def make_seqs(q_start, kv_len, pages, n_tokens: int, max_new: int) -> Seqs:
    """Describe a batch (tk_seqs in tierk.h): int32 device tensors q_start
    [n_seqs + 1], kv_len [n_seqs], pages [n_seqs, max_pages]."""
    B = kv_len.numel()
    for t in (q_start, kv_len, pages):
        if t.element_size() != 4 or t.is_floating_point() or not t.is_contiguous():
            raise ValueError("q_start, kv_len and pages must be contiguous int32 tensors")
    if q_start.numel() != B + 1 or pages.dim() != 2 or pages.shape[0] != B:
        raise ValueError("q_start must have n_seqs + 1 entries and pages n_seqs rows")
    s = Seqs(B, n_tokens, max_new, pages.shape[1], q_start.data_ptr(), kv_len.data_ptr(), pages.data_ptr())
    s._owner = (q_start, kv_len, pages)
    s._device = _one_device("q_start, kv_len and pages", s._owner)
    return s


from .host import LinearPath, LMHead  # noqa: E402  (host-side mirror of the reference's operators)

__all__ = ["Context", "Weight", "make_weight", "KvCache", "Seqs", "make_kvcache", "alloc_kvcache", "make_seqs", "load", "row_bytes", "lmhead_chunk", "IqGrids", "IQ_GRID_SHAPES",
           "iq_grids_from_gguf", "LinearPath", "LMHead", "TierkError"]

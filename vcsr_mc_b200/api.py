"""Python mirror of the reference's host interface, over the C ABI (include/vcsrmc.h).

Names follow the reference (MuuSeoTia/VCSR_MC):
  read_matrix_market / coo_to_csr        include/mmio.hpp:19, include/csr.hpp:16
  rcm_column_order / apply_column_permutation   include/reorder.hpp:17, :82
  half_scale / csr_to_vcsr_mc            src/vcsr_mc.cu:14, :25
  upload_vcsr_mc_device                  src/vcsr_mc.cu:332
  run_vcsr_mc_spmm_gpu                   src/vcsr_mc.cu:352 (blocking, returns ms)
  destroy_vcsr_mc_device                 src/vcsr_mc.cu:397
Errors raise VcsrmcError (the reference throws std::runtime_error or exits).

Device buffers are torch CUDA tensors (torch is used for device memory and streams only);
every computation runs in libvcsrmc.so.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import numpy as np

from . import _lib
from ._lib import (BF16, F16, F32, MXF4, MXF8, PLAN_AUTO, PLAN_BAND, PLAN_HYBRID, PLAN_ROWS, PLAN_SEGMENT, VcsrmcError,
                   call)


def _ptr(a: np.ndarray) -> ctypes.c_void_p:
    return ctypes.c_void_p(a.ctypes.data) if a.size else ctypes.c_void_p(0)


def _as_np(ptr, n: int, dtype) -> np.ndarray:
    if n == 0:
        return np.zeros(0, dtype=dtype)
    return np.ctypeslib.as_array(ptr, shape=(n,))


class CSR:
    """Host CSR owned by the library (fields of include/csr.hpp:8-13)."""

    def __init__(self, handle: ctypes.c_void_p):
        self._h = handle

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h and _lib._lib is not None:
            _lib.lib().vcsrmc_csr_free(h)

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._h

    def _view(self) -> _lib.CsrView:
        v = _lib.CsrView()
        call("vcsrmc_csr_view_get", self._h, ctypes.byref(v))
        return v

    @property
    def M(self) -> int:
        return self._view().M

    @property
    def N(self) -> int:
        return self._view().N

    @property
    def nnz(self) -> int:
        return self._view().nnz

    def arrays(self, copy: bool = True):
        """(row_ptr, col, val) as numpy arrays (views valid while this object lives if copy=False)."""
        v = self._view()
        rp = _as_np(v.row_ptr, v.M + 1, np.int32)
        col = _as_np(v.col, v.nnz, np.int32)
        val = _as_np(v.val, v.nnz, np.float32)
        if copy:
            return rp.copy(), col.copy(), val.copy()
        return rp, col, val

    def row_slice(self, r0: int, r1: int) -> "CSR":
        h = ctypes.c_void_p()
        call("vcsrmc_csr_row_slice", self._h, r0, r1, ctypes.byref(h))
        return CSR(h)

    def save(self, path: str) -> None:
        """Binary cache of this CSR (vcsrmc_csr_save); load it with load_csr."""
        call("vcsrmc_csr_save", self.handle, path.encode())

    @staticmethod
    def from_arrays(M: int, N: int, row_ptr, col, val) -> "CSR":
        rp = np.ascontiguousarray(row_ptr, dtype=np.int32)
        c = np.ascontiguousarray(col, dtype=np.int32)
        v = np.ascontiguousarray(val, dtype=np.float32)
        h = ctypes.c_void_p()
        call("vcsrmc_csr_from_arrays", M, N, int(c.size), _ptr(rp), _ptr(c), _ptr(v), ctypes.byref(h))
        return CSR(h)

    @staticmethod
    def generate(kind: int, param: int, seed: int = 0, nthreads: int = 0) -> "CSR":
        h = ctypes.c_void_p()
        call("vcsrmc_gen_csr", kind, param, seed, nthreads, ctypes.byref(h))
        return CSR(h)


def load_csr(path: str) -> CSR:
    """A CSR saved by CSR.save (binary cache; vcsrmc_csr_load)."""
    h = ctypes.c_void_p()
    call("vcsrmc_csr_load", path.encode(), ctypes.byref(h))
    return CSR(h)


def read_matrix_market(path: str) -> CSR:
    """read_matrix_market_coo + coo_to_csr (include/mmio.hpp:19-75, include/csr.hpp:16-41)."""
    h = ctypes.c_void_p()
    call("vcsrmc_csr_read_mtx", path.encode(), ctypes.byref(h))
    return CSR(h)


def coo_to_csr(M: int, N: int, rows, cols, vals) -> CSR:
    r = np.ascontiguousarray(rows, dtype=np.int32)
    c = np.ascontiguousarray(cols, dtype=np.int32)
    v = np.ascontiguousarray(vals, dtype=np.float32)
    h = ctypes.c_void_p()
    call("vcsrmc_csr_from_coo", M, N, int(v.size), _ptr(r), _ptr(c), _ptr(v), ctypes.byref(h))
    return CSR(h)


def rcm_column_order(csr: CSR) -> np.ndarray:
    pos = np.empty(csr.N, dtype=np.int32)
    call("vcsrmc_rcm_column_order", csr.handle, _ptr(pos))
    return pos


def apply_column_permutation(csr: CSR, B: Optional[np.ndarray], position: np.ndarray) -> Optional[np.ndarray]:
    """Relabels csr's columns in place; returns B (N x O fp32) with its rows permuted."""
    pos = np.ascontiguousarray(position, dtype=np.int32)
    if B is None:
        call("vcsrmc_apply_column_permutation", csr.handle, ctypes.c_void_p(0), 0, _ptr(pos))
        return None
    Bc = np.array(B, dtype=np.float32, order="C", copy=True)
    call("vcsrmc_apply_column_permutation", csr.handle, _ptr(Bc), int(Bc.shape[1]), _ptr(pos))
    return Bc


def half_scale(csr: CSR) -> float:
    s = ctypes.c_float()
    call("vcsrmc_half_scale", csr.handle, ctypes.byref(s))
    return s.value


class VCSRMC:
    """Host VCSR-MC format (struct VCSRMC, include/vcsr_formats.hpp:14-21)."""

    ARRAYS = ("group_ptr", "group_depth", "group_seg_base", "group_rows", "lcol", "val", "item_gbeg", "item_gend")

    def __init__(self, handle: ctypes.c_void_p):
        self._h = handle
        v = _lib.FormatView()
        call("vcsrmc_format_view_get", handle, ctypes.byref(v))
        self._v = v
        self.M, self.N, self.segw, self.bundle = v.M, v.N, v.segw, v.bundle
        self.num_segments, self.fp32, self.scale = v.num_segments, bool(v.fp32), v.scale
        self.n_groups, self.n_slots, self.n_items = v.n_groups, v.n_slots, v.n_items

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h and _lib._lib is not None:
            _lib.lib().vcsrmc_format_free(h)

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._h

    def array(self, name: str, copy: bool = True) -> np.ndarray:
        v = self._v
        n = {"group_ptr": v.n_groups + 1, "group_depth": v.n_groups, "group_seg_base": v.n_groups,
             "group_rows": 16 * v.n_groups, "lcol": v.n_slots, "val": v.n_slots,
             "item_gbeg": v.n_items, "item_gend": v.n_items}[name]
        a = _as_np(getattr(v, name), n, np.float32 if name == "val" else np.int32)
        return a.copy() if copy else a

    def arrays(self, copy: bool = True) -> dict:
        return {k: self.array(k, copy) for k in self.ARRAYS}


def csr_to_vcsr_mc(csr: CSR, fp32: bool = False, segw: int = 16, nthreads: int = 0) -> VCSRMC:
    h = ctypes.c_void_p()
    call("vcsrmc_build_host", csr.handle, 1 if fp32 else 0, segw, nthreads, ctypes.byref(h))
    return VCSRMC(h)


def _stream_handle(stream) -> ctypes.c_void_p:
    if stream is None:
        import torch
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(int(stream.cuda_stream) if hasattr(stream, "cuda_stream") else int(stream))


class DeviceVCSRMC:
    """A VCSR-MC format resident on one GPU (replaces src/vcsr_mc.cu:126-131's statics)."""

    def __init__(self, handle: ctypes.c_void_p, host: Optional[VCSRMC], device: int, **shape):
        self._h = handle
        self.device = device
        if host is not None:
            shape = dict(M=host.M, N=host.N, fp32=host.fp32, scale=host.scale, segw=host.segw)
        self.M, self.N, self.fp32, self.scale, self.segw = (shape[k] for k in ("M", "N", "fp32", "scale", "segw"))

    def info(self) -> dict:
        """Shape and resident layouts (vcsrmc_device_info_get); plans is a list of PLAN_* values."""
        i = _lib.DeviceInfo()
        call("vcsrmc_device_info_get", self._h, ctypes.byref(i))
        out = {k: getattr(i, k) for k, _ in _lib.DeviceInfo._fields_}
        out["plans"] = [p for p in (PLAN_SEGMENT, PLAN_ROWS, PLAN_BAND, PLAN_HYBRID) if i.plans & (1 << p)]
        return out

    def download(self) -> VCSRMC:
        """The SEGMENT arrays back on the host (FP16 formats: values as stored, rounded to fp16)."""
        h = ctypes.c_void_p()
        call("vcsrmc_device_download", self._h, ctypes.byref(h))
        return VCSRMC(h)

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._h

    def free(self) -> None:
        h, self._h = self._h, None
        if h:
            call("vcsrmc_device_free", h)

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def status(self, clear: bool = False) -> int:
        f = ctypes.c_uint32()
        call("vcsrmc_device_status", self._h, ctypes.byref(f), 1 if clear else 0)
        return f.value


def _upload_options(plans, rows_unit_nnz: int, band_rows: int, hot_rows: int, hot_budget_mib: int,
                    hot_persist: int, hot_evict_first: int) -> "_lib.UploadOptions":
    opts = _lib.UploadOptions()
    opts.plans = 0 if plans is None else sum(1 << p for p in set(plans))
    opts.rows_unit_nnz = rows_unit_nnz
    opts.band_rows = band_rows
    opts.hot_rows = hot_rows
    opts.hot_budget_mib = hot_budget_mib
    opts.hot_persist = hot_persist
    opts.hot_evict_first = hot_evict_first
    return opts


def upload_vcsr_mc_device(V: VCSRMC, device: int = 0, stream=None, plans=None,
                          rows_unit_nnz: int = 0, band_rows: int = 0, hot_rows: int = 0, hot_budget_mib: int = 0,
                          hot_persist: int = 0, hot_evict_first: int = 0) -> DeviceVCSRMC:
    """Copies the format to `device`. plans: iterable of PLAN_SEGMENT / PLAN_ROWS / PLAN_BAND /
    PLAN_HYBRID layouts to make resident (default: SEGMENT and ROWS, plus BAND for FP16 formats whose
    column tiles are dense enough; BAND and HYBRID need the FP16 format). rows_unit_nnz: entries per ROWS-plan work unit (0 = the library's
    choice for this matrix). band_rows: rows per BAND-plan band, 1 .. 128 (0 = chosen).
    hot_rows / hot_budget_mib / hot_persist / hot_evict_first: the ROWS plan's hot columns, off by
    default (vcsrmc_upload_options)."""
    opts = _upload_options(plans, rows_unit_nnz, band_rows, hot_rows, hot_budget_mib, hot_persist, hot_evict_first)
    h = ctypes.c_void_p()
    call("vcsrmc_upload_opts", V.handle, device, ctypes.byref(opts), _stream_handle(stream), ctypes.byref(h))
    return DeviceVCSRMC(h, V, device)


def build_vcsr_mc_device(row_ptr, col, val, M: int, N: int, fp32: bool = False, segw: int = 16, device: int = 0,
                         stream=None, plans=None, rows_unit_nnz: int = 0, band_rows: int = 0, hot_rows: int = 0,
                         hot_budget_mib: int = 0, hot_persist: int = 0, hot_evict_first: int = 0) -> DeviceVCSRMC:
    """Builds the format on the GPU from a CSR already in device memory (torch tensors: int32
    row_ptr[M+1], int32 col[nnz], float32 val[nnz], rows with strictly ascending columns) and
    keeps its plan layouts resident there. Equal-count rows of a segment come in ascending row
    order (see vcsrmc_build_device)."""
    import torch
    for t, dt in ((row_ptr, torch.int32), (col, torch.int32), (val, torch.float32)):
        if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dt and t.is_contiguous()):
            raise VcsrmcError(_lib.INVALID_ARG, "row_ptr/col/val must be contiguous CUDA tensors (int32, int32, float32)")
    opts = _upload_options(plans, rows_unit_nnz, band_rows, hot_rows, hot_budget_mib, hot_persist, hot_evict_first)
    h = ctypes.c_void_p()
    call("vcsrmc_build_device", M, N, int(col.numel()), ctypes.c_void_p(row_ptr.data_ptr()),
         ctypes.c_void_p(col.data_ptr()), ctypes.c_void_p(val.data_ptr()), 1 if fp32 else 0, segw, device,
         ctypes.byref(opts), _stream_handle(stream), ctypes.byref(h))
    info = _lib.DeviceInfo()
    call("vcsrmc_device_info_get", h, ctypes.byref(info))
    return DeviceVCSRMC(h, None, device, M=M, N=N, fp32=fp32, scale=float(info.scale), segw=segw)


def destroy_vcsr_mc_device(dV: DeviceVCSRMC) -> None:
    dV.free()


def _b_args(B):
    import torch
    if B.dtype == torch.float16:
        return F16
    if B.dtype == torch.float32:
        return F32
    raise VcsrmcError(_lib.INVALID_ARG, f"B must be float16 or float32, got {B.dtype}")


def _check_dense(B, C, O):
    import torch
    if not (B.is_cuda and C.is_cuda) or C.dtype != torch.float32:
        raise VcsrmcError(_lib.INVALID_ARG, "B and C must be CUDA tensors, C float32")
    if B.dim() != 2 or C.dim() != 2 or B.stride(1) != 1 or C.stride(1) != 1 or B.shape[1] < O or C.shape[1] < O:
        raise VcsrmcError(_lib.INVALID_ARG, "B and C must be 2-D row-major with >= O columns")


def spmm(dV: DeviceVCSRMC, B, C, tileK: int = 128, accumulate: bool = False, stream=None, O: Optional[int] = None,
         plan: int = PLAN_AUTO):
    """C[:, :O] (+)= A * B[:, :O] on the GPU, asynchronous on `stream` (default: torch's current).
    B: a float16 or float32 tensor, or an MXDense (ROWS plan; the same call gives the same bits; blocks of scale code 0 count as zero).
    stream: a torch stream or a raw handle (0: the default stream). Nothing is recorded for autograd."""
    if isinstance(B, MXDense):
        return _spmm_mx(dV, B, C, tileK, accumulate, stream, O, plan)
    O = int(B.shape[1]) if O is None else O
    _check_dense(B, C, O)
    call("vcsrmc_spmm_ex", dV.handle, ctypes.c_void_p(B.data_ptr()), _b_args(B), B.stride(0), O, tileK,
         ctypes.c_void_p(C.data_ptr()), C.stride(0), 1 if accumulate else 0, plan, _stream_handle(stream))
    return C


MX_BLOCK = 32  # columns of an MX matrix that share a scale


def _invalid(message: str) -> VcsrmcError:
    return VcsrmcError(_lib.INVALID_ARG, message)


class MXDense:
    """A microscaled (MX) matrix on one GPU: elements and one power-of-two scale per 32 columns of a row.

    data:  float8_e4m3fn [rows, cols] (MXF8), or uint8 [rows, ceil(cols / 2)] with two E2M1 elements per
           byte, the even column in the low half (MXF4)
    scale: float8_e8m0fnu (or uint8) [rows, ceil(cols / 32)]
    Rows may be strided; columns may not. `cols` is needed for an odd number of MXF4 columns. The tensors and the shape are set
    once, so that what was checked here is what the kernels get; the tensors' values may change."""

    __slots__ = ("_data", "_scale", "_kind", "_rows", "_cols", "_ldq", "_lds")

    def __init__(self, data, scale, cols: Optional[int] = None):
        import torch
        if not (isinstance(data, torch.Tensor) and isinstance(scale, torch.Tensor)) or data.dim() != 2 or scale.dim() != 2:
            raise _invalid("MX elements and scales must be 2-D tensors")
        if data.dtype == torch.float8_e4m3fn:
            kind, per_byte = MXF8, 1
        elif data.dtype == torch.uint8:
            kind, per_byte = MXF4, 2
        else:
            raise _invalid(f"MX elements must be float8_e4m3fn (MXF8) or uint8 (MXF4), got {data.dtype}")
        if scale.dtype not in (torch.float8_e8m0fnu, torch.uint8):
            raise _invalid(f"MX scales must be float8_e8m0fnu or uint8, got {scale.dtype}")
        rows, cols = int(data.shape[0]), int(data.shape[1]) * per_byte if cols is None else int(cols)
        if cols < 0 or data.shape[1] < -(-cols // per_byte) or scale.shape[1] < -(-cols // MX_BLOCK) or scale.shape[0] != rows:
            raise _invalid("MX elements and scales must hold every row and column")
        if (data.stride(1) != 1 and data.shape[1] > 1) or (scale.stride(1) != 1 and scale.shape[1] > 1):
            raise _invalid("the columns of MX elements and scales must be contiguous")
        if data.device != scale.device:
            raise _invalid("MX elements and scales must be on the same device")
        self._data, self._scale, self._kind, self._rows, self._cols = data, scale, kind, rows, cols
        self._ldq, self._lds = _row_stride(data), _row_stride(scale)

    data = property(lambda self: self._data)
    scale = property(lambda self: self._scale)
    kind = property(lambda self: self._kind)
    rows = property(lambda self: self._rows)
    cols = property(lambda self: self._cols)
    shape = property(lambda self: (self._rows, self._cols))
    device = property(lambda self: self._data.device)

    @staticmethod
    def empty(rows: int, cols: int, kind: int = MXF8, device=None) -> "MXDense":
        """An MXDense to write to. Its rows start at multiples of 16 bytes (those of its scales: 4), whatever `cols` is, so that
        every operator can use its widest loads and stores."""
        import torch
        if kind not in (MXF8, MXF4):
            raise _invalid("the microscaled kind must be MXF8 or MXF4")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise _invalid("microscaled operators run on CUDA tensors")
        index = torch.cuda.current_device() if device.index is None else device.index
        data, scale, ldq, lds = (_ops or _load_ops()).mx_empty(rows, cols, kind, index)
        return MXDense._of(data, scale, kind, rows, cols, ldq, lds)

    @staticmethod
    def _of(data, scale, kind: int, rows: int, cols: int, ldq: int, lds: int) -> "MXDense":
        out = MXDense.__new__(MXDense)
        out._data, out._scale, out._kind, out._rows, out._cols, out._ldq, out._lds = data, scale, kind, rows, cols, ldq, lds
        return out

    def _args(self):
        """Elements, scales, kind and the row strides of both, as _torch_ops takes them."""
        return self._data, self._scale, self._kind, self._ldq, self._lds


_NO_MX = (None,) * 5


def _row_stride(t) -> int:
    """Row stride of a 2-D tensor in elements; torch leaves the stride of a single row open."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


_ops = None


def _load_ops():
    """vcsr_mc_b200._torch_ops (csrc/torch_ops.cpp): checks, allocation and the C ABI call of the microscaled operators. Built in-tree
    with the library; there is no other path."""
    global _ops
    import torch  # noqa: F401  (the module links against it)
    _lib.lib()
    try:
        from . import _torch_ops
    except ImportError as e:
        raise ImportError(f"vcsr_mc_b200/_torch_ops.so is not built or does not load ({e}); run `make -C vcsr_mc_b200/csrc`") from e
    _torch_ops.set_error(VcsrmcError)
    _ops = _torch_ops
    return _ops


def _stream_guard(stream, device):
    """torch's guard that makes `stream` (a torch stream, or a raw handle; 0: the default stream) current on `device`, so that a call's launches and what it
    allocates belong to it."""
    import torch
    if device.type != "cuda":
        raise _invalid("microscaled operators run on CUDA tensors")
    if not isinstance(stream, torch.cuda.Stream):
        raw = int(stream.cuda_stream) if hasattr(stream, "cuda_stream") else int(stream)
        # 0 and 1 are the default stream, as torch and CUDA give it; torch makes another stream of an external 0
        stream = torch.cuda.default_stream(device) if raw in (0, 1) else torch.cuda.ExternalStream(raw, device=device)
    if stream.device != device:
        raise _invalid(f"the stream must be on {device}, with the tensors")
    return torch.cuda.stream(stream)


def _mx_out(out: Optional[MXDense], X, kind: int):
    if out is None:
        return _NO_MX
    if out.kind != kind or out.shape != tuple(X.shape) or out.device != X.device:
        raise _invalid("out must have X's shape and device, and the kind that is asked for")
    return out._args()


def _spmm_mx(dV: DeviceVCSRMC, B: MXDense, C, tileK: int, accumulate: bool, stream, O: Optional[int], plan: int):
    if stream is not None:
        with _stream_guard(stream, C.device):
            return _spmm_mx(dV, B, C, tileK, accumulate, None, O, plan)
    if plan != PLAN_AUTO and plan != PLAN_ROWS:
        raise _invalid("a microscaled B runs on the ROWS plan")
    if tileK not in (16, 32, 64, 128, 256):
        raise _invalid("tileK must be one of 16, 32, 64, 128, 256")
    h = dV._h
    (_ops or _load_ops()).spmm_mx(h.value if h else 0, dV.device, dV.M, dV.N, *B._args(), B._rows, B._cols, B._cols if O is None else O, C,
                                  1 if accumulate else 0)
    return C


def mx_quantize(X, kind: int = MXF8, out: Optional[MXDense] = None, stream=None) -> MXDense:
    """X (float32, float16 or bfloat16) in 8 (MXF8) or 4 bits (MXF4): the scale of 32 columns is the smallest power of two
    under which their largest magnitude fits the element type; elements are rounded to nearest, ties to even."""
    if stream is not None:
        with _stream_guard(stream, X.device):
            return mx_quantize(X, kind, out)
    data, scale, ldq, lds = (_ops or _load_ops()).mx_quantize(X, kind, *_mx_out(out, X, kind))
    return MXDense._of(data, scale, kind, *X.shape, ldq, lds) if out is None else out


def mx_dequantize(Q: MXDense, dtype=None, out=None, stream=None):
    """The values an MXDense stands for, rounded to `dtype` (default float32)."""
    if stream is not None:
        with _stream_guard(stream, Q.device):
            return mx_dequantize(Q, dtype, out)
    import torch
    if out is None:
        out = torch.empty(Q.rows, Q.cols, dtype=dtype or torch.float32, device=Q.data.device)
    elif dtype is not None and out.dtype != dtype:
        raise _invalid(f"out must be {dtype}, got {out.dtype}")
    (_ops or _load_ops()).mx_dequantize(*Q._args(), Q.rows, Q.cols, out)
    return out


def add_rms_norm(X, weight, residual=None, eps: float = 1e-6, kind: int = MXF8, out: Optional[MXDense] = None, residual_out=None,
                 stream=None):
    """(Q, residual_out, inv_rms): s = X + residual, rounded to the residual's type (residual_out); inv_rms = 1 / sqrt(mean(s^2) +
    eps) of every row (float32); Q = MX(s * inv_rms * weight). The residual has X's type, or X is float32 (a product's C). Without a
    residual s is X, which is then returned in residual_out's place. residual_out may be the residual, or X of the same type (in place).
    Nothing is recorded for autograd: new tensors do not require a gradient, whatever X does; add_rms_norm_backward is called by hand or from
    a torch.autograd.Function of the caller's."""
    if stream is not None:
        with _stream_guard(stream, X.device):
            return add_rms_norm(X, weight, residual, eps, kind, out, residual_out)
    data, scale, ldq, lds, hidden, inv_rms = (_ops or _load_ops()).add_rms_norm(X, weight, residual, eps, kind, *_mx_out(out, X, kind), residual_out)
    return MXDense._of(data, scale, kind, *X.shape, ldq, lds) if out is None else out, hidden if residual_out is None else residual_out, inv_rms


def add_rms_norm_backward(dY, weight, hidden, inv_rms, d_residual=None, out=None, stream=None):
    """(dX, dweight) of add_rms_norm: dY is the gradient of the values Q stands for (float32 or hidden's type; the elements' rounding
    counts as the identity), hidden and inv_rms are what the forward call returned, d_residual the gradient of its residual_out. dX, in
    hidden's type, is the gradient of X and of the residual; dweight is float32. out (dX) may be d_residual, or dY of the same type."""
    if stream is not None:
        with _stream_guard(stream, dY.device):
            return add_rms_norm_backward(dY, weight, hidden, inv_rms, d_residual, out)
    return (_ops or _load_ops()).add_rms_norm_backward(dY, weight, hidden, inv_rms, d_residual, out)


def run_vcsr_mc_spmm_gpu(dV: DeviceVCSRMC, B, O: int, tileK: int, C, stream=None, accumulate: bool = True) -> float:
    """Blocking, event-timed launch with the reference's C += A*B contract; returns ms."""
    _check_dense(B, C, O)
    ms = ctypes.c_float()
    call("vcsrmc_spmm_timed", dV.handle, ctypes.c_void_p(B.data_ptr()), _b_args(B), B.stride(0), O, tileK,
         ctypes.c_void_p(C.data_ptr()), C.stride(0), 1 if accumulate else 0, _stream_handle(stream),
         ctypes.byref(ms))
    return ms.value


def gen_dense_host(rows: int, cols: int, seed: int, nthreads: int = 0) -> np.ndarray:
    out = np.empty((rows, cols), dtype=np.float32)
    call("vcsrmc_gen_dense_host", rows, cols, seed, _ptr(out), nthreads)
    return out


def gen_dense_device(out, seed: int, stream=None):
    """Fills a 2-D CUDA tensor (float32 or float16) with the dense U(-1,1) stream."""
    dt = _b_args(out)
    call("vcsrmc_gen_dense_device", int(out.shape[0]), int(out.shape[1]), seed, dt,
         ctypes.c_void_p(out.data_ptr()), out.stride(0), _stream_handle(stream))
    return out


# Row weight of the multi-GPU partition that the benchmark and the sharded path use: a block's
# cost is nnz + SHARD_ROW_WEIGHT * rows. It is the ratio of the per-row to the per-entry cost of the
# ROWS plan fitted (least squares) to 56 measured shard times of the 2^24-row R-MAT: 0.118 ns per row
# (the C row store and the row bookkeeping) against 0.0312 ns per entry.
SHARD_ROW_WEIGHT = 3.8


def partition_rows(row_ptr: np.ndarray, parts: int, row_weight: float = 0.0) -> np.ndarray:
    """parts+1 row cuts balancing nnz + row_weight * rows per block (0: pure nnz balance)."""
    rp = np.ascontiguousarray(row_ptr, dtype=np.int32)
    cuts = np.empty(parts + 1, dtype=np.int32)
    if row_weight == 0.0:
        call("vcsrmc_partition_rows", _ptr(rp), int(rp.size - 1), parts, _ptr(cuts))
    else:
        call("vcsrmc_partition_rows_weighted", _ptr(rp), int(rp.size - 1), parts, float(row_weight), _ptr(cuts))
    return cuts

"""Host-side mirror of the reference's kernel strategy API.

Reference: src/main/java/com/arturskowronski/llama3babylon/hat/kernels/
  IKernelFactory.java:9-40, IGEMV.java:11-69, IRMSNorm.java:8-18, IRoPE.java:8-20,
  ISiLU.java:8-17, ISoftmax.java:8-27, IAttention.java:8-31.

`CudaKernelFactory` sits where `PlainJavaKernelFactory` / `HybridKernelFactory`
sit: same method names, same argument meaning, same in-place behaviour.  Each
kernel object forwards to the C ABI of libllamacuda.so; buffers may be numpy
arrays (host memory, staged by the library) or torch tensors (host or CUDA).
`Accelerator` stands in for hat.Accelerator: it owns the CUDA context of one
device.
"""
from __future__ import annotations

import ctypes
import weakref
from abc import ABC, abstractmethod

import numpy as np

from . import _lib
from .config import RopeConfig


def _addr(buf, kind: str, min_len: int, writable: bool = False) -> int:
    """Address of a contiguous buffer of the expected element type.

    kind: "f32", "f16" (IEEE half bits; numpy float16 or uint16), "i32".
    """
    want = {"f32": (np.float32,), "f16": (np.float16, np.uint16), "i32": (np.int32,)}[kind]
    if isinstance(buf, np.ndarray):
        if buf.dtype.type not in want:
            raise TypeError(f"expected {kind} buffer, got numpy {buf.dtype}")
        if not buf.flags.c_contiguous:
            raise ValueError("buffer must be C-contiguous")
        if writable and not buf.flags.writeable:
            raise ValueError("buffer is read-only")
        if buf.size < min_len:
            raise ValueError(f"buffer holds {buf.size} elements, need {min_len}")
        return buf.ctypes.data
    try:
        import torch
    except ImportError:  # pragma: no cover
        torch = None
    if torch is not None and isinstance(buf, torch.Tensor):
        tw = {"f32": (torch.float32,), "f16": (torch.float16, torch.int16), "i32": (torch.int32,)}[kind]
        if buf.dtype not in tw:
            raise TypeError(f"expected {kind} tensor, got {buf.dtype}")
        if not buf.is_contiguous():
            raise ValueError("tensor must be contiguous")
        if buf.numel() < min_len:
            raise ValueError(f"tensor holds {buf.numel()} elements, need {min_len}")
        return buf.data_ptr()
    raise TypeError(f"unsupported buffer type {type(buf)!r}")


_NP_ROWS = {np.dtype(np.float32): 0, np.dtype(np.float16): 1}
_TORCH_ROWS: dict = {}  # torch dtypes of rows, and of int32 arrays, filled at the first tensor
_TORCH_I32 = None


def _torch_types() -> None:
    global _TORCH_I32
    import torch
    _TORCH_ROWS.update({torch.float32: 0, torch.float16: 1})
    _TORCH_I32 = torch.int32


def _i32(buf, min_len: int, writable: bool = False) -> int:
    """_addr(buf, "i32", ...); what a tensor in order needs comes first, for
    these calls are short."""
    if buf.dtype is _TORCH_I32 and buf.numel() >= min_len and buf.is_contiguous():
        return buf.data_ptr()
    if _TORCH_I32 is None and not isinstance(buf, np.ndarray):
        _torch_types()
    return _addr(buf, "i32", min_len, writable)


def _f32(buf, min_len: int) -> int:
    """_addr(buf, "f32", min_len, writable=True), as _i32."""
    if _TORCH_ROWS.get(buf.dtype) == 0 and buf.numel() >= min_len and buf.is_contiguous():
        return buf.data_ptr()
    return _addr(buf, "f32", min_len, True)


def _bytes(buf, shape) -> int:
    """Address of contiguous bytes (uint8) of the given shape, numpy or torch."""
    if str(buf.dtype) not in ("uint8", "torch.uint8"):
        raise TypeError(f"expected uint8, got {buf.dtype}")
    if tuple(buf.shape) != shape:
        raise ValueError(f"expected shape {shape}, got {tuple(buf.shape)}")
    if isinstance(buf, np.ndarray):
        if not buf.flags.c_contiguous:
            raise ValueError("buffer must be C-contiguous")
        return buf.ctypes.data
    if not buf.is_contiguous():
        raise ValueError("tensor must be contiguous")
    return buf.data_ptr()


def _rows(buf, writable: bool = False):
    """(address, rows, width, row stride in elements, dtype id) of a buffer of
    F32 or F16 rows: [rows, ...] with contiguous rows, any row stride."""
    dt = _TORCH_ROWS.get(buf.dtype)
    if dt is not None and buf.is_contiguous() and buf.dim() >= 2:
        rows = buf.size(0)
        if rows:
            width = buf.numel() // rows
            return buf.data_ptr(), rows, width, width, dt
    shape = buf.shape
    if len(shape) < 2:
        raise ValueError(f"expected [rows, ...], got shape {tuple(shape)}")
    if isinstance(buf, np.ndarray):
        dt = _NP_ROWS.get(buf.dtype)
        if writable and not buf.flags.writeable:
            raise ValueError("buffer is read-only")
        whole, addr = buf.flags.c_contiguous, buf.ctypes.data
    else:
        if _TORCH_I32 is None:
            _torch_types()
        dt = _TORCH_ROWS.get(buf.dtype)
        whole, addr = buf.is_contiguous(), buf.data_ptr()
    if dt is None:
        raise TypeError(f"expected float32 or float16 rows, got {buf.dtype}")
    rows, width = shape[0], 1
    for n in shape[1:]:
        width *= n
    if whole:
        return addr, rows, width, width, dt
    strides = [s // buf.itemsize for s in buf.strides] if isinstance(buf, np.ndarray) else buf.stride()
    inner = 1
    for n, st in zip(reversed(shape[1:]), reversed(strides[1:])):
        if st != inner and n > 1:
            raise ValueError("rows must be contiguous")
        inner *= n
    stride = strides[0] if rows > 1 else width
    if stride < 0 or (writable and stride < width):
        raise ValueError(f"row stride {stride} of rows of {width}")
    return addr, rows, width, stride, dt


class Accelerator:
    """Device handle (hat.Accelerator's role): one lc_context per instance.

    Calls whose buffers are all CUDA tensors only enqueue on the context's own
    stream, which waits for no other stream, and return.  So a program makes the
    tensors of a call, uses its results and frees them on that stream, where
    torch's allocator then sees all uses of their memory too:

        with torch.cuda.stream(torch.cuda.ExternalStream(acc.stream)):
            ...

    or orders the streams by events and keeps the tensors until the calls are
    done, or calls synchronize() (which also reports device-side errors)."""

    def __init__(self, device: int = 0):
        lib = _lib.load()
        h = ctypes.c_void_p()
        _lib.check(lib.lc_context_create(device, ctypes.byref(h)))
        self.device = device
        self.handle = h
        self._fin = weakref.finalize(self, lib.lc_context_destroy, h)

    def synchronize(self) -> None:
        _lib.check(_lib.load().lc_context_synchronize(self.handle))

    @property
    def stream(self) -> int:
        return _lib.load().lc_context_stream(self.handle) or 0

    @property
    def sm_count(self) -> int:
        return _lib.load().lc_context_sm_count(self.handle)

    def close(self) -> None:
        self._fin()


_default_acc: Accelerator | None = None


def default_accelerator() -> Accelerator:
    global _default_acc
    if _default_acc is None:
        _default_acc = Accelerator(0)
    return _default_acc


# ---------------------------------------------------------------- interfaces

class IGEMV(ABC):
    """IGEMV.java:11-69: y = A x, A row-major [rows][cols]."""

    @abstractmethod
    def apply(self, matrix, vector, result, rows: int, cols: int) -> None: ...


class IRMSNorm(ABC):
    """IRMSNorm.java:8-18: in-place RMSNorm."""

    @abstractmethod
    def apply(self, input, weight, size: int) -> None: ...


class IRoPE(ABC):
    """IRoPE.java:8-20: in-place interleaved rotary embedding."""

    @abstractmethod
    def apply(self, vec, pos: int, numHeads: int, headDim: int, theta: float) -> None: ...


class ISiLU(ABC):
    """ISiLU.java:8-17: in-place SiLU."""

    @abstractmethod
    def apply(self, input, size: int) -> None: ...


class ISoftmax(ABC):
    """ISoftmax.java:8-27: in-place softmax of a vector / of one row."""

    @abstractmethod
    def apply(self, input, size: int) -> None: ...

    @abstractmethod
    def applyRow(self, input, rowOffset: int, rowSize: int) -> None: ...


class IAttention(ABC):
    """IAttention.java:8-31: scores and weighted values of one query head."""

    @abstractmethod
    def computeScores(self, query, keys, scores, seqLen: int, headDim: int) -> None: ...

    @abstractmethod
    def computeValues(self, scores, values, output, seqLen: int, headDim: int) -> None: ...


class IKernelFactory(ABC):
    """IKernelFactory.java:9-40."""

    @abstractmethod
    def createGEMV(self, acc: Accelerator | None = None) -> IGEMV: ...

    @abstractmethod
    def createRMSNorm(self, acc: Accelerator | None = None) -> IRMSNorm: ...

    @abstractmethod
    def createRoPE(self, acc: Accelerator | None = None) -> IRoPE: ...

    @abstractmethod
    def createSiLU(self, acc: Accelerator | None = None) -> ISiLU: ...

    @abstractmethod
    def createSoftmax(self, acc: Accelerator | None = None) -> ISoftmax: ...

    @abstractmethod
    def createAttention(self, acc: Accelerator | None = None) -> IAttention: ...


# ----------------------------------------------------------- CUDA kernels

class _CudaKernel:
    def __init__(self, acc: Accelerator | None):
        self.acc = acc or default_accelerator()
        self.lib = _lib.load()

    @property
    def ctx(self):
        return self.acc.handle


class CudaGEMV(_CudaKernel, IGEMV):
    """GEMV on the GPU.  F16 matrices (numpy float16/uint16, the F16Array /
    F16Weights overloads, IGEMV.java:34,50) use the streaming F16 kernel;
    F32 matrices (IGEMV.java:22) the fp32 kernel."""

    def apply(self, matrix, vector, result, rows: int, cols: int) -> None:
        n = rows * cols
        is_f16 = (isinstance(matrix, np.ndarray) and matrix.dtype.type in (np.float16, np.uint16)) or (
            not isinstance(matrix, np.ndarray) and str(getattr(matrix, "dtype", "")) in ("torch.float16", "torch.int16"))
        x = _addr(vector, "f32", cols)
        y = _addr(result, "f32", rows, writable=True)
        if is_f16:
            _lib.check(self.lib.lc_gemv_f16(self.ctx, _addr(matrix, "f16", n), x, y, rows, cols))
        else:
            _lib.check(self.lib.lc_gemv_f32(self.ctx, _addr(matrix, "f32", n), x, y, rows, cols))

    def apply_batched(self, matrix, X, Y, rows: int, cols: int, batch: int) -> None:
        """Y[b] = matrix @ X[b] for b < batch (no reference counterpart)."""
        _lib.check(self.lib.lc_gemv_f16_batched(self.ctx, _addr(matrix, "f16", rows * cols),
                                                _addr(X, "f32", batch * cols),
                                                _addr(Y, "f32", batch * rows, writable=True), rows, cols, batch))

    def tile(self, matrix, tiled, rows: int, cols: int) -> None:
        """Row-major F16 matrix -> the tiled layout of the tensor-core product
        (`tiled`: device memory, rows * cols halves)."""
        n = rows * cols
        _lib.check(self.lib.lc_weights_tile(self.ctx, _addr(matrix, "f16", n), _addr(tiled, "f16", n, writable=True),
                                            rows, cols))

    def apply_batched_tiled_argmax(self, tiled, X, Y, rows: int, cols: int, batch: int, index_offset: int,
                                   keys) -> None:
        """apply_batched_tiled plus packed argmax keys per row (keys: uint64 /
        int64 buffer of `batch`; Y may be None)."""
        y = None if Y is None else _addr(Y, "f32", batch * rows, writable=True)
        if isinstance(keys, np.ndarray):
            if keys.dtype not in (np.uint64, np.int64) or keys.size < batch:
                raise TypeError("keys must be a uint64/int64 array of `batch` entries")
            k = keys.ctypes.data
        else:
            if str(keys.dtype) not in ("torch.int64", "torch.uint64") or keys.numel() < batch:
                raise TypeError("keys must be an int64 tensor of `batch` entries")
            k = keys.data_ptr()
        _lib.check(self.lib.lc_gemm_f16_tiled_argmax(self.ctx, _addr(tiled, "f16", rows * cols),
                                                     _addr(X, "f32", batch * cols), y, rows, cols, batch,
                                                     int(index_offset), k))

    def apply_batched_tiled(self, tiled, X, Y, rows: int, cols: int, batch: int) -> None:
        """Y[b] = W @ X[b] for b < batch <= 64 on the tcgen05 tensor cores; W
        given in the tiled layout (`tile`)."""
        _lib.check(self.lib.lc_gemm_f16_tiled(self.ctx, _addr(tiled, "f16", rows * cols),
                                              _addr(X, "f32", batch * cols),
                                              _addr(Y, "f32", batch * rows, writable=True), rows, cols, batch))


class CudaRMSNorm(_CudaKernel, IRMSNorm):
    """RMSNorm.java:35-50 on the GPU: one fused reduce + normalise kernel."""

    def apply(self, input, weight, size: int) -> None:
        _lib.check(self.lib.lc_rmsnorm(self.ctx, _addr(input, "f32", size, True), _addr(weight, "f32", size), size))

    def apply_rows(self, input, weight, rows: int, width: int, eps: float = 1e-5) -> None:
        _lib.check(self.lib.lc_rmsnorm_rows(self.ctx, _addr(input, "f32", rows * width, True),
                                            _addr(weight, "f32", width), rows, width, eps))


class CudaRoPE(_CudaKernel, IRoPE):
    """RoPE.java:36-52 on the GPU."""

    def apply(self, vec, pos: int, numHeads: int, headDim: int, theta: float) -> None:
        _lib.check(self.lib.lc_rope(self.ctx, _addr(vec, "f32", numHeads * headDim, True), pos, numHeads, headDim,
                                    theta))

    def apply_rows(self, vec, positions, rows: int, numHeads: int, headDim: int, theta: float) -> None:
        _lib.check(self.lib.lc_rope_rows(self.ctx, _addr(vec, "f32", rows * numHeads * headDim, True),
                                         _addr(positions, "i32", rows), rows, numHeads, headDim, theta))


    def apply_scaled(self, x, out, positions, config: RopeConfig, transpose: bool = False) -> None:
        """Rows [rows, heads, head_dim] (F32 or F16) at their positions under a
        RopeConfig (see lc_rope_apply); out may be x.  transpose: the gradient
        of x from that of out.  Rows at negative positions are left as they are.
        CUDA tensors: on the accelerator's stream (see Accelerator)."""
        xa, rows, width, xs, dt = _rows(x)
        if out is x:
            ya, ys = xa, xs
        else:
            ya, orows, owidth, ys, odt = _rows(out, True)
            if (orows, owidth, odt) != (rows, width, dt):
                raise ValueError("x and out differ in shape or type")
        d = config.head_dim
        if width == 0 or width % d:
            raise ValueError(f"rows of {width} elements, head_dim {d}")
        rc = self.lib.lc_rope_apply(self.acc.handle, config.lc, xa, ya, _i32(positions, rows), rows, width // d, xs, ys,
                                    dt, transpose)
        if rc:
            _lib.check(rc)


class CudaPages(_CudaKernel):
    """Page bookkeeping of one serving step (see lc_pages_step), on the
    accelerator's stream (see Accelerator)."""

    def step(self, lens, n_new, table, free_list, free_count, page_size: int, lens_out, q_start, slots, positions,
             seq_ids, free_count_out, status) -> None:
        """lens, n_new [n]; table [n, stride]; free_list [n_pages]; slots,
        positions, seq_ids [capacity]; q_start [n + 1]; free_count(_out) [1];
        status [2] = (code, detail), code 0 when the step was done."""
        n, stride = table.shape
        cap = len(slots)
        rc = self.lib.lc_pages_step(
            self.acc.handle, _i32(lens, n), _i32(n_new, n), n, page_size, _i32(table, n * stride, True),
            stride, _i32(free_list, 1, True), _i32(free_count, 1), len(free_list), cap,
            _i32(lens_out, n, True), _i32(q_start, n + 1, True), _i32(slots, cap, True),
            _i32(positions, cap, True), _i32(seq_ids, cap, True),
            _i32(free_count_out, 1, True), _i32(status, 2, True))
        if rc:
            _lib.check(rc)


class PagedKV8(_CudaKernel):
    """A paged KV cache in 8 bits (see lc_kv8): codes k, v [n_pages, n_kv_heads,
    page_size, head_dim] (uint8, int8 or float8_e4m3fn) and scales k_scale,
    v_scale [n_pages, n_kv_heads] (float32), CUDA tensors that this object keeps
    alive and the caller owns.  Its calls run on the accelerator's stream (see
    Accelerator): what makes or reads these tensors elsewhere is ordered against it."""

    FORMATS = {"i8": 0, "e4m3": 1}

    def __init__(self, k, v, k_scale, v_scale, format: str = "i8", acc: Accelerator | None = None):
        super().__init__(acc)
        if format not in self.FORMATS:
            raise ValueError(f"format {format!r} (of {tuple(self.FORMATS)})")
        n_pages, n_kv, page, d = k.shape
        for codes, scale in ((k, k_scale), (v, v_scale)):
            if tuple(codes.shape) != (n_pages, n_kv, page, d) or tuple(scale.shape) != (n_pages, n_kv):
                raise ValueError("codes are [n_pages, n_kv_heads, page_size, head_dim], scales [n_pages, n_kv_heads]")
            if str(codes.dtype) not in ("torch.uint8", "torch.int8", "torch.float8_e4m3fn"):
                raise TypeError(f"expected 8-bit codes, got {codes.dtype}")
            if str(scale.dtype) != "torch.float32":
                raise TypeError(f"expected float32 scales, got {scale.dtype}")
            if not codes.is_contiguous() or not scale.is_contiguous():
                raise ValueError("codes and scales must be contiguous")
        self.tensors = (k, v, k_scale, v_scale)
        self.n_kv_heads, self.page_size, self.head_dim = n_kv, page, d
        self._width, self._scale = n_kv * d, d ** -0.5
        c = _lib.LcKv8(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n_pages, page, n_kv, d,
                       self.FORMATS[format])
        self._kv = c

    def _two(self, k, v, slots, writable: bool):
        ka, rows, width, stride, dt = _rows(k, writable)
        va, vrows, vwidth, vstride, vdt = _rows(v, writable)
        if vrows != rows or vwidth != width or vstride != stride or vdt != dt:
            raise ValueError("k and v rows differ in shape, stride or type")
        if width != self._width:
            raise ValueError(f"rows of {width} elements, the cache holds {self.n_kv_heads} x {self.head_dim}")
        return ka, va, stride, dt, _i32(slots, rows), rows

    def append(self, k, v, slots) -> None:
        """Rows [rows, n_kv_heads, head_dim] (F32 or F16) into their slots (see lc_kv8_append)."""
        rc = self.lib.lc_kv8_append(self.acc.handle, self._kv, *self._two(k, v, slots, False))
        if rc:
            _lib.check(rc)

    def read(self, k, v, slots) -> None:
        """Rows [rows, n_kv_heads, head_dim] (F32 or F16) = the values at their slots (see lc_kv8_read)."""
        rc = self.lib.lc_kv8_read(self.acc.handle, self._kv, *self._two(k, v, slots, True))
        if rc:
            _lib.check(rc)

    def attention(self, q, out, q_start, kv_lens, table, max_q: int = 1, scale: float | None = None) -> None:
        """Causal attention of rows q [rows, n_heads, head_dim] (see
        lc_kv8_attention); table [n_seqs, stride]; q_start [n_seqs + 1], or None
        when every sequence has one query; scale None: 1 / sqrt(head_dim)."""
        qa, rows, width, qs, dt = _rows(q)
        oa, orows, owidth, os_, odt = _rows(out, True)
        if orows != rows or owidth != width or odt != dt:
            raise ValueError("q and out differ in shape or type")
        d = self.head_dim
        if width == 0 or width % d:
            raise ValueError(f"rows of {width} elements, head_dim {d}")
        n, stride = table.shape
        rc = self.lib.lc_kv8_attention(
            self.acc.handle, self._kv, qa, oa, qs, os_, dt, rows, None if q_start is None else _i32(q_start, n + 1),
            _i32(kv_lens, n), _i32(table, n * stride), stride, n, max_q, width // d,
            self._scale if scale is None else scale)
        if rc:
            _lib.check(rc)


class Weights4(_CudaKernel):
    """A weight matrix [rows, cols] in 4 bits under one scale, and one zero point
    or none, per row and `group` columns (see lc_w4), in CUDA tensors that this
    object keeps alive: codes (uint8), scales (float16) and zeros (uint8, or None
    for 8 throughout), of the sizes that lc_w4_sizes gives; `empty` makes them.
    Its calls run on the accelerator's stream (see Accelerator)."""

    def __init__(self, codes, scales, zeros, rows: int, cols: int, group: int = 128, acc: Accelerator | None = None):
        super().__init__(acc)
        n, m = self.sizes(rows, cols, group)
        for name, t, dtype, want in (("codes", codes, "torch.uint8", n), ("scales", scales, "torch.float16", m),
                                     ("zeros", zeros, "torch.uint8", m)):
            if t is None and name == "zeros":
                continue
            if str(t.dtype) != dtype:
                raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
            if not t.is_contiguous() or t.numel() < want:
                raise ValueError(f"{name}: {t.numel()} elements (contiguous: {t.is_contiguous()}), need {want}")
        self.tensors = (codes, scales, zeros)
        self.rows, self.cols, self.group = rows, cols, group
        self._w = _lib.LcW4(codes.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(), rows, cols,
                            group)

    @staticmethod
    def sizes(rows: int, cols: int, group: int = 128) -> tuple[int, int]:
        """(bytes of codes, number of scales) that a matrix takes."""
        n, m = ctypes.c_int64(), ctypes.c_int64()
        _lib.check(_lib.load().lc_w4_sizes(rows, cols, group, ctypes.byref(n), ctypes.byref(m)))
        return n.value, m.value

    @classmethod
    def empty(cls, rows: int, cols: int, group: int = 128, zeros: bool = False, acc: Accelerator | None = None) -> "Weights4":
        """Room for a matrix on the accelerator's device, to be filled by quantize or pack."""
        import torch
        acc = acc or default_accelerator()
        n, m = cls.sizes(rows, cols, group)
        at = torch.device("cuda", acc.device)
        return cls(torch.empty(n, dtype=torch.uint8, device=at), torch.empty(m, dtype=torch.float16, device=at),
                   torch.empty(m, dtype=torch.uint8, device=at) if zeros else None, rows, cols, group, acc)

    def _values(self, values, writable: bool):
        a, rows, width, stride, dt = _rows(values, writable)
        if (rows, width) != (self.rows, self.cols):
            raise ValueError(f"values [{rows}, {width}], the matrix is [{self.rows}, {self.cols}]")
        return a, stride, dt

    def quantize(self, values) -> None:
        """The matrix from values [rows, cols] (F32 or F16; see lc_w4_quantize)."""
        _lib.check(self.lib.lc_w4_quantize(self.ctx, self._w, *self._values(values, False)))

    def read(self, values) -> None:
        """values [rows, cols] (F32 or F16) = the matrix."""
        _lib.check(self.lib.lc_w4_read(self.ctx, self._w, *self._values(values, True)))

    def pack(self, codes, scales, zeros=None) -> None:
        """The matrix from codes [rows, (cols + 1) // 2] (uint8, the lower column
        in the low half), scales [rows, groups] (F16) and zero points [rows,
        groups] (uint8), as a checkpoint holds them (see lc_w4_pack)."""
        if (zeros is None) != (self.tensors[2] is None):
            raise ValueError("zero points on one side only")
        groups = -(-self.cols // self.group)
        if len(scales.shape) != 1 and tuple(scales.shape) != (self.rows, groups):
            raise ValueError(f"scales {tuple(scales.shape)}, expected [{self.rows}, {groups}]")
        _lib.check(self.lib.lc_w4_pack(
            self.ctx, self._w, _bytes(codes, (self.rows, (self.cols + 1) // 2)),
            _addr(scales, "f16", self.rows * groups), None if zeros is None else _bytes(zeros, (self.rows, groups))))

    def apply(self, x, y, residual=None) -> None:
        """y [batch, rows] = x [batch, cols] W^T, plus residual [batch, rows],
        which may be y; all F32 or all F16 (see lc_w4_product).  The first call
        of an accelerator with more than a few rows makes its workspace: not
        within a graph's capture."""
        xa, batch, width, xs, dt = _rows(x)
        ya, yb, ywidth, ys, ydt = _rows(y, True)
        if width != self.cols or ywidth != self.rows or yb != batch or ydt != dt:
            raise ValueError(f"x [{batch}, {width}] and y [{yb}, {ywidth}] (types {dt}, {ydt}) for a matrix [{self.rows}, {self.cols}]")
        ra, rs = None, 0
        if residual is y:
            ra, rs = ya, ys
        elif residual is not None:
            ra, rb, rwidth, rs, rdt = _rows(residual)
            if rb != batch or rwidth != ywidth or rdt != dt:
                raise ValueError("residual and y differ in shape or type")
        rc = self.lib.lc_w4_product(self.acc.handle, self._w, xa, xs, ya, ys, ra, rs, batch, dt)
        if rc:
            _lib.check(rc)


class CudaLogProbs(_CudaKernel):
    """Log probabilities of given tokens with their ranks, the entropy and the
    best alternatives (see lc_logprobs), on the accelerator's stream (see
    Accelerator)."""

    def apply(self, logits, tokens=None, token_logprobs=None, token_ranks=None, entropy=None, top_ids=None,
              top_logprobs=None, scale: float = 1.0) -> None:
        """logits [rows, vocab] (F32 or F16); tokens, token_ranks [rows] (int32);
        token_logprobs, entropy [rows] (float32); top_ids (int32) and
        top_logprobs (float32) [rows, k], k <= 32.  Outputs that are None are not
        computed.  scale: 1 / temperature."""
        xa, rows, vocab, stride, dt = _rows(logits)
        top = top_ids if top_ids is not None else top_logprobs
        k = 0
        if top is not None:
            k = top.shape[-1]
            for t in (top_ids, top_logprobs):
                if t is not None and tuple(t.shape) != (rows, k):
                    raise ValueError(f"top outputs are [{rows}, k], got {tuple(t.shape)}")
        rc = self.lib.lc_logprobs(
            self.acc.handle, xa, stride, dt, rows, vocab, scale, None if tokens is None else _i32(tokens, rows),
            None if token_logprobs is None else _f32(token_logprobs, rows),
            None if token_ranks is None else _i32(token_ranks, rows, True),
            None if entropy is None else _f32(entropy, rows), k,
            None if top_ids is None else _i32(top_ids, rows * k, True),
            None if top_logprobs is None else _f32(top_logprobs, rows * k))
        if rc:
            _lib.check(rc)


class CudaSiLU(_CudaKernel, ISiLU):
    """SiLU.java:32-40 on the GPU."""

    def apply(self, input, size: int) -> None:
        _lib.check(self.lib.lc_silu(self.ctx, _addr(input, "f32", size, True), size))

    def swiglu(self, gate, up, n: int) -> None:
        """gate = silu(gate) * up (TransformerBlock.java:209-210)."""
        _lib.check(self.lib.lc_swiglu(self.ctx, _addr(gate, "f32", n, True), _addr(up, "f32", n), n))


class CudaSoftmax(_CudaKernel, ISoftmax):
    """Softmax.java:28-84 on the GPU (online-statistics single kernel)."""

    def apply(self, input, size: int) -> None:
        _lib.check(self.lib.lc_softmax(self.ctx, _addr(input, "f32", size, True), size))

    def applyRow(self, input, rowOffset: int, rowSize: int) -> None:
        _lib.check(self.lib.lc_softmax_row(self.ctx, _addr(input, "f32", rowOffset + rowSize, True), rowOffset,
                                           rowSize))

    def apply_rows(self, input, rows: int, width: int) -> None:
        _lib.check(self.lib.lc_softmax_rows(self.ctx, _addr(input, "f32", rows * width, True), rows, width))


class CudaAttention(_CudaKernel, IAttention):
    """Attention.java:32-61 on the GPU, plus the fused GQA decode kernel."""

    def computeScores(self, query, keys, scores, seqLen: int, headDim: int) -> None:
        _lib.check(self.lib.lc_attn_scores(self.ctx, _addr(query, "f32", headDim), _addr(keys, "f32", seqLen * headDim),
                                           _addr(scores, "f32", seqLen, True), seqLen, headDim))

    def computeValues(self, scores, values, output, seqLen: int, headDim: int) -> None:
        _lib.check(self.lib.lc_attn_values(self.ctx, _addr(scores, "f32", seqLen), _addr(values, "f32", seqLen * headDim),
                                           _addr(output, "f32", headDim, True), seqLen, headDim))

    def decode(self, q, k, v, out, seq_len, batch: int, n_heads: int, n_kv_heads: int, head_dim: int,
               seq_stride: int, head_stride: int, pos_stride: int) -> None:
        """Fused GQA attention for one query token per sequence (see lc_attention_decode)."""
        _lib.check(self.lib.lc_attention_decode(
            self.ctx, _addr(q, "f32", batch * n_heads * head_dim), _addr(k, "f32", 1), _addr(v, "f32", 1),
            _addr(out, "f32", batch * n_heads * head_dim, True), _addr(seq_len, "i32", batch), batch, n_heads,
            n_kv_heads, head_dim, seq_stride, head_stride, pos_stride))

    def decode_maxlen(self, q, k, v, out, seq_len, batch: int, n_heads: int, n_kv_heads: int, head_dim: int,
                      seq_stride: int, head_stride: int, pos_stride: int, max_len: int) -> None:
        """decode with the split plan sized for max_len >= every seq_len (see
        lc_attention_decode_maxlen): enqueue-only with device buffers."""
        _lib.check(self.lib.lc_attention_decode_maxlen(
            self.ctx, _addr(q, "f32", batch * n_heads * head_dim), _addr(k, "f32", 1), _addr(v, "f32", 1),
            _addr(out, "f32", batch * n_heads * head_dim, True), _addr(seq_len, "i32", batch), batch, n_heads,
            n_kv_heads, head_dim, seq_stride, head_stride, pos_stride, max_len))


class CudaKernelFactory(IKernelFactory):
    """The B200 sibling of PlainJavaKernelFactory (PlainJavaKernelFactory.java:9-40)."""

    def createGEMV(self, acc=None) -> CudaGEMV:
        return CudaGEMV(acc)

    def createRMSNorm(self, acc=None) -> CudaRMSNorm:
        return CudaRMSNorm(acc)

    def createRoPE(self, acc=None) -> CudaRoPE:
        return CudaRoPE(acc)

    def createPages(self, acc=None) -> CudaPages:
        return CudaPages(acc)

    def createLogProbs(self, acc=None) -> CudaLogProbs:
        return CudaLogProbs(acc)

    def createSiLU(self, acc=None) -> CudaSiLU:
        return CudaSiLU(acc)

    def createSoftmax(self, acc=None) -> CudaSoftmax:
        return CudaSoftmax(acc)

    def createAttention(self, acc=None) -> CudaAttention:
        return CudaAttention(acc)


def argmax(values, acc: Accelerator | None = None) -> int:
    """LlamaInference.argmax (LlamaInference.java:252-262) on the GPU."""
    acc = acc or default_accelerator()
    out = np.zeros(1, np.int32)
    _lib.check(_lib.load().lc_argmax(acc.handle, _addr(values, "f32", 1), int(np.asarray(values).size if isinstance(values, np.ndarray) else values.numel()), out.ctypes.data))
    return int(out[0])

"""8-bit rows and their product (clq_quantize_rows_device, clq_norm_quantize_device,
clq_swiglu_quantize_device, clq_dequantize_rows_device, clq_linear_int8_device).

An Int8Rows holds rows of int8 codes with one f32 scale a row: the tokens of an
activation, or the output channels of a weight.  The steps of a decoder layer
(local/blocks.lisp:327-392) in 8-bit activations:

  wq = quantize_rows(w)                       once: a weight [n, k], or store.dequantize()
  q, h = norm_quantize(y, norm_w, eps, residual=h)   residual add + RMSNorm + rounding
  gate_up = linear_int8(q, wq)                [m, 2 f], f32 / bf16 / f16
  q = swiglu_quantize(gate_up[:, :f], gate_up[:, f:])
  y = linear_int8(q, w_down)

Tensors are on the current CUDA device, rows with a unit last stride (others
are copied) and any row stride (of codes and of a product's residual, rows that
share memory are copied).  Work is queued on the current stream, or on
STREAM (a cudaStream_t handle): outputs then belong to that stream.
"""
from . import _lib
from .store import _XTYPE

_lib_quantize = _lib.lib.clq_norm_quantize_device
_lib_swiglu = _lib.lib.clq_swiglu_quantize_device
_lib_dequantize = _lib.lib.clq_dequantize_rows_device
_lib_linear = _lib.lib.clq_linear_int8_device

# Filled in by _torch() at the first call: the package imports without torch.
_t = None           # the torch module
_types = {}         # torch dtype -> clq_xtype
_device = None      # () -> index of the current device
_stream = None      # device index -> handle of its current stream


def _torch():
    global _t, _device, _stream
    if _t is None:
        import torch
        _types.update((getattr(torch, name), code) for name, code in _XTYPE.items())
        # a decoded token's call takes a few microseconds: torch's own accessors, without the objects around them
        _device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        _stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda d: torch.cuda.current_stream(d).cuda_stream)
        _t = torch
    return _t


def _type_code(dtype, what):
    code = _types.get(dtype)
    if code is None:
        raise ValueError(f"{what}: float32, bfloat16 or float16, not {dtype}")
    return code


def _plain(t, dtype, dims):
    """Whether T is a tensor of that type and rank on the current device with
    unit last stride: what nearly every call has, told in one go."""
    return (type(t) is _t.Tensor and t.dtype is dtype and t.dim() == dims and t.is_cuda and t.get_device() == _device()
            and t.stride(dims - 1) == 1)


def _matrix(t, what, shape=None):
    """T as a CUDA matrix on the current device with unit last stride."""
    if not isinstance(t, _t.Tensor) or not t.is_cuda or t.dim() != 2:
        raise ValueError(f"{what}: a CUDA matrix")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what} is {tuple(t.shape)}, {tuple(shape)} is wanted")
    _here(t, what)
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _rows_apart(t):
    """T and its row stride, or a copy's where rows share memory (one row for every token, say)."""
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t, t.stride(0)


def _vector(t, n, what):
    if not isinstance(t, _t.Tensor) or not t.is_cuda or t.dtype != _t.float32 or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{what}: a CUDA float32 vector of {n}")
    _here(t, what)
    return t if n <= 1 or t.stride(0) == 1 else t.contiguous()


def _writable(t, what, shape, dtype):
    """T as an output: nothing may be copied, and its rows must not share memory."""
    if (not isinstance(t, _t.Tensor) or not t.is_cuda or t.dtype != dtype or t.shape != shape
            or t.get_device() != _device() or (shape[1] > 1 and t.stride(1) != 1)
            or (shape[0] > 1 and t.stride(0) < shape[1])):
        raise ValueError(f"{what}: a {dtype} matrix {tuple(shape)} on the current device, rows apart with unit last stride")
    return t


def _here(t, what):
    """The current device's index, which must be T's."""
    device = _device()
    if t.get_device() != device:
        raise ValueError(f"{what} lives on device {t.get_device()}, current device is {device}")
    return device


def _on(stream, tensors, call):
    """CALL() with STREAM (a handle) as the current stream, so that what it
    allocates belongs to that stream; TENSORS are kept until STREAM is done
    (CALL refuses what is none, or not on the device)."""
    side = _t.cuda.ExternalStream(stream)
    for t in tensors:
        if isinstance(t, _t.Tensor) and t.is_cuda:
            t.record_stream(side)
    with _t.cuda.stream(side):
        return call()


class Int8Rows:
    """CODES int8 [m, k] (any row stride, unit last stride) and SCALES f32 [m]."""

    __slots__ = ("codes", "scales")

    def __init__(self, codes, scales):
        torch = _t or _torch()
        if not (_plain(codes, torch.int8, 2) and _plain(scales, torch.float32, 1)
                and scales.shape[0] == codes.shape[0]):
            codes = _matrix(codes, "codes")
            if codes.dtype != torch.int8:
                raise ValueError(f"codes: int8, not {codes.dtype}")
            scales = _vector(scales, codes.shape[0], "scales")
        self.codes, self.scales = codes, scales

    @property
    def shape(self):
        return self.codes.shape

    def __len__(self):
        return self.codes.shape[0]

    def __getitem__(self, rows):
        """Rows by a slice with step 1, sharing the memory (a row range of a weight)."""
        if not isinstance(rows, slice) or rows.step not in (None, 1):
            raise TypeError("Int8Rows takes slices of rows")
        return Int8Rows(self.codes[rows], self.scales[rows])

    def dequantize(self, dtype=None, out=None, stream=None):
        """codes * scales in DTYPE (float32 without one), into OUT when given."""
        torch = _t or _torch()
        codes, scales = self.codes, self.scales
        if stream is not None:
            return _on(stream, (codes, scales, out), lambda: self.dequantize(dtype, out))
        m, k = codes.shape
        device = _device()
        if codes.get_device() != device:
            _here(codes, "codes")
        if dtype is None:
            dtype = torch.float32 if out is None else getattr(out, "dtype", None)
        code = _types.get(dtype)
        if code is None:
            _type_code(dtype, "dtype")
        ldo = k
        if out is not None:
            _writable(out, "out", (m, k), dtype)
            ldo = out.stride(0)
        elif codes.is_contiguous():
            out = torch.empty_like(codes, dtype=dtype)
        else:
            out = codes.new_empty((m, k), dtype=dtype)
        ldc = codes.stride(0)
        if ldc < k:
            codes, ldc = _rows_apart(codes)
        status = _lib_dequantize(codes.data_ptr(), ldc, scales.data_ptr(), m, k, out.data_ptr(), code, ldo,
                                 _stream(device))
        if status:
            _lib.check(status)
        return out


def _empty_rows(x, m, k):
    """Uninitialised Int8Rows beside X whose code rows start on 16-byte
    boundaries, and their row stride."""
    q = Int8Rows.__new__(Int8Rows)
    pitch = (k + 15) // 16 * 16
    if pitch == k and x.is_contiguous():
        q.codes = _t.empty_like(x, dtype=_t.int8)
    else:
        q.codes = x.new_empty((m, pitch), dtype=_t.int8)[:, :k]
    q.scales = x.new_empty(m, dtype=_t.float32)
    return q, pitch


def quantize_rows(x, stream=None):
    """The Int8Rows of X [m, k] (float32, bfloat16 or float16)."""
    return norm_quantize(x, stream=stream)


def norm_quantize(x, norm_weight=None, eps=1e-5, residual=None, residual_out=None, stream=None):
    """The Int8Rows of RMSNorm(x + residual) * norm_weight, in one pass over the rows.

    Without NORM_WEIGHT (f32 [k]) the sum itself is coded; without RESIDUAL (x's
    type, or f32) x alone.  With a residual returns (rows, x + residual), the sum
    in the residual's type: RESIDUAL_OUT, which may be RESIDUAL, or a new tensor.
    A row that is not finite, or whose mean square + EPS is not within f32 (from 2^-125
    on), has codes 0 and the scale NaN.
    """
    torch = _t or _torch()
    if stream is not None:
        return _on(stream, (x, norm_weight, residual, residual_out),
                   lambda: norm_quantize(x, norm_weight, eps, residual, residual_out))
    if not _plain(x, getattr(x, "dtype", None), 2):
        x = _matrix(x, "x")
    m, k = x.shape
    xtype = _types.get(x.dtype)
    if xtype is None:
        _type_code(x.dtype, "x")
    wptr = rptr = optr = None
    rtype, ldr, ldo = xtype, 0, 0
    if norm_weight is not None:
        if not _plain(norm_weight, torch.float32, 1) or norm_weight.shape[0] != k:
            norm_weight = _vector(norm_weight, k, "norm_weight")
        wptr = norm_weight.data_ptr()
    if residual is not None:
        given = residual
        if not _plain(residual, getattr(residual, "dtype", None), 2) or residual.shape != x.shape:
            residual = _matrix(residual, "residual", x.shape)
        rtype = _type_code(residual.dtype, "residual")
        if rtype not in (xtype, _lib.CLQ_X_F32):
            raise ValueError(f"residual: {x.dtype} or float32, not {residual.dtype}")
        if residual_out is None:
            residual_out = torch.empty_like(residual) if residual.is_contiguous() else residual.new_empty((m, k))
        else:
            _writable(residual_out, "residual_out", (m, k), residual.dtype)
            _apart(residual_out, given, "residual_out")
            _apart(residual_out, x, "residual_out")
        rptr, ldr = residual.data_ptr(), residual.stride(0)
        optr, ldo = residual_out.data_ptr(), residual_out.stride(0)
    elif residual_out is not None:
        raise ValueError("residual_out needs a residual")
    q, pitch = _empty_rows(x, m, k)
    status = _lib_quantize(x.data_ptr(), xtype, m, k, x.stride(0), wptr, eps, rptr, rtype, ldr, optr, ldo, q.codes.data_ptr(),
                           pitch, q.scales.data_ptr(), _stream(_device()))
    if status:
        _lib.check(status)
    return q if residual is None else (q, residual_out)


def swiglu_quantize(gate, up, stream=None):
    """The Int8Rows of silu(gate) * up, both [m, k] of one type (two halves of one product, say)."""
    _t or _torch()
    if stream is not None:
        return _on(stream, (gate, up), lambda: swiglu_quantize(gate, up))
    if not _plain(gate, getattr(gate, "dtype", None), 2):
        gate = _matrix(gate, "gate")
    if not _plain(up, getattr(up, "dtype", None), 2) or up.shape != gate.shape:
        up = _matrix(up, "up", gate.shape)
    if gate.dtype != up.dtype:
        raise ValueError(f"gate is {gate.dtype}, up is {up.dtype}")
    xtype = _type_code(gate.dtype, "gate")
    m, k = gate.shape
    q, pitch = _empty_rows(gate, m, k)
    status = _lib_swiglu(gate.data_ptr(), gate.stride(0), up.data_ptr(), up.stride(0), xtype, m, k, q.codes.data_ptr(), pitch,
                         q.scales.data_ptr(), _stream(_device()))
    if status:
        _lib.check(status)
    return q


def linear_int8(x, w, out=None, dtype=None, residual=None, stream=None):
    """out[m, n] = X [m, k] . W [n, k]^T of two Int8Rows, plus an optional f32
    RESIDUAL [m, n] (which may be OUT), rounded once to DTYPE (OUT's, or float32).
    The products are summed in 32-bit integers: exact, for k up to 131071."""
    torch = _t or _torch()
    if not isinstance(x, Int8Rows) or not isinstance(w, Int8Rows):
        raise ValueError("linear_int8 multiplies Int8Rows")
    if stream is not None:
        return _on(stream, (x.codes, x.scales, w.codes, w.scales, out, residual),
                   lambda: linear_int8(x, w, out, dtype, residual))
    xc, wc = x.codes, w.codes
    m, k = xc.shape
    n, wk = wc.shape
    if wk != k:
        raise ValueError(f"rows of {k} codes against a weight of {tuple(wc.shape)}")
    device = _device()
    if xc.get_device() != device or wc.get_device() != device:
        _here(xc, "x")
        _here(wc, "w")
    if dtype is None:
        dtype = torch.float32 if out is None else getattr(out, "dtype", None)
    code = _types.get(dtype)
    if code is None:
        _type_code(dtype, "dtype")
    rptr, ldr, ldo = None, 0, n
    if out is not None:
        _writable(out, "out", (m, n), dtype)
        ldo = out.stride(0)
    if residual is not None:
        given = residual
        if not _plain(residual, torch.float32, 2) or residual.shape != (m, n):
            residual = _matrix(residual, "residual", (m, n))
            if residual.dtype != torch.float32:
                raise ValueError(f"residual: float32, not {residual.dtype}")
        if out is not None:
            _apart(out, given, "out")
        ldr = residual.stride(0)
        if ldr < n:
            residual, ldr = _rows_apart(residual)
        rptr = residual.data_ptr()
    if out is None:
        out = xc.new_empty((m, n), dtype=dtype)
    ldx, ldw = xc.stride(0), wc.stride(0)
    if ldx < k:
        xc, ldx = _rows_apart(xc)
    if ldw < k:
        wc, ldw = _rows_apart(wc)
    status = _lib_linear(xc.data_ptr(), ldx, x.scales.data_ptr(), m, wc.data_ptr(), ldw, w.scales.data_ptr(), n, k, rptr, ldr,
                         out.data_ptr(), code, ldo, _stream(device))
    if status:
        _lib.check(status)
    return out


def _span(t):
    """First byte and the byte after the last of a matrix."""
    a = t.data_ptr()
    reach = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
    return a, a + (reach + 1) * t.element_size()


def _overlap(a, b):
    """Whether two matrices of unit last stride share memory."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a0 >= b1 or b0 >= a1:
        return False
    pitch = a.stride(0) * a.element_size()
    if pitch > 0 and pitch == b.stride(0) * b.element_size():  # columns of one buffer, side by side
        at = (b0 - a0) % pitch
        return at < a.shape[1] * a.element_size() or at + b.shape[1] * b.element_size() > pitch
    return True


def _apart(out, given, what):
    """Refuses an output that shares memory with an input other than by being it."""
    if out is not given and _overlap(out, given) and not (
            out.data_ptr() == given.data_ptr() and out.stride() == given.stride() and out.dtype == given.dtype):
        raise ValueError(f"{what}: the input itself, or memory apart from it")

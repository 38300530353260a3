"""Activations kept in 8 bits for the backward pass.

A fault-tolerant replica holds more than its model: DiLoCo and LocalSGD keep a backup (and an
outer momentum) of every parameter on the GPU, DDP its gradient buckets.  What is left for
activations decides the micro-batch, and a linear layer needs its input in the backward pass for
one thing only, the weight gradient.  Here that input is kept as E4M3 numbers with one
power-of-two scale per block of 128 features - half the bytes of bf16, a quarter of fp32's - and
the weight gradient is computed from that form directly.  The root-mean-square norm writes its
normalised rows in the same form on its way, for its own backward pass and for every linear layer
behind it: one byte per element in place of the norm's input and output.

The forward pass computes what it computes without packing; gradients are those of the stored
values (an element is off by at most 2^-4 of itself, or 2^-10 of its block's scale where it is
tiny).

``pack_activations(module)`` switches the ``nn.Linear`` and ``nn.RMSNorm`` modules of a model
over; ``DistributedDataParallel(..., packed_activations=True)`` does it while wrapping.  The
functions below work on tensors.  All of them enqueue on torch's current stream of the tensors'
device, never synchronise, and have no CPU path.  The reference has no counterpart.
"""

from __future__ import annotations

import math
from collections import OrderedDict
from typing import NamedTuple, Optional, Tuple

import torch
import torch.nn.functional as F
from torch import nn
from torch.utils.weak import TensorWeakRef

from . import _native

BLOCK = 128  # features that share a scale
MAX_NORM_FEATURES = 16384
_WGRAD_ROW_BYTES = 1 << 25  # the weight gradient's kernel addresses 64 rows of a gradient with 31 bits

_DTYPES = {
    torch.float32: _native.TFT_F32,
    torch.bfloat16: _native.TFT_BF16,
    torch.float16: _native.TFT_F16,
}


def _dtype_code(dtype: torch.dtype, what: str) -> int:
    try:
        return _DTYPES[dtype]
    except KeyError:
        raise TypeError(f"{what}: float32, bfloat16 and float16 are supported, got {dtype}") from None


def _raw_stream(index: int) -> int:
    # looked up when called, as below: a build of torch without GPU support lacks it, and imports this
    return torch._C._cuda_getCurrentRawStream(index)


def _launch(name: str, device: torch.device, *args: object) -> None:
    """One C entry on the device's current stream.  The smallest calls are a few microseconds of
    GPU time, so the device is only switched where it is not the current one, and the stream is
    asked for without an object around it (1.2 and 1.8 microseconds of 10)."""
    index = device.index
    fn = getattr(_native.lib(), name)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _native.check(rc, name)


def _require_gpu(t: torch.Tensor, what: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(
            f"{what}: tensor is on {t.device}; the torchft_amd kernels only run on GPU "
            "tensors (there is no CPU path)"
        )


def _require_same_device(t: torch.Tensor, device: torch.device, what: str) -> None:
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        _require_gpu(t, what)
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, expected {device}")


def _matrix(x: torch.Tensor, what: str) -> Tuple[int, int, int]:
    """(rows, features, row stride) of a tensor as the matrix of its last dimension's rows."""
    _require_gpu(x, what)
    if x.dim() == 0:
        raise ValueError(f"{what}: a scalar has no rows")
    features = x.shape[-1]
    if features == 0 or x.numel() == 0:
        return math.prod(x.shape[:-1]), features, features
    if features > 1 and x.stride(-1) != 1:
        raise ValueError(f"{what}: the elements of a row must be consecutive, strides are {x.stride()}")
    if x.dim() == 2 and x.shape[0] > 1:
        return x.shape[0], features, x.stride(0)
    if x.is_contiguous() or x.numel() == features:
        return x.numel() // features, features, features
    try:
        m = x.view(-1, features)
    except RuntimeError:
        raise ValueError(
            f"{what}: shape {tuple(x.shape)} with strides {x.stride()} is not one matrix of rows; "
            "call .contiguous() first"
        ) from None
    return m.shape[0], features, m.stride(0)


def _as_rows(x: torch.Tensor) -> torch.Tensor:
    """x, or a contiguous copy where its rows have no common stride."""
    try:
        _matrix(x, "")
    except ValueError:
        return x.contiguous()
    return x


def _contiguous_like(x: torch.Tensor) -> torch.Tensor:
    if x.is_contiguous():
        return torch.empty_like(x, requires_grad=False)
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _pitch(features: int) -> int:
    return (features + 15) // 16 * 16


def _blocks(features: int) -> int:
    return (features + BLOCK - 1) // BLOCK


def _vector(t: Optional[torch.Tensor], features: int, device: torch.device, what: str) -> None:
    if t is None:
        return
    _require_same_device(t, device, what)
    if t.dim() != 1 or t.shape[0] != features or (features > 1 and t.stride(0) != 1):
        raise ValueError(
            f"{what}: expected {features} consecutive elements, got shape {tuple(t.shape)} "
            f"with strides {t.stride()}"
        )
    _dtype_code(t.dtype, what)


def _version(t: Optional[torch.Tensor]) -> Optional[int]:
    """How often t was written to, as far as torch counts (not for tensors of inference mode)."""
    return None if t is None or t.is_inference() else t._version


class PackedActivation:
    """An activation in 8 bits: E4M3 ``values`` of [rows, features rounded up to 16] and biased
    ``exponents`` (uint8) of [rows, blocks of 128 features].  An element stands for
    ``value * 2 ** (exponent - 127)``, times ``column_scale`` of its feature where there is one
    (a norm's weight, the live one: a write to it changes what the form stands for, and
    :func:`linear` refuses the form from then on).  ``shape`` is the packed tensor's and ``dtype`` its
    type."""

    __slots__ = ("values", "exponents", "features", "shape", "dtype", "column_scale", "_scale_version")

    def __init__(
        self,
        values: torch.Tensor,
        exponents: torch.Tensor,
        features: int,
        column_scale: Optional[torch.Tensor] = None,
        shape: Optional[Tuple[int, ...]] = None,
        dtype: Optional[torch.dtype] = None,
    ) -> None:
        _require_gpu(values, "PackedActivation: values")
        device = values.device
        _require_same_device(exponents, device, "PackedActivation: exponents")
        if values.dtype not in (torch.float8_e4m3fn, torch.uint8) or exponents.dtype != torch.uint8:
            raise TypeError("PackedActivation: expected float8_e4m3fn (or uint8) values and uint8 "
                            f"exponents, got {values.dtype} and {exponents.dtype}")
        if features < 0 or values.dim() != 2 or values.shape[1] != _pitch(features) \
                or not values.is_contiguous():
            raise ValueError(f"PackedActivation: values must be contiguous [rows, {_pitch(features)}] for "
                             f"{features} features, got {tuple(values.shape)}")
        rows = values.shape[0]
        if exponents.shape != (rows, _blocks(features)) or not exponents.is_contiguous():
            raise ValueError(f"PackedActivation: exponents must be contiguous "
                             f"{(rows, _blocks(features))}, got {tuple(exponents.shape)}")
        if values.data_ptr() % 16:
            raise ValueError("PackedActivation: values must start at a multiple of 16 bytes")
        _vector(column_scale, features, device, "PackedActivation: column_scale")
        if shape is None:
            shape = (rows, features)
        else:
            shape = tuple(shape)
            if not shape or shape[-1] != features or math.prod(shape[:-1]) != rows:
                raise ValueError(f"PackedActivation: shape {shape} does not hold {rows} rows of "
                                 f"{features} features")
        if dtype is None:
            dtype = torch.bfloat16 if column_scale is None else column_scale.dtype
        _dtype_code(dtype, "PackedActivation")
        self.values = values
        self.exponents = exponents
        self.features = features
        self.shape = shape
        self.dtype = dtype
        self.column_scale = column_scale
        self._scale_version = _version(column_scale)

    @property
    def rows(self) -> int:
        return self.values.shape[0]

    @property
    def device(self) -> torch.device:
        return self.values.device

    @property
    def nbytes(self) -> int:
        return self.values.numel() + self.exponents.numel()

    def record_stream(self, stream: "torch.cuda.Stream") -> None:
        """``torch.Tensor.record_stream`` of the two buffers: for a packed form that another stream
        than the one it was made on reads."""
        self.values.record_stream(stream)
        self.exponents.record_stream(stream)

    def _scale_is_as_packed(self) -> bool:
        """Whether the column scale (a norm's live weight) is still the one that the packed
        tensor was computed with."""
        return _version(self.column_scale) == self._scale_version

    def __reduce__(self) -> tuple:  # a copy's column scale counts its writes anew
        return _restored, (self.values, self.exponents, self.features, self.column_scale, self.shape, self.dtype,
                           self._scale_is_as_packed())

    def unpack(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The stored values, contiguous, rounded to ``dtype`` (the packed tensor's own by
        default; without a column scale they are exact in bf16 and fp32)."""
        dtype = self.dtype if dtype is None else dtype
        code = _dtype_code(dtype, "unpack")
        device = self.values.device
        out = torch.empty(self.shape, dtype=dtype, device=device)
        scale = self.column_scale
        _launch(
            "tft_unpack_e4m3", device, out.data_ptr(), self.values.data_ptr(), self.exponents.data_ptr(),
            None if scale is None else scale.data_ptr(), self.rows, self.features,
            self.values.shape[1], code if scale is None else _DTYPES[scale.dtype], code,
        )
        return out


def _trusted(values, exponents, features, column_scale, shape, dtype) -> PackedActivation:
    """A PackedActivation of buffers made here."""
    p = PackedActivation.__new__(PackedActivation)
    p.values, p.exponents, p.features = values, exponents, features
    p.shape, p.dtype, p.column_scale = shape, dtype, column_scale
    p._scale_version = _version(column_scale)
    return p


def _restored(values, exponents, features, column_scale, shape, dtype, scale_is_as_packed) -> PackedActivation:
    p = _trusted(values, exponents, features, column_scale, shape, dtype)
    if not scale_is_as_packed:
        p._scale_version = -1
    return p


def _buffers(rows: int, features: int, device: torch.device) -> Tuple[torch.Tensor, torch.Tensor]:
    return (
        torch.empty(rows, _pitch(features), dtype=torch.float8_e4m3fn, device=device),
        torch.empty(rows, _blocks(features), dtype=torch.uint8, device=device),
    )


def pack(x: torch.Tensor) -> PackedActivation:
    """x in 8 bits, blocks of 128 along its last dimension.  The rows of x may have any common
    stride.  Infinities and NaN are kept as NaN and do not touch their block's other elements."""
    rows, features, stride = _matrix(x, "pack")
    code = _dtype_code(x.dtype, "pack")
    device = x.device
    values, exponents = _buffers(rows, features, device)
    _launch(
        "tft_pack_e4m3", device, values.data_ptr(), exponents.data_ptr(), x.data_ptr(), rows, features,
        stride, values.shape[1], code,
    )
    return _trusted(values, exponents, features, None, tuple(x.shape), x.dtype)


def _check_norm_weight(weight: Optional[torch.Tensor], dtype: torch.dtype, what: str) -> None:
    if weight is not None and weight.dtype not in (dtype, torch.float32):
        raise TypeError(f"{what}: the weight is {weight.dtype}, expected {dtype} or float32")


def rms_norm_forward(
    x: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    eps: Optional[float] = None,
    residual: Optional[torch.Tensor] = None,
    pack: bool = True,
) -> Tuple[torch.Tensor, torch.Tensor, Optional[PackedActivation], torch.Tensor]:
    """(y, h, packed, rstd) with h = x + residual rounded to x's type (x itself without a
    residual), rstd = 1 / sqrt(mean(h^2) + eps) in fp32 of [rows], y = h * rstd * weight, and the
    normalised rows h * rstd packed with ``weight`` as their column scale.  ``eps=None`` is fp32's
    machine epsilon whatever x's type, as torch's norm takes that of the type it computes in.  No
    autograd: see :func:`rms_norm`."""
    rows, features, stride = _matrix(x, "rms_norm: x")
    dtype, device = x.dtype, x.device
    code = _dtype_code(dtype, "rms_norm")
    if features > MAX_NORM_FEATURES:
        raise ValueError(f"rms_norm: {features} features, at most {MAX_NORM_FEATURES}")
    _vector(weight, features, device, "rms_norm: weight")
    _check_norm_weight(weight, dtype, "rms_norm")
    if eps is None:
        eps = torch.finfo(torch.float32).eps
    if not eps >= 0.0:
        raise ValueError(f"rms_norm: eps must be at least 0, got {eps}")
    residual_stride = 0
    if residual is not None:
        _require_same_device(residual, device, "rms_norm: residual")
        if residual.shape != x.shape or residual.dtype != dtype:
            raise ValueError(f"rms_norm: residual is {residual.dtype}{list(residual.shape)}, "
                             f"x is {dtype}{list(x.shape)}")
        _, _, residual_stride = _matrix(residual, "rms_norm: residual")
    y = _contiguous_like(x)
    h = x if residual is None else _contiguous_like(x)
    rstd = torch.empty(rows, dtype=torch.float32, device=device)
    if features == 0:
        rstd.fill_(math.nan)  # the mean of nothing; the kernel has no rows to write it for
    values = exponents = packed = None
    if pack:
        values, exponents = _buffers(rows, features, device)
        packed = _trusted(values, exponents, features, weight, tuple(x.shape), dtype)
    _launch(
        "tft_rms_norm", device, y.data_ptr(), None if residual is None else h.data_ptr(),
        values.data_ptr() if pack else None, exponents.data_ptr() if pack else None,
        rstd.data_ptr(), x.data_ptr(), None if residual is None else residual.data_ptr(),
        None if weight is None else weight.data_ptr(), rows, features, stride, residual_stride,
        values.shape[1] if pack else 0, eps, code if weight is None else _DTYPES[weight.dtype], code,
    )
    return y, h, packed, rstd


def rms_norm_backward(
    grad_y: torch.Tensor,
    packed: PackedActivation,
    rstd: torch.Tensor,
    grad_h: Optional[torch.Tensor] = None,
    weight_grad: bool = True,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(grad_x, grad_weight) of :func:`rms_norm_forward` from what it packed.  ``grad_h`` is the
    gradient that reaches h from its other readers; ``grad_x`` is the residual's gradient too.
    ``grad_weight`` has the weight's type and is None where there is no weight."""
    rows, features, stride = _matrix(grad_y, "rms_norm_backward: grad_y")
    dtype, device = grad_y.dtype, grad_y.device
    code = _dtype_code(dtype, "rms_norm_backward")
    weight = packed.column_scale
    if (rows, features) != (packed.rows, packed.features):
        raise ValueError(f"rms_norm_backward: grad_y has {rows} rows of {features}, packed {packed.rows} "
                         f"rows of {packed.features}")
    if features > MAX_NORM_FEATURES:
        raise ValueError(f"rms_norm_backward: {features} features, at most {MAX_NORM_FEATURES}")
    _require_same_device(packed.values, device, "rms_norm_backward: packed")
    _check_norm_weight(weight, dtype, "rms_norm_backward")
    _require_same_device(rstd, device, "rms_norm_backward: rstd")
    if rstd.dtype != torch.float32 or rstd.numel() != rows or not rstd.is_contiguous():
        raise ValueError(f"rms_norm_backward: rstd must be {rows} consecutive float32 numbers")
    grad_h_stride = 0
    if grad_h is not None:
        _require_same_device(grad_h, device, "rms_norm_backward: grad_h")
        if grad_h.shape != grad_y.shape or grad_h.dtype != dtype:
            raise ValueError(f"rms_norm_backward: grad_h is {grad_h.dtype}{list(grad_h.shape)}, grad_y is "
                             f"{dtype}{list(grad_y.shape)}")
        _, _, grad_h_stride = _matrix(grad_h, "rms_norm_backward: grad_h")
    grad_x = _contiguous_like(grad_y)
    grad_weight = workspace = None
    need = 0
    if weight is not None and weight_grad:
        grad_weight = torch.empty(features, dtype=weight.dtype, device=device)
        need = _native.lib().tft_rms_norm_backward_workspace(rows, features)
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    _launch(
        "tft_rms_norm_backward", device, grad_x.data_ptr(),
        None if grad_weight is None else grad_weight.data_ptr(),
        None if workspace is None else workspace.data_ptr(), need, grad_y.data_ptr(),
        None if grad_h is None else grad_h.data_ptr(), packed.values.data_ptr(),
        packed.exponents.data_ptr(), rstd.data_ptr(),
        None if weight is None else weight.data_ptr(), rows, features, stride, grad_h_stride,
        packed.values.shape[1], code if weight is None else _DTYPES[weight.dtype], code,
    )
    return grad_x, grad_weight


def linear_weight_grad(
    grad_out: torch.Tensor, packed: PackedActivation, dtype: Optional[torch.dtype] = None
) -> torch.Tensor:
    """grad_out^T . packed of [out_features, features]: a linear layer's weight gradient from its
    packed input.  Sums are held in fp32 and rounded once to ``dtype`` (grad_out's by default);
    fp16 gradients lose no bits, nor do fp32 ones above 2^-110 (what lies under 2^-133 is cut off)."""
    rows, out_features, stride = _matrix(grad_out, "linear_weight_grad: grad_out")
    code = _dtype_code(grad_out.dtype, "linear_weight_grad")
    dtype = grad_out.dtype if dtype is None else dtype
    out_code = _dtype_code(dtype, "linear_weight_grad")
    device = grad_out.device
    if stride > out_features and stride * grad_out.element_size() >= _WGRAD_ROW_BYTES:
        grad_out, stride = grad_out.contiguous(), out_features
    if rows != packed.rows:
        raise ValueError(f"linear_weight_grad: grad_out has {rows} rows, packed {packed.rows}")
    _require_same_device(packed.values, device, "linear_weight_grad: packed")
    scale = packed.column_scale
    features, pitch = packed.features, packed.values.shape[1]
    out = torch.empty(out_features, features, dtype=dtype, device=device)
    need = _native.lib().tft_linear_weight_grad_workspace(
        grad_out.data_ptr(), rows, out_features, features, stride, pitch, code
    )
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _launch(
        "tft_linear_weight_grad", device, out.data_ptr(),
        None if workspace is None else workspace.data_ptr(), need, grad_out.data_ptr(),
        packed.values.data_ptr(), packed.exponents.data_ptr(),
        None if scale is None else scale.data_ptr(), rows, out_features, features, stride, pitch,
        out_code, code if scale is None else _DTYPES[scale.dtype], code,
    )
    return out


def column_sum(x: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The sum of x's rows in fp32, rounded once to ``dtype`` (x's by default): a bias's gradient.
    Rows are added in a fixed order."""
    rows, columns, stride = _matrix(x, "column_sum")
    code = _dtype_code(x.dtype, "column_sum")
    dtype = x.dtype if dtype is None else dtype
    out = torch.empty(columns, dtype=dtype, device=x.device)
    need = _native.lib().tft_column_sum_workspace(rows, columns)
    workspace = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _launch(
        "tft_column_sum", x.device, out.data_ptr(), None if workspace is None else workspace.data_ptr(),
        need, x.data_ptr(), rows, columns, stride, _dtype_code(dtype, "column_sum"), code,
    )
    return out


# --- autograd -----------------------------------------------------------------------------


class _RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h, packed, rstd = rms_norm_forward(x, weight, eps, residual, pack=True)
        ctx.save_for_backward(packed.values, packed.exponents, rstd, weight)
        ctx.features, ctx.shape = packed.features, packed.shape
        ctx.mark_non_differentiable(packed.values, packed.exponents)
        ctx.set_materialize_grads(False)
        return y, (None if residual is None else h), packed.values, packed.exponents

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_h, _values, _exponents):
        need_x, need_residual, need_weight, _ = ctx.needs_input_grad
        if grad_y is None:
            return grad_h, grad_h if need_residual else None, None, None
        values, exponents, rstd, weight = ctx.saved_tensors
        packed = _trusted(values, exponents, ctx.features, weight, ctx.shape, grad_y.dtype)
        grad_x, grad_weight = rms_norm_backward(
            _as_rows(grad_y), packed, rstd, None if grad_h is None else _as_rows(grad_h),
            weight_grad=need_weight,
        )
        return grad_x if need_x else None, grad_x if need_residual else None, grad_weight, None


class NormOutput(NamedTuple):
    y: torch.Tensor
    h: torch.Tensor
    packed: Optional[PackedActivation]


def rms_norm(
    x: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    eps: Optional[float] = None,
    residual: Optional[torch.Tensor] = None,
) -> NormOutput:
    """Differentiable root-mean-square norm of h = x + residual: (y, h, packed).  ``packed`` is
    what the backward pass keeps, and what :func:`linear` takes for a layer that reads y; it is
    None where nothing needs a gradient, and nothing is packed then.  y and h have x's type; a weight
    of a third type takes part as its fp32 numbers, as in torch's norm.  ``packed``'s buffers belong to the
    current stream: a layer on another one needs ``packed.record_stream`` as it needs y's."""
    x = _as_rows(x)
    residual = None if residual is None else _as_rows(residual)
    if weight is not None and weight.dtype != x.dtype and weight.dtype in (torch.bfloat16, torch.float16):
        weight = weight.float()
    if not (torch.is_grad_enabled()
            and any(t is not None and t.requires_grad for t in (x, residual, weight))):
        y, h, _, _ = rms_norm_forward(x, weight, eps, residual, pack=False)
        return NormOutput(y, h, None)
    y, h, values, exponents = _RMSNormFunction.apply(x, residual, weight, eps)
    column_scale = None if weight is None else weight.detach()
    packed = _trusted(values, exponents, x.shape[-1], column_scale, tuple(x.shape), x.dtype)
    return NormOutput(y, x if residual is None else h, packed)


class _LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, values, exponents, column_scale):
        need_x, need_weight = ctx.needs_input_grad[:2]
        if need_weight and values is None:
            packed = pack(_as_rows(x))
            values, exponents = packed.values, packed.exponents
        ctx.save_for_backward(
            weight if need_x else None,
            values if need_weight else None,
            exponents if need_weight else None,
            column_scale if need_weight else None,
        )
        ctx.features, ctx.weight_dtype = x.shape[-1], weight.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        return F.linear(x, weight, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        weight, values, exponents, column_scale = ctx.saved_tensors
        need_x, need_weight, need_bias = ctx.needs_input_grad[:3]
        grad_x = grad_weight = grad_bias = None
        rows = _as_rows(grad_out)
        if need_x:
            grad_x = grad_out.matmul(weight)
        if need_weight:
            packed = _trusted(values, exponents, ctx.features, column_scale,
                              (values.shape[0], ctx.features), grad_out.dtype)
            grad_weight = linear_weight_grad(rows, packed, dtype=ctx.weight_dtype)
        if need_bias:
            grad_bias = column_sum(rows, dtype=ctx.bias_dtype)
        return grad_x, grad_weight, grad_bias, None, None, None


def linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    packed: Optional[PackedActivation] = None,
) -> torch.Tensor:
    """``torch.nn.functional.linear`` that keeps its input in 8 bits.  ``packed`` is x in that form
    where the caller has it (:func:`rms_norm`, or another layer's :func:`pack` of the same x);
    otherwise x is packed here, unless the weight needs no gradient."""
    return _linear(x, weight, bias, packed, share=False)


def _linear(
    x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], packed: Optional[PackedActivation],
    share: bool,
) -> torch.Tensor:
    given = x
    _require_gpu(x, "linear: x")
    if x.dim() == 0 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x of shape {tuple(x.shape)} does not fit a weight of {tuple(weight.shape)}")
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        # as torch: 64-bit tensors are left as they are (and refused below)
        x, weight, bias = (t if t is None or t.dtype == torch.float64 else t.to(dtype) for t in (x, weight, bias))
    _dtype_code(x.dtype, "linear")
    if packed is None and share and torch.is_grad_enabled():
        packed = _carried(given)
    if packed is not None:
        _require_same_device(packed.values, x.device, "linear: packed")
        if packed.shape != tuple(x.shape):
            raise ValueError(f"linear: packed is of shape {packed.shape}, x of {tuple(x.shape)}")
        if not packed._scale_is_as_packed():
            raise ValueError("linear: packed's column scale was written to since x was packed")
    if not (torch.is_grad_enabled()
            and any(t is not None and t.requires_grad for t in (x, weight, bias))):
        return F.linear(x, weight, bias)
    if packed is None and share and given.grad_fn is not None and weight.requires_grad:
        packed = _shared(given, x)
    return _LinearFunction.apply(
        x, weight, bias,
        None if packed is None else packed.values,
        None if packed is None else packed.exponents,
        None if packed is None else packed.column_scale,
    )


# --- modules ------------------------------------------------------------------------------

# A norm's output carries its packed form with it, so that the linear layers reading it share one
# copy.  An output that was written to since or given other storage, or whose norm's weight was
# written to, or a tensor made from it (all its rows in another shape apart), does not have it and is
# packed by the layer.  Nor is it used by a graph capture that the norm was not part of: the replays
# would read rows that nobody packs again.
_CARRIED = "_torchft_amd_packed"


class _Carried(NamedTuple):
    packed: PackedActivation
    version: int  # of the output, when it was made
    address: int
    capture: int  # the graph capture that it was made under
    stream: int

    def __reduce_ex__(self, protocol: object) -> tuple:  # a saved or copied output is not packed
        return OrderedDict, ()


_UNKNOWN_CAPTURE = (1 << 64) - 1


def _carry(y: torch.Tensor, packed: PackedActivation) -> None:
    stream = _raw_stream(y.device.index)
    capture = _native.lib().tft_capture_id(stream)
    setattr(y, _CARRIED, _Carried(packed, y._version, y.data_ptr(), capture, stream))


def _carried(x: torch.Tensor) -> Optional[PackedActivation]:
    """x's packed form, where x carries one and it is still x's, or where x is a view of all rows of
    a tensor that does."""
    c = getattr(x, _CARRIED, None)
    if c is None and x._is_view():
        c = getattr(x._base, _CARRIED, None)
    if type(c) is not _Carried or c.version != x._version or c.address != x.data_ptr():
        return None
    p = c.packed
    if x.shape[-1:] != p.shape[-1:] or x.numel() != math.prod(p.shape) or x.dtype != p.dtype \
            or not x.is_contiguous() or not p._scale_is_as_packed():
        return None
    stream = _raw_stream(x.device.index)
    capture = _native.lib().tft_capture_id(stream)
    if capture != c.capture or capture == _UNKNOWN_CAPTURE:
        return None
    if stream != c.stream:  # the caller has seen to x; nobody but us knows of what lies behind it
        p.record_stream(torch.cuda.current_stream(x.device))
    if p.shape != tuple(x.shape):
        p = _trusted(p.values, p.exponents, p.features, p.column_scale, tuple(x.shape), p.dtype)
    return p


# Several layers may read an activation that no norm of ours made.  The first of them packs it, and
# the others find its packed form by weak references on the activation: it lives as long as the
# backward pass of one of them needs it, and no longer because the activation does.  The same layers
# have to read it on the same stream: nothing makes another one wait for the packing.  Tensors that
# autograd did not make are packed by every layer: a program's input buffers are written to in ways
# that torch does not count (graph replays among them).
_SHARED = "_torchft_amd_shared"


class _Shared(NamedTuple):
    values: TensorWeakRef
    exponents: TensorWeakRef
    dtype: torch.dtype  # what was packed: the activation, or what autocast made of it
    version: int  # of the activation
    address: int
    strides: Tuple[int, ...]
    shape: Tuple[int, ...]
    capture: int
    stream: int

    def __reduce_ex__(self, protocol: object) -> tuple:  # a saved or copied activation is not packed
        return OrderedDict, ()


def _shared(given: torch.Tensor, x: torch.Tensor) -> Optional[PackedActivation]:
    """x, which is ``given`` itself or its cast, packed once for all layers that read ``given``."""
    stream = _raw_stream(given.device.index)
    capture = _native.lib().tft_capture_id(stream)
    if capture == _UNKNOWN_CAPTURE:
        return None
    now = (x.dtype, given._version, given.data_ptr(), given.stride(), tuple(given.shape), capture, stream)
    s = getattr(given, _SHARED, None)
    if type(s) is _Shared and s[2:] == now:
        values, exponents = s.values(), s.exponents()
        if values is not None and exponents is not None:
            return _trusted(values, exponents, x.shape[-1], None, tuple(x.shape), x.dtype)
    packed = pack(_as_rows(x))
    setattr(given, _SHARED, _Shared(TensorWeakRef(packed.values), TensorWeakRef(packed.exponents), *now))
    return packed


class RMSNorm(nn.RMSNorm):
    """``torch.nn.RMSNorm`` over the last dimension that keeps its normalised rows in 8 bits.
    ``forward(x, residual)`` norms h = x + residual and returns (y, h).  The output has x's type."""

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        if len(self.normalized_shape) != 1 or x.shape[-1:] != tuple(self.normalized_shape):
            raise ValueError(f"RMSNorm over {tuple(self.normalized_shape)} does not fit {tuple(x.shape)}")
        out = rms_norm(x, self.weight, self.eps, residual)
        if out.packed is not None:
            _carry(out.y, out.packed)
        return out.y if residual is None else (out.y, out.h)


class Linear(nn.Linear):
    """``torch.nn.Linear`` that keeps its input in 8 bits for the weight gradient, once for all such
    layers that read it."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return _linear(x, self.weight, self.bias, None, share=True)


def pack_activations(module: nn.Module) -> nn.Module:
    """Makes every ``nn.Linear`` and ``nn.RMSNorm`` of ``module`` (itself included) keep its
    activations in 8 bits, in place, and returns ``module``.  Parameters, names and state dicts
    stay as they are.  Subclasses, and norms over several dimensions or more than 16384 features,
    are left alone."""
    for m in module.modules():
        if type(m) is nn.Linear:
            m.__class__ = Linear
        elif (type(m) is nn.RMSNorm and len(m.normalized_shape) == 1
              and m.normalized_shape[0] <= MAX_NORM_FEATURES):
            m.__class__ = RMSNorm
    return module

"""Block-scaled ("MX") 8- and 4-bit tensors and the product over them (``csrc/kernels/mx_quant.hip``, ``mx_linear.hip``).

32 consecutive values of the last axis share a power-of-two scale (one byte, ``2^(code - 127)``), the smallest that needs
no clipping; an element is the value over the scale, rounded to nearest even. ``e2m1`` holds 4 bits (0, 0.5, 1, 1.5, 2, 3,
4, 6 and their negatives; two in a byte, the even element in the low half), ``e4m3`` 8 bits (up to 448). A block that
holds a NaN or an infinity gets the scale's NaN (code 255) and stands for 32 NaN.

``mx_quantize`` lays weights out once and activations on every call; ``norm.rms_norm_mx8`` writes e4m3 activations straight
from a norm; ``mx_linear`` multiplies them with e2m1 weights on gfx950's block-scaled matrix instructions. The PyTorch
path (CPU) is the reference. No backward pass: inputs that require a gradient are refused.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
import torch.nn.functional as F

from . import _ext

BLOCK, ALIGN = 32, 128
MAX_WIDTH = 1 << 30  # values of a row, here and where a row of logits or of a norm is taken
DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # element types at the C entries (csrc/kernels/mx.h)
FMT_CODE = {"e4m3": 0, "e2m1": 1}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


class MxTensor(NamedTuple):
    """``k`` values per row in blocks of 32. A row is stored up to a multiple of 128 values, ``kp``; what lies behind ``k``
    is zero. Contiguous; may be built from a checkpoint's codes of this layout."""

    data: torch.Tensor   # float8_e4m3fn [..., kp], or uint8 [..., kp / 2] (e2m1)
    scale: torch.Tensor  # float8_e8m0fnu (or its bytes as uint8) [..., kp / 32]
    k: int

    @property
    def fmt(self) -> str:
        return "e2m1" if self.data.dtype == torch.uint8 else "e4m3"

    @property
    def shape(self) -> Tuple[int, ...]:
        return (*self.data.shape[:-1], self.k)

    @property
    def device(self) -> torch.device:
        return self.data.device

    def to(self, device) -> "MxTensor":
        return MxTensor(self.data.to(device), self.scale.to(device), self.k)


def padded(k: int) -> int:
    """Stored values of a row of ``k``."""
    return -(-k // ALIGN) * ALIGN


def new(shape, dtype: torch.dtype, device) -> torch.Tensor:
    """An uninitialised contiguous tensor (of few axes by its strides, 0.5 us less than ``torch.empty`` takes)."""
    if len(shape) == 2:
        return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=device)
    if len(shape) == 1:
        return torch.empty_strided(shape, (1,), dtype=dtype, device=device)
    return torch.empty(shape, dtype=dtype, device=device)


def empty(lead, k: int, fmt: str, device) -> MxTensor:
    """An uninitialised MxTensor of ``(*lead, k)``."""
    kp = padded(k)
    data = new((*lead, kp), torch.float8_e4m3fn, device) if fmt == "e4m3" else new((*lead, kp // 2), torch.uint8, device)
    return MxTensor(data, new((*lead, kp // BLOCK), torch.float8_e8m0fnu, device), k)


def check(name: str, q: MxTensor) -> None:
    """Raises TypeError or ValueError unless ``q`` has the layout that MxTensor describes."""
    if not isinstance(q, MxTensor):
        raise TypeError(f"{name}: an MxTensor is expected, not {type(q).__name__}")
    data, scale, k = q
    e2m1 = data.dtype == torch.uint8
    if not (e2m1 or data.dtype == torch.float8_e4m3fn) or scale.dtype not in (torch.uint8, torch.float8_e8m0fnu):
        raise ValueError(f"{name}: data is uint8 (e2m1) or float8_e4m3fn, scale float8_e8m0fnu or uint8")
    kp, shape, scales = padded(k), data.shape, scale.shape
    if (not 0 < k <= MAX_WIDTH or len(shape) < 1 or len(scales) < 1 or scales[-1] * BLOCK != kp or shape[-1] != (kp // 2 if e2m1 else kp)
            or shape[:-1] != scales[:-1]):
        raise ValueError(f"{name}: data {tuple(shape)} and scale {tuple(scales)} do not hold rows of {k}")
    if data.get_device() != scale.get_device() or not data.is_contiguous() or not scale.is_contiguous():
        raise ValueError(f"{name}: data and scale have to be contiguous and on one device")
    if data.data_ptr() % 16 or scale.data_ptr() % 4:
        raise ValueError(f"{name}: data has to be 16-byte aligned, scale 4-byte aligned")


def rows_2d(t: torch.Tensor) -> torch.Tensor:
    """``[..., K]`` as ``[rows, K]`` with unit stride along K; a copy only where no view has that."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    pitch, step = t.stride()
    return t if step == 1 and (pitch >= t.shape[1] or t.shape[0] <= 1) else t.contiguous()


def quantize_reference(x: torch.Tensor, fmt: str) -> MxTensor:
    """fp32 ``[..., K]`` -> MxTensor in plain PyTorch."""
    k = x.shape[-1]
    x = F.pad(x.float(), (0, padded(k) - k))
    b = x.reshape(*x.shape[:-1], padded(k) // BLOCK, BLOCK)
    bits = b.abs().amax(-1).view(torch.int32)
    e, m = bits >> 23, bits & 0x7FFFFF
    code = (e - 8 + (m > 0x600000).int()) if fmt == "e4m3" else (e - 2 + (m > 0x400000).int())
    code = torch.where(torch.isfinite(b).all(-1), code.clamp_min(0), torch.full_like(code, 255))
    inv = ((254 - code.clamp_max(253)) << 23).view(torch.float32)
    v = torch.where(code[..., None] == 255, torch.zeros_like(b), b * inv[..., None]).reshape(x.shape)
    scale = code.to(torch.uint8).view(torch.float8_e8m0fnu)
    if fmt == "e4m3":
        return MxTensor(v.to(torch.float8_e4m3fn), scale, k)
    a = v.abs()
    q = sum((a >= t if even else a > t).to(torch.uint8)
            for t, even in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)))
    q = q + 8 * torch.signbit(v).to(torch.uint8)
    return MxTensor((q[..., 0::2] + 16 * q[..., 1::2]).contiguous(), scale, k)


def dequantize_reference(q: MxTensor) -> torch.Tensor:
    """The fp32 values that codes stand for, in plain PyTorch."""
    if q.fmt == "e2m1":
        table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=q.device)
        v = torch.stack((table[(q.data & 15).long()], table[(q.data >> 4).long()]), -1).flatten(-2)
    else:
        v = q.data.float()
    code = q.scale.view(torch.uint8)
    s = torch.where(code == 255, torch.full_like(code, 0, dtype=torch.float32).fill_(float("nan")),
                    q.scale.view(torch.float8_e8m0fnu).float())
    return (v.reshape(*code.shape, BLOCK) * s[..., None]).reshape(v.shape)[..., :q.k]


# scale bytes of a launch of quantisation, which has fewer than 2^32 threads, of 16 values each
MAX_SCALES = (1 << 31) - 128


def mx_quantize(x: torch.Tensor, fmt: str = "e2m1") -> MxTensor:
    """``[..., K]`` (bf16, fp16 or fp32; rows may be strided) -> MxTensor of ``fmt`` ("e2m1" or "e4m3")."""
    if fmt not in FMT_CODE:
        raise ValueError(f"mx_quantize: fmt is 'e2m1' or 'e4m3', not {fmt!r}")
    if x.dtype not in DTYPE_CODE or x.dim() < 1 or not 0 < x.shape[-1] <= MAX_WIDTH:
        raise ValueError("mx_quantize expects bfloat16, float16 or float32 with a last axis of 1 to 2^30 values")
    _ext.refuse_grad("mx_quantize", x)
    # rows of one value, stored as 128, reach the limit first
    if x.numel() >= 1 << 28 and x.numel() // x.shape[-1] * (padded(x.shape[-1]) // BLOCK) > MAX_SCALES:
        raise ValueError(f"mx_quantize: {tuple(x.shape)} are over 2^36 stored values")
    if _ext.backend_for(x) != "hip":
        return quantize_reference(x, fmt)
    k = x.shape[-1]
    q = empty(x.shape[:-1], k, fmt, x.device)
    x = rows_2d(x)
    _ext.call_on(x.get_device(), "ai4e_mx_quantize", x.data_ptr(), max(x.stride(0), k), x.shape[0], k, DTYPE_CODE[x.dtype],
                 FMT_CODE[fmt], q.data.data_ptr(), q.scale.data_ptr())
    return q


def mx_dequantize(q: MxTensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that ``q`` stands for, ``[..., k]`` in ``dtype`` (one rounding; exact in float32)."""
    check("mx_dequantize", q)
    if dtype not in DTYPE_CODE:
        raise ValueError("mx_dequantize gives bfloat16, float16 or float32")
    _ext.refuse_grad("mx_dequantize", q.data, q.scale)
    if q.scale.numel() > MAX_SCALES:
        raise ValueError(f"mx_dequantize: {tuple(q.shape)} are over 2^36 stored values")
    if _ext.backend_for(q.data) != "hip":
        return dequantize_reference(q).to(dtype)
    y = new(q.shape, dtype, q.data.device)
    if y.numel():
        _ext.call_on(y.get_device(), "ai4e_mx_dequantize", q.data.data_ptr(), q.scale.data_ptr(), y.numel() // q.k, q.k,
                     DTYPE_CODE[dtype], FMT_CODE[q.fmt], y.data_ptr())
    return y


def _linear_fits(m: int, n: int, kp: int) -> bool:
    """Whether a launch holds ``m`` rows of ``kp`` stored values by ``n`` outputs (``fits`` in csrc/kernels/mx_linear.hip)."""
    rows, cols = -(-m // 128), -(-n // 128)
    slices = kp < 512 and (m <= 32 or n < 4)
    return kp <= 1 << 23 and rows * cols <= 1 << 22 and not (slices and -(-m // 32) * -(-n // 64) >= 1 << 23)


def mx_linear(x: MxTensor, w: MxTensor, bias: Optional[torch.Tensor] = None,
              out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x @ w.T + bias``: ``x`` [..., K] e4m3 or e2m1, ``w`` [N, K] e2m1, ``bias`` [N] -> [..., N].

    The accumulators are 32 bits wide. Between 4-bit operands the products and their sums inside an instruction are
    exact; with e4m3 the matrix unit adds the products of one instruction to about 17 bits (measured, relative 5e-6 for
    normally distributed values), far below a 16-bit result but not a 32-bit one: float32 results are given for e2m1
    only."""
    check("mx_linear: x", x)
    check("mx_linear: w", w)
    data, scale, k = x
    fmt = x.fmt
    if w.fmt != "e2m1" or w.data.dim() != 2:
        raise ValueError("mx_linear: w is an e2m1 MxTensor [N, K]")
    if k != w.k:
        raise ValueError(f"mx_linear: x has rows of {k}, w of {w.k}")
    if out_dtype not in DTYPE_CODE:
        raise ValueError("mx_linear gives bfloat16, float16 or float32")
    if out_dtype == torch.float32 and fmt != "e2m1":
        raise ValueError("mx_linear: float32 results need e2m1 activations (8-bit products are added to about 17 bits)")
    n = w.data.shape[0]
    if bias is not None and (tuple(bias.shape) != (n,) or not bias.is_floating_point()):
        raise ValueError(f"mx_linear: bias is a floating tensor of {n} values")
    m = scale.numel() // scale.shape[-1]
    if (m > 1 << 15 or n > 1 << 18 or k > 1 << 23) and not _linear_fits(m, n, padded(k)):  # smaller ones do
        raise ValueError(f"mx_linear: {m} rows of {k} by {n} outputs are more than a launch holds (k up to 2^23, 2^22 tiles of "
                         "128 rows by 128 outputs)")
    index = data.get_device()
    if w.data.get_device() != index or (bias is not None and bias.get_device() != index):
        raise ValueError("mx_linear: x, w and bias have to be on one device")
    _ext.refuse_grad("mx_linear", data, scale, w.scale, bias)
    if _ext.backend_for(data) != "hip":
        y = dequantize_reference(x) @ dequantize_reference(w).T
        return (y if bias is None else y + bias.float()).to(out_dtype)
    y = new((*data.shape[:-1], n), out_dtype, data.device)
    if y.numel():
        b32 = None if bias is None else bias.to(torch.float32).contiguous()
        _ext.call_on(index, "ai4e_mx_linear", data.data_ptr(), scale.data_ptr(), FMT_CODE[fmt], w.data.data_ptr(),
                     w.scale.data_ptr(), _ext.ptr(b32), m, n, padded(k), y.data_ptr(), DTYPE_CODE[out_dtype])
    return y

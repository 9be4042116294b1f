"""Microscaled 4-bit floating point: formats, quantisation, products and the linear layer on them.

Beside the group-64 INT4 layer (16-bit activations, integer weights) this module offers the formats
that the block-scaled tensor cores of sm_100a multiply directly, both operands in FP4:

* ``"mxfp4"`` -- blocks of 32 columns, scale ``2^e`` (E8M0 byte ``e + 127``) with
  ``e = max(floor(log2(amax)) - 2, -127)``;
* ``"nvfp4"`` -- blocks of 16 columns, scale ``s`` (E4M3), the nearest to ``amax / (6 g)`` and at most
  448, with one FP32 factor ``g`` per tensor (``tensor_scale``; 1 when omitted, otherwise between
  2^-64 and 2^64).

A code is the E2M1 number (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign) nearest to ``x / step``, ``step``
being ``2^e`` or ``s g`` rounded to FP32; ties go to the even code and magnitudes above 6 become 6.  A
block that holds a NaN or an infinity (every block, if ``g`` is outside its range) gets the NaN scale
and zero codes, so that it reads back as NaN.

Storage: ``codes`` uint8 ``[R, 16 ceil(K / 32)]``, two codes to a byte, low nibble first, zero past
column K; ``scales`` uint8 ``[ceil(R / 128), ceil(blocks / 4), 32, 4, 4]``: the byte of row ``r`` and
block ``j`` lies at ``[r // 128, j // 4, r % 32, r % 128 // 32, j % 4]``, the order in which the tensor
cores take it, and bytes without a row or block are zero (``blocks`` counts the padded columns).  The tensor cores
read an E4M3 scale without its sign, so bit 7 of an nvfp4 scale is clear.
``tile_scales`` and ``untile_scales`` convert from and to plain ``[R, blocks]`` rows, as checkpoints
store them.

CUDA tensors run the library's kernels (``ImportError`` when it is not built), CPU tensors the torch
arithmetic below, which gives the same codes and scales bit for bit.  Everything here is for
inference: no gradients are recorded.
"""
import torch

from . import _ops
from .quantization import _row_chunks, _validate_matrix

# format -> (code of the C ABI, columns per block)
FORMATS = {"mxfp4": (0, 32), "nvfp4": (1, 16)}
_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_FLOAT_TYPES = (torch.float16, torch.bfloat16, torch.float32)
_HALF_TYPES = (torch.float16, torch.bfloat16)


def _validate_format(format):
    if not isinstance(format, str) or format not in FORMATS:
        raise ValueError(f"format must be one of {', '.join(FORMATS)}")
    return FORMATS[format]


def _validate_factor(factor, name, format, device):
    if factor is None:
        return
    if format != "nvfp4":
        raise ValueError(f"{name} belongs to nvfp4 only")
    if not isinstance(factor, torch.Tensor):
        raise TypeError(f"{name} must be a Tensor")
    if factor.dtype != torch.float32:
        raise TypeError(f"{name} has unsupported dtype {factor.dtype}")
    if factor.numel() != 1:
        raise ValueError(f"{name} must hold one value")
    if factor.device != device:
        raise ValueError("All tensors must be on the same device")


def code_columns(in_features):
    """Bytes of a row of codes."""
    return (in_features + 31) // 32 * 16


def scale_shape(rows, in_features, format="mxfp4"):
    """Shape of the tiled scales of a ``[rows, in_features]`` operand."""
    _, block = _validate_format(format)
    blocks = code_columns(in_features) * 2 // block
    return ((rows + 127) // 128, (blocks + 3) // 4, 32, 4, 4)


def tile_scales(scales):
    """Scale bytes ``[R, blocks]`` -> tiles ``[ceil(R / 128), ceil(blocks / 4), 32, 4, 4]``."""
    _validate_matrix(scales, "scales", (torch.uint8,))
    rows, blocks = scales.shape
    padded = torch.nn.functional.pad(scales, (0, -blocks % 4, 0, -rows % 128))
    tiles = padded.reshape((rows + 127) // 128, 4, 32, (blocks + 3) // 4, 4)
    return tiles.permute(0, 3, 2, 1, 4).contiguous()


def untile_scales(tiles, rows, blocks):
    """The inverse of ``tile_scales``."""
    if not isinstance(tiles, torch.Tensor):
        raise TypeError("tiles must be a Tensor")
    if tiles.dtype != torch.uint8:
        raise TypeError(f"tiles has unsupported dtype {tiles.dtype}")
    if tuple(tiles.shape) != ((rows + 127) // 128, (blocks + 3) // 4, 32, 4, 4) or rows <= 0 or blocks <= 0:
        raise ValueError("Invalid scales shape")
    flat = tiles.permute(0, 3, 2, 1, 4).reshape(tiles.shape[0] * 128, tiles.shape[1] * 4)
    return flat[:rows, :blocks].contiguous()


def _validate_operand(codes, scales, format, in_features, name=""):
    """Codes and tiled scales of one operand; returns its row count."""
    _validate_matrix(codes, f"{name}codes", (torch.uint8,))
    if isinstance(in_features, bool) or not isinstance(in_features, int) or in_features <= 0:
        raise ValueError("in_features must be a positive integer")
    rows, width = codes.shape
    if width != code_columns(in_features):
        raise ValueError(f"Invalid {name}codes shape")
    if not isinstance(scales, torch.Tensor):
        raise TypeError(f"{name}scales must be a Tensor")
    if scales.dtype != torch.uint8:
        raise TypeError(f"{name}scales has unsupported dtype {scales.dtype}")
    if tuple(scales.shape) != scale_shape(rows, in_features, format):
        raise ValueError(f"Invalid {name}scales shape")
    if scales.device != codes.device:
        raise ValueError("All tensors must be on the same device")
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError(f"{name}codes and {name}scales must be contiguous")
    return rows


# ---- CPU arithmetic ------------------------------------------------------------------------------


def _quantize_rows(x, format, factor):
    """(codes [R, bytes], scale bytes [R, blocks]).  Quotients are taken in 64 bits, where a value that
    is not on the border between two codes cannot be rounded onto it."""
    rows, k = x.shape
    _, block = FORMATS[format]
    values = torch.nn.functional.pad(x.float(), (0, -k % 32)).reshape(rows, -1, block)
    amax = values.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    amax = torch.where(bad, 0.0, amax)
    if format == "mxfp4":
        exponent = torch.frexp(amax)[1] - 3  # floor(log2(amax)) - 2
        byte = torch.where(amax > 0, exponent.clamp(min=-127), -127) + 127
        step = torch.ldexp(torch.ones_like(amax, dtype=torch.float64), byte - 127)
        byte = torch.where(bad, 255, byte).to(torch.uint8)
    else:
        g = torch.ones(1) if factor is None else factor.detach().reshape(1).float()
        if not bool((g >= 2.0**-64) & (g <= 2.0**64)):
            bad, g = torch.ones_like(bad), torch.ones(1)
        quotient = (amax.double() / (6.0 * g).double()).clamp(max=448.0)
        unit = torch.ldexp(torch.ones_like(quotient), (torch.frexp(quotient)[1] - 1).clamp(min=-6) - 3)
        scale = (torch.round(quotient / unit) * unit).float()
        byte = torch.where(bad, 127, scale.to(torch.float8_e4m3fn).view(torch.uint8))
        step = (scale * g).double()
    usable = (step > 0)[..., None]
    size = torch.where(usable, values.double() / torch.where(step > 0, step, 1.0)[..., None], 0.0).abs()
    grid = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = (torch.round(size / grid) * grid).clamp(max=6.0)
    code = torch.where(size < 2, size * 2, torch.where(size < 4, size + 2, size / 2 + 4)).to(torch.uint8)
    code |= torch.signbit(values).to(torch.uint8) << 3
    code = torch.where(bad[..., None], 0, code).reshape(rows, -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte


def _operand_values(codes, scales, format, factor):
    """FP32 ``[R, padded K]`` that codes and tiled scales stand for."""
    _, block = FORMATS[format]
    rows, blocks = codes.shape[0], codes.shape[1] * 2 // block
    byte = untile_scales(scales, rows, blocks)
    if format == "mxfp4":
        step = torch.ldexp(torch.ones(byte.shape), byte.to(torch.int32) - 127)
        step = torch.where(byte == 255, float("nan"), step)
    else:
        step = byte.view(torch.float8_e4m3fn).float()
        if factor is not None:
            step = step * factor.detach().reshape(1)
    table = torch.tensor(_MAGNITUDES)
    table = torch.cat((table, -table))
    code = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(rows, blocks, block)
    return (table[code.long()] * step[..., None]).reshape(rows, -1)


# ---- operators -----------------------------------------------------------------------------------
#
# At decode sizes the checks of a call cost more host time than its kernel runs.  The torch binding looks at the
# same things without the interpreter and answers None to whatever is not a plain call on CUDA tensors; the
# checks here then say what is wrong, or the call goes its other way.


def quantize_fp4(x, format="mxfp4", tensor_scale=None):
    """Quantise ``x`` ``[R, K]`` (FP16, BF16 or FP32): ``(codes, scales)`` in the layout above.

    ``tensor_scale`` is the FP32 factor ``g`` of nvfp4, one value on ``x``'s device."""
    if _ops.binding is not None:
        result = _ops.binding.quantize(x, format, tensor_scale)
        if result is not None:
            return result
    _validate_matrix(x, "x", _FLOAT_TYPES)
    _validate_format(format)
    _validate_factor(tensor_scale, "tensor_scale", format, x.device)
    if x.is_cuda:
        return _ops.fp4_quantize(x, format, tensor_scale)
    rows, k = x.shape
    _, block = FORMATS[format]
    codes = torch.empty((rows, code_columns(k)), dtype=torch.uint8)
    scales = torch.empty((rows, code_columns(k) * 2 // block), dtype=torch.uint8)
    for r0, r1 in _row_chunks(rows, k):
        codes[r0:r1], scales[r0:r1] = _quantize_rows(x.detach()[r0:r1], format, tensor_scale)
    return codes, tile_scales(scales)


def dequantize_fp4(codes, scales, in_features=None, format="mxfp4", tensor_scale=None, dtype=torch.float16):
    """``code * step`` as ``[R, in_features]``, computed in FP32 and rounded once to ``dtype`` (FP16,
    BF16 or FP32).  ``in_features`` defaults to the padded column count."""
    if _ops.binding is not None:
        result = _ops.binding.dequantize(codes, scales, in_features, format, tensor_scale, dtype)
        if result is not None:
            return result
    _validate_format(format)
    if dtype not in _FLOAT_TYPES:
        raise TypeError("dtype must be FP16, BF16 or FP32")
    _validate_matrix(codes, "codes", (torch.uint8,))
    k = codes.shape[1] * 2 if in_features is None else in_features
    _validate_operand(codes, scales, format, k)
    _validate_factor(tensor_scale, "tensor_scale", format, codes.device)
    if codes.is_cuda:
        return _ops.fp4_dequantize(codes, scales, k, format, tensor_scale, dtype)
    return _operand_values(codes, scales, format, tensor_scale)[:, :k].to(dtype).contiguous()


def matmul_fp4(a_codes, a_scales, b_codes, b_scales, format="mxfp4", a_scale=None, b_scale=None,
               dtype=torch.float16):
    """``a . b^T`` of two quantised operands ``[Ra, K]`` and ``[Rb, K]``: ``[Ra, Rb]`` in ``dtype`` (FP16
    or BF16), FP32 sums, one rounding.  ``a_scale`` and ``b_scale`` are the operands' nvfp4 factors.
    What the codes past column K hold is multiplied too: they are zero as ``quantize_fp4`` writes them."""
    if _ops.binding is not None:
        result = _ops.binding.matmul(a_codes, a_scales, b_codes, b_scales, format, a_scale, b_scale, dtype, _ops._flags)
        if result is not None:
            return result
    _validate_format(format)
    if dtype not in _HALF_TYPES:
        raise TypeError("dtype must be FP16 or BF16")
    _validate_matrix(a_codes, "a_codes", (torch.uint8,))
    k = a_codes.shape[1] * 2
    _validate_operand(a_codes, a_scales, format, k, "a_")
    _validate_matrix(b_codes, "b_codes", (torch.uint8,))
    if b_codes.shape[1] != a_codes.shape[1]:
        raise ValueError("a_codes and b_codes have incompatible K")
    _validate_operand(b_codes, b_scales, format, k, "b_")
    if a_codes.device != b_codes.device:
        raise ValueError("All tensors must be on the same device")
    _validate_factor(a_scale, "a_scale", format, a_codes.device)
    _validate_factor(b_scale, "b_scale", format, a_codes.device)
    if a_codes.is_cuda:
        return _ops.fp4_matmul(a_codes, a_scales, b_codes, b_scales, format, a_scale, b_scale, dtype)
    y = _operand_values(a_codes, a_scales, format, None) @ _operand_values(b_codes, b_scales, format, None).T
    for factor in (a_scale, b_scale):
        if factor is not None:
            y = y * factor.detach().reshape(1)
    return y.to(dtype)


def linear_fp4(x, codes, scales, format="mxfp4", tensor_scale=None, input_scale=None):
    """``x`` ``[M, K]`` (FP16 or BF16) quantised in ``format`` with factor ``input_scale``, times the quantised
    weight ``codes`` / ``scales`` / ``tensor_scale`` ``[N, K]``: ``[M, N]`` in ``x``'s type.

    ``matmul_fp4(*quantize_fp4(x, format, input_scale), codes, scales, ...)`` in one call."""
    if _ops.binding is not None:
        result = _ops.binding.linear(x, codes, scales, format, tensor_scale, input_scale, _ops._flags)
        if result is not None:
            return result
    _validate_format(format)
    _validate_matrix(x, "x", _HALF_TYPES)
    _validate_matrix(codes, "codes", (torch.uint8,))
    k = x.shape[1]
    if codes.shape[1] != code_columns(k):
        raise ValueError("x and codes have incompatible K")
    _validate_operand(codes, scales, format, k)
    if x.device != codes.device:
        raise ValueError("All tensors must be on the same device")
    _validate_factor(tensor_scale, "tensor_scale", format, x.device)
    _validate_factor(input_scale, "input_scale", format, x.device)
    if x.is_cuda:
        return _ops.fp4_linear(x, codes, scales, format, tensor_scale, input_scale)
    x_codes, x_scales = quantize_fp4(x, format, input_scale)
    return matmul_fp4(x_codes, x_scales, codes, scales, format, input_scale, tensor_scale, x.dtype)


class MicroscaledLinear(torch.nn.Module):
    """Inference-only linear layer with microscaled FP4 weights and activations.

    Beside ``QuantizedLinear``: its activations are quantised on the way in, so the product runs at the
    FP4 rate of the tensor cores.  Buffers: ``codes``, ``scales`` and, for nvfp4, the FP32 factors
    ``tensor_scale`` (weights) and ``input_scale`` (activations; a calibrated
    ``amax / (6 * 448)``, or None for 1)."""

    def __init__(self, codes, scales, tensor_scale=None, input_scale=None, *, in_features, format="mxfp4"):
        super().__init__()
        _validate_format(format)
        self.out_features = _validate_operand(codes, scales, format, in_features)
        _validate_factor(tensor_scale, "tensor_scale", format, codes.device)
        _validate_factor(input_scale, "input_scale", format, codes.device)
        self.in_features = in_features
        self.format = format
        self.register_buffer("codes", codes)
        self.register_buffer("scales", scales)
        self.register_buffer("tensor_scale", tensor_scale)
        self.register_buffer("input_scale", input_scale)

    @classmethod
    def from_float(cls, weight, format="mxfp4", input_scale=None):
        """Quantise ``weight`` ``[N, K]``; the nvfp4 factor is ``amax / (6 * 448)``, the least that keeps
        every block scale within E4M3."""
        _validate_matrix(weight, "weight", _FLOAT_TYPES)
        _validate_format(format)
        with torch.no_grad():
            factor = None
            if format == "nvfp4":
                factor = (weight.detach().abs().amax().float() / (6.0 * 448.0)).reshape(1)
                factor = torch.where(factor > 0, factor.clamp(2.0**-64, 2.0**64), torch.ones_like(factor))
            codes, scales = quantize_fp4(weight, format, factor)
        return cls(codes, scales, factor, input_scale, in_features=weight.shape[1], format=format)

    def forward(self, x):
        if isinstance(x, torch.Tensor) and x.ndim == 2 and x.shape[1] != self.in_features:
            raise ValueError("x and codes have incompatible K")
        return linear_fp4(x, self.codes, self.scales, self.format, self.tensor_scale, self.input_scale)

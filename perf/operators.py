"""Cases of the microscaled FP4 operators: quantisation, its inverse, the product of two quantised
operands, and the linear layer that quantises its own activations.

Two storage formats, both with E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives):

  mxfp4   blocks of 32 columns, scale 2^e (E8M0): e = floor(log2(largest magnitude)) - 2, at
          least -127
  nvfp4   blocks of 16 columns, scale s (E4M3): the nearest to (largest magnitude) / (6 g), at
          most 448, with one FP32 factor g for the whole tensor

and code = the nearest E2M1 value to x / scale (x / (s g) in nvfp4, s g rounded to FP32), ties to
the even code, magnitudes above 6 becoming 6.  Codes lie two to a byte, low nibble first, rows
padded with zeros to a multiple of 32 columns.  Scales lie in tiles of 128 rows by 4 blocks: the
byte of row r and block j is at [r // 128, j // 4, r % 32, r % 128 // 32, j % 4].
"""
import math

import torch

own = False

BLOCK = {"mxfp4": 32, "nvfp4": 16}
DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# Of one operand's work: one pass over the widest benchmark weight; of one product: its prompt pass.
MOST_ELEMENTS = 24576 * 4096
MOST_PRODUCT = 8192 * 24576 * 4096


def listed():
    return [
        # One token's activations on their way into a projection: nothing but latency.
        {"name": "round_token", "op": "round", "rows": 1, "cols": 4096, "format": "mxfp4", "dtype": "bf16"},
        # A prompt's activations in front of the down projection.
        {"name": "round_prompt", "op": "round", "rows": 2048, "cols": 12288, "format": "nvfp4", "dtype": "bf16"},
        # A gate/up weight in full precision being converted, and checked by its inverse.
        {"name": "round_weight", "op": "round", "rows": 24576, "cols": 4096, "format": "mxfp4", "dtype": "fp32"},
        # A ragged activation: odd rows, columns that fill neither a block nor a vector load.
        {"name": "round_ragged", "op": "round", "rows": 333, "cols": 1003, "format": "nvfp4", "dtype": "fp16"},
        # A stored weight expanded for a consumer that wants it dense.
        {"name": "expand_weight", "op": "expand", "rows": 24576, "cols": 4096, "format": "mxfp4", "dtype": "bf16"},
        # A small odd adapter expanded in full precision.
        {"name": "expand_ragged", "op": "expand", "rows": 515, "cols": 1234, "format": "nvfp4", "dtype": "fp32"},
        # Activations quantised once for several projections: the product alone, an ordinary batch.
        {"name": "product_batch", "op": "product", "rows": 256, "n": 6144, "cols": 4096, "format": "nvfp4", "dtype": "bf16"},
        # The same for a long prompt: the largest work there is.
        {"name": "product_prompt", "op": "product", "rows": 8192, "n": 24576, "cols": 4096, "format": "mxfp4", "dtype": "bf16"},
        # Decode of one sequence through the attention output projection.
        {"name": "linear_token", "op": "linear", "rows": 1, "n": 4096, "cols": 4096, "format": "mxfp4", "dtype": "bf16"},
        # Decode of sixteen sequences through gate/up.
        {"name": "linear_decode", "op": "linear", "rows": 16, "n": 24576, "cols": 4096, "format": "nvfp4", "dtype": "fp16"},
        # A ragged batch through a layer with odd sizes.
        {"name": "linear_ragged", "op": "linear", "rows": 77, "n": 5001, "cols": 1000, "format": "mxfp4", "dtype": "fp16"},
        # A prompt through the down projection.
        {"name": "linear_prompt", "op": "linear", "rows": 2048, "n": 4096, "cols": 12288, "format": "nvfp4", "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """Even over the logarithm; a third of the results are rounded to a multiple of 64."""
    value = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if value >= 64 and rng.random() < 0.33:
        value -= value % 64
    return max(low, min(high, value))


def draw(rng):
    op = rng.choice(["round", "expand", "product", "product", "linear", "linear"])
    case = {"op": op, "format": rng.choice(["mxfp4", "nvfp4"])}
    if op in ("round", "expand"):
        case["cols"] = _spread(rng, 16, 12288)
        case["rows"] = _spread(rng, 1, min(24576, MOST_ELEMENTS // case["cols"]))
        case["dtype"] = rng.choice(["fp16", "bf16", "fp32"])
    else:
        case["cols"] = _spread(rng, 64, 12288)
        case["n"] = _spread(rng, 64, min(24576, MOST_ELEMENTS // case["cols"]))
        case["rows"] = _spread(rng, 1, min(8192, MOST_PRODUCT // (case["n"] * case["cols"])))
        case["dtype"] = rng.choice(["fp16", "bf16"])
    return case


# ---- inputs ------------------------------------------------------------------------------------


def _activations(generator, rows, cols, dtype):
    """Normal values, one column in 128 as a wide outlier channel, one row in 32 padding."""
    x = torch.randn(rows, cols, generator=generator, device="cuda")
    x[:, 5::128] *= 20.0
    x[31::32] = 0.0
    return x.to(dtype)


def _stored(generator, rows, cols, fmt, std, scale):
    """A quantised operand as a program has it in hand: codes, tiled scales, FP32 factor."""
    values = torch.randn(rows, cols, generator=generator, device="cuda") * std
    factor = torch.full((1,), scale, device="cuda") if fmt == "nvfp4" else None
    magnitude, sign, scales = _quantize(values, fmt, factor)
    return {"codes": _pack(magnitude, sign), "scales": _tile(scales, fmt), "factor": factor}


def prepare(case, seed):
    generator = torch.Generator("cuda").manual_seed(seed)
    fmt, rows, cols = case["format"], case["rows"], case["cols"]
    state = {"case": dict(case), "dtype": DTYPE[case["dtype"]]}
    # Powers of two near (largest magnitude) / (448 * 6), as a calibration would give them.
    if case["op"] == "round":
        state["x"] = _activations(generator, rows, cols, state["dtype"])
        state["factor"] = torch.full((1,), 2.0**-4, device="cuda") if fmt == "nvfp4" else None
    elif case["op"] == "expand":
        state["w"] = _stored(generator, rows, cols, fmt, 0.02, 2.0**-14)
    else:
        state["w"] = _stored(generator, case["n"], cols, fmt, 0.02, 2.0**-14)
        if case["op"] == "product":
            state["a"] = _stored(generator, rows, cols, fmt, 1.0, 2.0**-8)
        else:
            state["x"] = _activations(generator, rows, cols, state["dtype"])
            state["factor"] = torch.full((1,), 2.0**-4, device="cuda") if fmt == "nvfp4" else None
    return state


# ---- plain form --------------------------------------------------------------------------------


def _quantize(x, fmt, factor):
    """(magnitude, sign bit, scale byte) of every padded column and block.  In 64 bits, so that a
    value next to the border between two codes falls on the right side."""
    rows, cols = x.shape
    block = BLOCK[fmt]
    padded = torch.nn.functional.pad(x.float(), (0, -cols % 32)).reshape(rows, -1, block)
    largest = padded.abs().amax(-1)
    if fmt == "mxfp4":
        exponent = torch.frexp(largest)[1] - 1  # floor(log2)
        byte = torch.where(largest > 0, (exponent - 2).clamp(min=-127), -127) + 127
        step = torch.ldexp(torch.ones_like(largest, dtype=torch.float64), byte - 127)
    else:
        quotient = (largest.double() / (6.0 * factor).double()).clamp(max=448.0)
        place = (torch.frexp(quotient)[1] - 1).clamp(min=-6) - 3
        unit = torch.ldexp(torch.ones_like(quotient), place)
        scale = (torch.round(quotient / unit) * unit).float()
        byte = scale.to(torch.float8_e4m3fn).view(torch.uint8)
        step = (scale * factor).double()
    ratio = padded.double() / torch.where(step > 0, step, 1.0)[..., None]
    ratio = torch.where((step > 0)[..., None], ratio, 0.0)
    size = ratio.abs()
    grid = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    magnitude = (torch.round(size / grid) * grid).clamp(max=6.0).float()
    return magnitude.reshape(rows, -1), torch.signbit(padded).reshape(rows, -1), byte.to(torch.uint8)


def _pack(magnitude, sign):
    code = torch.where(magnitude < 2, magnitude * 2, torch.where(magnitude < 4, magnitude + 2, magnitude / 2 + 4))
    code = code.to(torch.uint8) | (sign.to(torch.uint8) << 3)
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _tile(scales, fmt):
    rows, blocks = scales.shape
    padded = torch.nn.functional.pad(scales, (0, -blocks % 4, 0, -rows % 128))
    tiles = padded.reshape((rows + 127) // 128, 4, 32, (blocks + 3) // 4, 4)
    return tiles.permute(0, 3, 2, 1, 4).contiguous()


def _untile(tiles, rows, blocks):
    flat = tiles.permute(0, 3, 2, 1, 4).reshape(tiles.shape[0] * 128, tiles.shape[1] * 4)
    return flat[:rows, :blocks]


def _scale_values(byte, fmt, factor):
    if fmt == "mxfp4":
        return torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte.to(torch.int32) - 127)
    return byte.view(torch.float8_e4m3fn).float() * factor


def _values(operand, fmt):
    """The FP32 values that codes and scales stand for, padded columns included."""
    codes, factor = operand["codes"], operand["factor"]
    rows, blocks = codes.shape[0], codes.shape[1] * 2 // BLOCK[fmt]
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat((table, -table))
    code = torch.stack((codes & 15, codes >> 4), -1).reshape(rows, blocks, BLOCK[fmt])
    scale = _scale_values(_untile(operand["scales"], rows, blocks).contiguous(), fmt, factor)
    return (table[code.int()] * scale[..., None]).reshape(rows, -1)


def _rounded(x, fmt, factor):
    """What a quantised x stands for, FP32, padded columns included."""
    magnitude, sign, byte = _quantize(x, fmt, factor)
    scale = _scale_values(byte.contiguous(), fmt, factor)
    value = torch.where(sign, -magnitude, magnitude).reshape(*scale.shape, BLOCK[fmt])
    return (value * scale[..., None]).reshape(x.shape[0], -1)


def run(state):
    case, dtype = state["case"], state["dtype"]
    fmt, cols = case["format"], case["cols"]
    if own:
        from lowbitlinear_b200 import microscaling

        if case["op"] == "round":
            codes, scales = microscaling.quantize_fp4(state["x"], format=fmt, tensor_scale=state["factor"])
            return microscaling.dequantize_fp4(codes, scales, cols, format=fmt, tensor_scale=state["factor"], dtype=dtype)
        w = state["w"]
        if case["op"] == "expand":
            return microscaling.dequantize_fp4(w["codes"], w["scales"], cols, format=fmt, tensor_scale=w["factor"], dtype=dtype)
        if case["op"] == "product":
            a = state["a"]
            return microscaling.matmul_fp4(a["codes"], a["scales"], w["codes"], w["scales"], format=fmt,
                                           a_scale=a["factor"], b_scale=w["factor"], dtype=dtype)
        return microscaling.linear_fp4(state["x"], w["codes"], w["scales"], format=fmt, tensor_scale=w["factor"],
                                       input_scale=state["factor"])
    if case["op"] == "round":
        return _rounded(state["x"], fmt, state["factor"])[:, :cols].to(dtype)
    if case["op"] == "expand":
        return _values(state["w"], fmt)[:, :cols].to(dtype)
    left = _values(state["a"], fmt) if case["op"] == "product" else _rounded(state["x"], fmt, state["factor"])
    return (left @ _values(state["w"], fmt).T).to(dtype)


def work(case):
    """Each input once, each output once; a rounding keeps nothing but the rounded values."""
    rows, cols, fmt = case["rows"], case["cols"], case["format"]
    size = 4 if case["dtype"] == "fp32" else 2
    stored = lambda r: r * cols / 2 + r * cols / BLOCK[fmt]  # noqa: E731
    if case["op"] == "round":
        return {"bytes": 2 * size * rows * cols, "flops": 0}
    if case["op"] == "expand":
        return {"bytes": stored(rows) + size * rows * cols, "flops": 0}
    left = stored(rows) if case["op"] == "product" else size * rows * cols
    n = case["n"]
    return {"bytes": left + stored(n) + size * rows * n, "flops": 2 * rows * n * cols}


# ---- definition in 64 bits ---------------------------------------------------------------------

_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_stored(operand, fmt):
    """Every code looked up by its bits, every scale byte decoded by its fields."""
    codes, tiles = operand["codes"].long(), operand["scales"].long()
    rows, block = codes.shape[0], BLOCK[fmt]
    cols = codes.shape[1] * 2
    column = torch.arange(cols, device=codes.device)
    nibble = (codes[:, column // 2] >> (4 * (column % 2))) & 15
    value = torch.tensor(_MAGNITUDES, dtype=torch.float64, device=codes.device)[nibble & 7]
    value = torch.where(nibble >= 8, -value, value)
    r = torch.arange(rows, device=codes.device)[:, None]
    j = (torch.arange(cols // block, device=codes.device))[None, :]
    byte = tiles[r // 128, j // 4, r % 32, r % 128 // 32, j % 4]
    if fmt == "mxfp4":
        scale = torch.pow(2.0, (byte - 127).double())
    else:
        power, fraction = (byte >> 3) & 15, (byte & 7).double()
        scale = torch.where(power == 0, fraction * 2.0**-9, (1 + fraction / 8) * torch.pow(2.0, (power - 7).double()))
        scale = scale * operand["factor"].double()
    return value * scale.repeat_interleave(block, 1)


def _exact_rounded(x, fmt, factor):
    """Quantisation by its borders: a code is the number of borders below the magnitude, and a
    magnitude on a border goes to the even side."""
    rows, cols = x.shape
    block = BLOCK[fmt]
    width = -(-cols // block) * block
    padded = torch.zeros(rows, width, dtype=torch.float64, device=x.device)
    padded[:, :cols] = x.double()
    size = padded.abs().reshape(rows, width // block, block)
    largest = size.max(-1).values
    if fmt == "mxfp4":
        # floor(log2) of an FP32 number by its exponent field; subnormal ones fall under the limit.
        field = (largest.float().view(torch.int32) >> 23).long()
        step = torch.pow(2.0, (field - 2).clamp(min=0).double() - 127)
    else:
        levels = torch.tensor([(f * 2.0**-9 if p == 0 else (1 + f / 8) * 2.0 ** (p - 7))
                               for p in range(16) for f in range(8)][:127], dtype=torch.float64, device=x.device)
        middle = (levels[1:] + levels[:-1]) / 2
        quotient = largest / (6 * factor).double()
        low = torch.searchsorted(middle, quotient)  # borders strictly below
        on_border = (low < 126) & (middle[low.clamp(max=125)] == quotient)
        step = levels[torch.where(on_border & (low % 2 == 1), low + 1, low)] * factor.double()
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=x.device)
    code = torch.zeros_like(size, dtype=torch.int8)
    for index, b in enumerate(border.tolist()):
        edge = step[..., None] * b
        code += (size >= edge if index % 2 else size > edge).to(torch.int8)
    code = torch.where(step[..., None] > 0, code, 0)
    value = torch.tensor(_MAGNITUDES, dtype=torch.float64, device=x.device)[code.int()] * step[..., None]
    return torch.where(padded < 0, -value.reshape(rows, width), value.reshape(rows, width))


def exact(case, seed):
    state = prepare(case, seed)
    fmt, cols = case["format"], case["cols"]
    if case["op"] == "round":
        return _exact_rounded(state["x"], fmt, state["factor"])[:, :cols]
    if case["op"] == "expand":
        return _exact_stored(state["w"], fmt)[:, :cols]
    left = _exact_stored(state["a"], fmt) if case["op"] == "product" else _exact_rounded(state["x"], fmt, state["factor"])
    return left[:, :cols] @ _exact_stored(state["w"], fmt)[:, :cols].T

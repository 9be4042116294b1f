"""Microscaled FP4 on CPU tensors: the torch arithmetic against the 64-bit oracle, the storage
layout, the module, and every refusal that needs no GPU."""
import ctypes

import numpy as np
import pytest
import torch

from lowbitlinear_b200 import MicroscaledLinear, microscaling
from lowbitlinear_b200.microscaling import (dequantize_fp4, linear_fp4, matmul_fp4, quantize_fp4, scale_shape,
                                            tile_scales, untile_scales)
from oracle import fp4_oracle as oracle

FORMATS = ("mxfp4", "nvfp4")
TYPES = (torch.float16, torch.bfloat16, torch.float32)


def hard_values(rows, cols, dtype, seed):
    """Normal values with every magnitude a format has to deal with: borders, zeros of both signs,
    subnormal numbers, wide blocks, values far above a block's other values."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    pick = torch.randint(0, 8, (rows, 1), generator=g)
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.0, -0.0])
    on_border = borders[torch.randint(0, len(borders), (rows, cols), generator=g)] * torch.sign(x)
    x = torch.where(pick == 0, on_border, x)
    x = torch.where(pick == 1, x * torch.exp2(torch.randint(-20, 12, (rows, cols), generator=g).float()), x)
    x = torch.where(pick == 2, x * 2.0**-16, x)
    x = torch.where(pick == 3, x * 2.0**13, x)
    x = torch.where(pick == 4, torch.zeros(()), x)
    return x.to(dtype)


def factor_of(fmt, value):
    return torch.tensor([value]) if fmt == "nvfp4" and value is not None else None


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (40, 32), (9, 33), (130, 100), (64, 1003)])
@pytest.mark.parametrize("factor", [None, 2.0**-6, 0.0123])
def test_quantize_matches_the_oracle(fmt, dtype, rows, cols, factor):
    x = hard_values(rows, cols, dtype, rows + cols)
    g = factor_of(fmt, factor)
    codes, scales = quantize_fp4(x, fmt, g)
    want_codes, want_bytes = oracle.quantize(x.double().numpy(), fmt, None if g is None else g.item())
    assert np.array_equal(codes.numpy(), oracle.pack(want_codes))
    assert np.array_equal(scales.numpy(), oracle.tile(want_bytes))
    for out in TYPES:
        got = dequantize_fp4(codes, scales, cols, fmt, g, out)
        want = torch.from_numpy(oracle.values(want_codes, want_bytes, fmt, None if g is None else g.item()))[:, :cols]
        # code * step in FP32 is at most one rounding away from the 64-bit product.
        assert torch.equal(got, want.float().to(out))


@pytest.mark.parametrize("fmt", FORMATS)
def test_blocks_that_are_not_finite_read_back_as_nan(fmt):
    x = torch.ones(3, 64)
    x[0, 5], x[1, 40], x[2, 63] = float("nan"), float("inf"), float("-inf")
    codes, scales = quantize_fp4(x, fmt)
    y = dequantize_fp4(codes, scales, 64, fmt)
    block = microscaling.FORMATS[fmt][1]
    # Ones: 2^-2 * 4 in mxfp4; in nvfp4 1 / 6 lies between the E4M3 numbers 10/64 and 11/64, nearer to the
    # upper one (10.67 / 64), and 1 / (11/64) = 5.8 is nearest to 6.
    one = 1.0 if fmt == "mxfp4" else 6 * 11 / 64
    for row, col in ((0, 5), (1, 40), (2, 63)):
        first = col // block * block
        bad = torch.zeros(64, dtype=torch.bool)
        bad[first:first + block] = True
        assert torch.equal(torch.isnan(y[row]), bad)
        assert torch.equal(y[row][~bad], torch.full((int((~bad).sum()),), one, dtype=torch.float16))
    if fmt == "nvfp4":
        for factor in (0.0, float("nan"), 2.0**70, -1.0):
            codes, scales = quantize_fp4(torch.ones(2, 32), fmt, torch.tensor([factor]))
            assert torch.equal(untile_scales(scales, 2, 2), torch.full((2, 2), 127, dtype=torch.uint8))


def test_scale_tiles_are_a_permutation():
    for rows, blocks in ((1, 1), (128, 4), (129, 5), (300, 33)):
        plain = torch.randint(0, 256, (rows, blocks), dtype=torch.uint8)
        tiles = tile_scales(plain)
        assert np.array_equal(tiles.numpy(), oracle.tile(plain.numpy()))
        assert torch.equal(untile_scales(tiles, rows, blocks), plain)
    assert scale_shape(129, 100, "mxfp4") == (2, 1, 32, 4, 4)
    assert scale_shape(129, 100, "nvfp4") == (2, 2, 32, 4, 4)


@pytest.mark.parametrize("fmt", FORMATS)
def test_products_and_layer_on_cpu(fmt):
    g = torch.Generator().manual_seed(3)
    weight = torch.randn(70, 100, generator=g) * 0.05
    x = torch.randn(9, 100, generator=g).half()
    layer = MicroscaledLinear.from_float(weight, fmt, input_scale=factor_of(fmt, 0.01))
    y = layer(x)
    xc, xb = oracle.quantize(x.double().numpy(), fmt, 0.01 if fmt == "nvfp4" else None)
    wf = None if layer.tensor_scale is None else layer.tensor_scale.item()
    wc, wb = oracle.quantize(weight.double().numpy(), fmt, wf)
    want = oracle.values(xc, xb, fmt, 0.01 if fmt == "nvfp4" else None) @ oracle.values(wc, wb, fmt, wf).T
    assert y.shape == (9, 70) and y.dtype == torch.float16
    # FP32 sums of 128 terms and one rounding to FP16.
    bound = np.abs(want) * 2.0**-11 + 256 * 2.0**-24 * np.abs(want).max() + 2.0**-24
    assert (np.abs(y.double().numpy() - want) <= bound * 1.01).all()
    codes, scales = quantize_fp4(x, fmt, layer.input_scale)
    assert torch.equal(matmul_fp4(codes, scales, layer.codes, layer.scales, fmt, layer.input_scale, layer.tensor_scale), y)
    again = MicroscaledLinear(layer.codes, layer.scales, layer.tensor_scale, layer.input_scale, in_features=100, format=fmt)
    again.load_state_dict(layer.state_dict())
    assert torch.equal(again(x), y)


def test_refusals():
    x = torch.ones(4, 64, dtype=torch.float16)
    codes, scales = quantize_fp4(x)
    nv_codes, nv_scales = quantize_fp4(x, "nvfp4")
    with pytest.raises(ValueError, match="format"):
        quantize_fp4(x, "int4")
    with pytest.raises(TypeError, match="Tensor"):
        quantize_fp4([1.0])
    with pytest.raises(TypeError, match="dtype"):
        quantize_fp4(x.double())
    with pytest.raises(ValueError, match="nonempty 2D"):
        quantize_fp4(x[0])
    with pytest.raises(ValueError, match="nonempty 2D"):
        quantize_fp4(x[:0])
    with pytest.raises(ValueError, match="nvfp4 only"):
        quantize_fp4(x, "mxfp4", torch.ones(1))
    with pytest.raises(TypeError, match="Tensor"):
        quantize_fp4(x, "nvfp4", 1.0)
    with pytest.raises(TypeError, match="dtype"):
        quantize_fp4(x, "nvfp4", torch.ones(1, dtype=torch.float16))
    with pytest.raises(ValueError, match="one value"):
        quantize_fp4(x, "nvfp4", torch.ones(2))
    with pytest.raises(ValueError, match="in_features"):
        dequantize_fp4(codes, scales, 0)
    with pytest.raises(ValueError, match="codes shape"):
        dequantize_fp4(codes, scales, 65)
    with pytest.raises(ValueError, match="scales shape"):
        dequantize_fp4(codes, tile_scales(torch.zeros(4, 5, dtype=torch.uint8)), 64, "nvfp4")
    with pytest.raises(TypeError, match="dtype"):
        dequantize_fp4(codes, scales, 64, dtype=torch.float64)
    with pytest.raises(TypeError, match="dtype"):
        dequantize_fp4(codes.int(), scales, 64)
    with pytest.raises(TypeError, match="dtype"):
        dequantize_fp4(codes, scales.int(), 64)
    with pytest.raises(ValueError, match="contiguous"):
        dequantize_fp4(codes.repeat(1, 2)[:, ::2], scales, 64)
    with pytest.raises(ValueError, match="incompatible K"):
        matmul_fp4(codes, scales, *quantize_fp4(torch.ones(4, 96)))
    with pytest.raises(TypeError, match="FP16 or BF16"):
        matmul_fp4(codes, scales, codes, scales, dtype=torch.float32)
    with pytest.raises(ValueError, match="incompatible K"):
        linear_fp4(torch.ones(4, 96, dtype=torch.float16), codes, scales)
    with pytest.raises(TypeError, match="dtype"):
        linear_fp4(x.float(), codes, scales)
    layer = MicroscaledLinear(nv_codes, nv_scales, in_features=64, format="nvfp4")
    with pytest.raises(ValueError, match="incompatible K"):
        layer(torch.ones(2, 63, dtype=torch.float16))
    with pytest.raises(ValueError, match="nonempty 2D"):
        layer(torch.ones(64, dtype=torch.float16))
    with pytest.raises(ValueError, match="scales shape"):
        MicroscaledLinear(torch.zeros(4, 64, dtype=torch.uint8), scales, in_features=128, format="nvfp4")


def test_c_entry_points_refuse_bad_arguments_without_a_gpu():
    from lowbitlinear_b200 import _extension

    if not _extension.load_cuda_extension(required=False):
        pytest.skip("native library not built")
    lib = _extension.native()
    error = lambda: lib.lbl_last_error()  # noqa: E731
    assert lib.lbl_fp4_quantize(16, 0, 4, 64, 64, 2, None, 16, 16, 0, None) == -1 and b"format" in error()
    assert lib.lbl_fp4_quantize(16, 3, 4, 64, 64, 0, None, 16, 16, 0, None) == -1 and b"type" in error()
    assert lib.lbl_fp4_quantize(16, 0, 4, 0, 64, 0, None, 16, 16, 0, None) == -1 and b"shape" in error()
    assert lib.lbl_fp4_quantize(16, 0, 4, 64, 64, 0, 16, 16, 16, 0, None) == -1 and b"NV format" in error()
    assert lib.lbl_fp4_quantize(16, 0, 4, 64, -64, 0, None, 16, 16, 0, None) == -1 and b"stride" in error()
    assert lib.lbl_fp4_quantize(None, 0, 4, 64, 64, 0, None, 16, 16, 0, None) == -1 and b"null" in error()
    assert lib.lbl_fp4_quantize(16, 0, 4, 64, 64, 0, None, 24, 16, 0, None) == -1 and b"aligned" in error()
    assert lib.lbl_fp4_quantize(None, 0, 0, 64, 64, 0, None, None, None, 0, None) == 0  # nothing to do
    assert lib.lbl_fp4_dequantize(16, 16, 4, 64, 0, None, 16, 5, 0, None) == -1 and b"type" in error()
    assert lib.lbl_fp4_dequantize(16, 16, 4, 64, 0, None, 18, 2, 0, None) == -1 and b"aligned" in error()
    assert lib.lbl_fp4_dequantize(16, None, 4, 64, 0, None, 16, 2, 0, None) == -1 and b"null" in error()
    assert lib.lbl_fp4_matmul(16, 16, None, 16, 16, None, 16, 4, 4, 64, 0, 2, 0, 0, None) == -1 and b"FP16 or BF16" in error()
    assert lib.lbl_fp4_matmul(16, 16, None, 8, 16, None, 16, 4, 4, 64, 0, 0, 0, 0, None) == -1 and b"aligned" in error()
    assert lib.lbl_fp4_matmul(16, 16, None, 16, 16, None, 16, 4, (1 << 30) + 1, 64, 0, 0, 0, 0, None) == -1
    assert lib.lbl_fp4_matmul(None, None, None, None, None, None, None, 0, 4, 64, 0, 0, 0, 0, None) == 0
    need = lib.lbl_fp4_linear_workspace_bytes(300, 128, 4096, 1)
    call = lambda ws, size: lib.lbl_fp4_linear(16, 0, 4096, None, 16, 16, None, 16, 300, 128, 4096, 1, ws, size, 0, 0, None)  # noqa: E731
    assert need > 0 and call(None, 0) == -3 and b"scratch" in error()
    assert call(16, need - 1) == -3 and call(8, need) == -1 and b"16-byte" in error()
    assert isinstance(error(), bytes) and ctypes.sizeof(ctypes.c_void_p) == 8

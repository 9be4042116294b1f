"""Microscaled FP4 on the GPU: codes and scales bit for bit against the 64-bit oracle, products and
the linear layer against 64-bit sums, and the calls a serving program makes: strides, other streams,
captured graphs, empty and extreme rows."""
import numpy as np
import pytest
import torch

from lowbitlinear_b200 import MicroscaledLinear
from lowbitlinear_b200.microscaling import dequantize_fp4, linear_fp4, matmul_fp4, quantize_fp4, untile_scales
from oracle import fp4_oracle as oracle
from test_microscaling import FORMATS, TYPES, factor_of, hard_values

pytestmark = pytest.mark.gpu
HALVES = (torch.float16, torch.bfloat16)


def on(device, t):
    return None if t is None else t.to(device)


def item(t):
    return None if t is None else t.item()


def stored(rows, cols, fmt, seed, factor=None, std=1.0):
    """An operand quantised by the oracle: tensors on the CPU and what they stand for, in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * std).double().numpy()
    codes, byte = oracle.quantize(x, fmt, factor)
    return (torch.from_numpy(oracle.pack(codes)), torch.from_numpy(oracle.tile(byte)),
            oracle.values(codes, byte, fmt, factor))


def check_product(got, a, b, dtype):
    """|got - sum| within: FP32 accumulation (one rounding of the running sum per 64 columns, three more
    within and after, each at most 2^-22 of the sum of magnitudes), one rounding to the output type, half
    a step of its subnormal numbers."""
    want = torch.from_numpy(a) @ torch.from_numpy(b).T
    size = torch.from_numpy(np.abs(a)) @ torch.from_numpy(np.abs(b)).T
    additions = -(-a.shape[1] // 64) + 4
    eps = torch.finfo(dtype).eps
    bound = additions * 2.0**-22 * size
    bound = bound + (want.abs() + bound) * eps / 2 + torch.finfo(dtype).tiny * eps / 2
    off = (got.double().cpu() - want).abs() - bound
    assert off.max().item() <= 0, f"outside the bound by {off.max().item():.3e} at {np.unravel_index(off.argmax().item(), off.shape)}"


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factor", [None, 2.0**-6, 0.0123])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 31), (40, 32), (129, 33), (130, 100), (300, 520), (7, 12288)])
def test_quantize_and_dequantize_match_the_oracle(cuda_ops, fmt, dtype, factor, rows, cols):
    x = hard_values(rows, cols, dtype, rows + cols)
    g = factor_of(fmt, factor)
    codes, scales = quantize_fp4(x.to(cuda_ops), fmt, on(cuda_ops, g))
    want_codes, want_bytes = oracle.quantize(x.double().numpy(), fmt, item(g))
    assert np.array_equal(codes.cpu().numpy(), oracle.pack(want_codes))
    assert np.array_equal(scales.cpu().numpy(), oracle.tile(want_bytes))  # padding included
    for out in TYPES:
        got = dequantize_fp4(codes, scales, cols, fmt, on(cuda_ops, g), out)
        want = torch.from_numpy(oracle.values(want_codes, want_bytes, fmt, item(g)))[:, :cols]
        assert torch.equal(got.cpu(), want.float().to(out))


@pytest.mark.parametrize("dtype", TYPES)
def test_values_next_to_the_borders_fall_on_the_right_side(cuda_ops, dtype):
    """NVFP4 values on a border between two codes and one or two units in the last place beside it, for tensor
    factors that are powers of two and others; for the 16-bit types the factor is moved instead, since their
    own numbers are too coarse to come that near."""
    rng = np.random.default_rng(11)
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    scales = oracle.E4M3[rng.integers(40, 120, 60)]
    if dtype == torch.float32:
        factors = [2.0**-6, 0.0123, 1 / 3, 7.1e-5]
    else:
        grid = torch.tensor([1.0009765625, 1.37, 1.9, 2.0**-3 * 1.21]).to(dtype).double().numpy()
        factors = [float(np.float32(x / (b * s)) + np.float32(k) * np.spacing(np.float32(x / (b * s))))
                   for x in grid for b, s in ((1.25, 13.0), (3.5, 0.6875), (0.75, 28.0)) for k in (-1, 0, 1)]
    for factor in factors:
        g = np.float32(factor)
        step = (scales.astype(np.float32) * g).astype(np.float32)
        near = (step[:, None].astype(np.float64) * borders).astype(np.float32)
        rows = [near]
        for _ in range(2):
            rows += [np.nextafter(rows[-1], np.float32(np.inf)), np.nextafter(near, np.float32(0))]
        x = np.concatenate([np.concatenate([(6 * step)[:, None], r, -r, np.zeros((len(step), 1), np.float32)], 1) for r in rows])
        x = torch.from_numpy(x).to(dtype)
        codes, got_scales = quantize_fp4(x.to(cuda_ops), "nvfp4", torch.tensor([factor], device=cuda_ops))
        want_codes, want_bytes = oracle.quantize(x.double().numpy(), "nvfp4", factor)
        assert np.array_equal(got_scales.cpu().numpy(), oracle.tile(want_bytes))
        assert np.array_equal(codes.cpu().numpy(), oracle.pack(want_codes))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite_and_extremes(cuda_ops, fmt, dtype):
    top = torch.finfo(dtype).max
    x = torch.randn(6, 96)
    x[0, 5], x[1, 40], x[2, 63] = float("nan"), float("inf"), float("-inf")
    x[3] = top
    x[4] = torch.where(torch.arange(96) % 2 == 0, -top, torch.finfo(dtype).tiny * 2.0**-4)
    x[5] = torch.finfo(dtype).tiny * 2.0**-3
    x = x.to(dtype)
    codes, scales = quantize_fp4(x.to(cuda_ops), fmt)
    want_codes, want_bytes = oracle.quantize(x.double().numpy(), fmt)
    assert np.array_equal(codes.cpu().numpy(), oracle.pack(want_codes))
    assert np.array_equal(scales.cpu().numpy(), oracle.tile(want_bytes))
    y = dequantize_fp4(codes, scales, 96, fmt, dtype=torch.float32).cpu()
    assert torch.equal(torch.isnan(y).any(1), torch.tensor([True, True, True, False, False, False]))
    if fmt == "nvfp4":
        for factor in (0.0, float("nan"), float("inf"), 2.0**70, -1.0):
            _, scales = quantize_fp4(x.to(cuda_ops), fmt, torch.tensor([factor], device=cuda_ops))
            assert (untile_scales(scales, 6, 6) == 127).all()


def test_quantize_takes_strided_and_unaligned_rows(cuda_ops):
    base = torch.randn(50, 200, device=cuda_ops).half()
    for view in (base[:, 3:131], base[::2, :128], base[:, ::2], base.t(), base[:1].expand(40, 200), base[10:]):
        for fmt in FORMATS:
            got, want = quantize_fp4(view, fmt), quantize_fp4(view.contiguous(), fmt)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1, 2, 35, 511, 512, 513, 1003, 1026])
def test_many_rows_that_start_on_any_address(cuda_ops, fmt, dtype, cols):
    """Enough rows that every multiprocessor works on several, one after the other: nothing of an earlier row
    reaches the padding of a later one."""
    rows = 4000
    x = hard_values(64, cols, dtype, cols).repeat(rows // 64 + 1, 1)[:rows]
    base = torch.full((rows * cols + 3,), 100.0, dtype=dtype, device=cuda_ops)
    codes, byte = oracle.quantize(x[:64].double().numpy(), fmt)
    packed = torch.from_numpy(oracle.pack(codes)).to(cuda_ops)
    values = torch.from_numpy(oracle.values(codes, byte, fmt))[:, :cols].float().to(dtype)
    byte = torch.from_numpy(byte).to(cuda_ops)
    for start in (0, 1, 2):
        view = base[start:start + rows * cols].view(rows, cols)
        view.copy_(x)
        got = quantize_fp4(view, fmt)
        assert torch.equal(got[0], packed.repeat(rows // 64 + 1, 1)[:rows])
        assert torch.equal(untile_scales(got[1], rows, byte.size(1)), byte.repeat(rows // 64 + 1, 1)[:rows])
    y = dequantize_fp4(*got, cols, fmt, dtype=dtype).cpu()
    assert torch.equal(y, values.repeat(rows // 64 + 1, 1)[:rows])


@pytest.mark.parametrize("fmt", FORMATS)
def test_more_rows_than_one_grid_holds(cuda_ops, fmt):
    rows, cols = 70001, 40
    x = torch.randn(rows, cols, device=cuda_ops).bfloat16()
    codes, scales = quantize_fp4(x, fmt)
    y = dequantize_fp4(codes, scales, cols, fmt, dtype=torch.bfloat16)
    picked = [0, 1, 65407, 65408, 65535, 65536, 70000]
    want_codes, want_bytes = oracle.quantize(x[picked].double().cpu().numpy(), fmt)
    assert np.array_equal(codes[picked].cpu().numpy(), oracle.pack(want_codes))
    want = torch.from_numpy(oracle.values(want_codes, want_bytes, fmt))[:, :cols]
    assert torch.equal(y[picked].cpu(), want.bfloat16())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,cols", [(2500, 8000), (1301, 15368), (9000, 2200)])
def test_large_matrices_get_the_codes_of_small_ones(cuda_ops, fmt, dtype, rows, cols):
    """Large matrices take more columns per thread: same codes and scales as block after block of 128 rows, and
    the oracle's for some of the rows."""
    x = hard_values(64, cols, dtype, cols).to(cuda_ops).repeat(rows // 64 + 1, 1)[:rows].contiguous()
    x[1::3] = torch.randn(x[1::3].shape, device=cuda_ops).to(dtype)
    g = on(cuda_ops, factor_of(fmt, 2.0**-6))
    codes, scales = quantize_fp4(x, fmt, g)
    for r0 in range(0, rows, 128):
        small = quantize_fp4(x[r0:r0 + 128], fmt, g)
        assert torch.equal(codes[r0:r0 + 128], small[0]) and torch.equal(scales[r0 // 128], small[1][0])
    picked = [0, 1, 2, 63, 130, rows - 1]
    want, _ = oracle.quantize(x[picked].double().cpu().numpy(), fmt, item(g))
    assert np.array_equal(codes[picked].cpu().numpy(), oracle.pack(want))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 64), (1, 129, 32), (2, 127, 33), (8, 64, 31), (9, 300, 96), (16, 256, 128),
                                   (17, 513, 160), (32, 130, 256), (33, 128, 257), (64, 200, 1000), (65, 77, 288),
                                   (128, 256, 512), (129, 255, 320), (256, 512, 1024), (300, 1030, 900), (520, 520, 4096)])
def test_product_matches_64_bits(cuda_ops, fmt, m, n, k):
    for dtype, fa, fb in ((torch.float16, None, 2.0**-7), (torch.bfloat16, 0.37, None)):
        fa, fb = (fa, fb) if fmt == "nvfp4" else (None, None)
        ac, as_, a = stored(m, k, fmt, m + k, fa)
        bc, bs, b = stored(n, k, fmt, n + k + 1, fb, 0.1)
        got = matmul_fp4(ac.to(cuda_ops), as_.to(cuda_ops), bc.to(cuda_ops), bs.to(cuda_ops), fmt,
                         on(cuda_ops, factor_of(fmt, fa)), on(cuda_ops, factor_of(fmt, fb)), dtype)
        assert got.shape == (m, n) and got.dtype == dtype
        check_product(got, a, b, dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1030, 2100, 320), (1537, 2048, 33), (257, 9601, 1500), (4097, 1000, 100), (2000, 4096, 2048),
                                   (200, 6150, 1100), (513, 2304, 4096)])
def test_large_products_match_64_bits(cuda_ops, fmt, m, n, k):
    """Persistent tiles: several per CTA pair, ragged edges, rows past the last one in half of a pair; the last two
    have so few tiles that two pairs share each."""
    test_product_matches_64_bits(cuda_ops, fmt, m, n, k)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n", [257, 258, 259, 260, 319, 321, 322, 323, 328, 511])
def test_rows_of_any_alignment_leave_the_large_product(cuda_ops, dtype, n):
    """Outputs whose rows start on a word or not, with the last columns in every place of a store."""
    m, k = 3001, 64
    ac, as_, a = stored(m, k, "mxfp4", n)
    bc, bs, b = stored(n, k, "mxfp4", n + 1)
    got = matmul_fp4(ac.to(cuda_ops), as_.to(cuda_ops), bc.to(cuda_ops), bs.to(cuda_ops), "mxfp4", dtype=dtype)
    check_product(got, a, b, dtype)


@pytest.mark.parametrize("fmt", FORMATS)
def test_offsets_past_32_bits(cuda_ops, fmt):
    """Matrices and products of more than 2^31 elements: their last rows are what the same rows are alone."""
    rows, cols = 66001, 33000
    tail = hard_values(300, cols, torch.bfloat16, 1).to(cuda_ops)
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=cuda_ops)
    x[-300:] = tail
    codes, scales = quantize_fp4(x, fmt)
    want = quantize_fp4(tail, fmt)
    assert torch.equal(codes[-300:], want[0]) and not codes[:-300].any()
    y = dequantize_fp4(codes, scales, cols, fmt, dtype=torch.bfloat16)
    assert torch.equal(y[-300:], dequantize_fp4(*want, cols, fmt, dtype=torch.bfloat16)) and not y[:-300].any()
    del x, y, codes, scales
    a = quantize_fp4(torch.randn(rows, 96, device=cuda_ops), fmt)
    b = quantize_fp4(torch.randn(cols, 96, device=cuda_ops), fmt)
    got = matmul_fp4(*a, *b, fmt)
    values = [dequantize_fp4(*t, 96, fmt, dtype=torch.float32).double().cpu().numpy() for t in (a, b)]
    for r in (slice(0, 2), slice(65534, 65538), slice(rows - 2, rows)):
        check_product(got[r], values[0][r], values[1], torch.float16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 3, 16, 40, 200, 600, 3000])
def test_rows_do_not_touch_each_other(cuda_ops, fmt, m):
    """A row whose blocks are NaN makes its own outputs NaN; an all-zero row gives zeros; every other
    row keeps its bits."""
    g = torch.Generator().manual_seed(m)
    x = torch.randn(m, 512, generator=g).half()
    w = torch.randn(1500 if m > 1000 else 320, 512, generator=g).half()
    operands = quantize_fp4(w.to(cuda_ops), fmt)
    clean = linear_fp4(x.to(cuda_ops), *operands, fmt).cpu()
    x[m // 2] = float("nan")
    if m > 2:
        x[0] = 0
    w[7, 100] = float("inf")
    got = linear_fp4(x.to(cuda_ops), *quantize_fp4(w.to(cuda_ops), fmt), fmt).cpu()
    assert torch.isnan(got[m // 2]).all() and torch.isnan(got[:, 7]).all()
    keep = torch.ones(m, w.size(0), dtype=torch.bool)
    keep[m // 2], keep[:, 7] = False, False
    if m > 2:
        assert (got[0, :7] == 0).all() and (got[0, 8:] == 0).all()
        keep[0] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 31, 64, 100, 128, 129, 300])
@pytest.mark.parametrize("n,k", [(256, 512), (1000, 4096), (130, 1003), (40, 12288)])
def test_linear_matches_64_bits(cuda_ops, fmt, dtype, m, n, k):
    x = hard_values(m, k, torch.bfloat16, m + n).clamp(-500, 500).to(dtype)
    g = factor_of(fmt, 0.02)
    wf = 2.0**-10 if fmt == "nvfp4" else None
    wc, ws, w = stored(n, k, fmt, n + k, wf, 0.02)
    xc, xb = oracle.quantize(x.double().numpy(), fmt, item(g))
    got = linear_fp4(x.to(cuda_ops), wc.to(cuda_ops), ws.to(cuda_ops), fmt, on(cuda_ops, factor_of(fmt, wf)), on(cuda_ops, g))
    assert got.dtype == dtype
    check_product(got, oracle.values(xc, xb, fmt, item(g)), w, dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1, 9601, 4000), (4, 9601, 4000), (5, 9601, 4000), (6, 8200, 8100), (7, 8200, 8100), (4, 5000, 12201),
                                   (3, 20001, 1500), (16, 33001, 500), (12, 2049, 8191)])
def test_wide_layers_with_few_rows_match_64_bits(cuda_ops, fmt, m, n, k):
    """Few rows on wide weights: one CTA per SM or several, long slices of K and short ones, and row counts on
    both sides of where the activations are quantised by a launch of their own."""
    g = torch.Generator(cuda_ops).manual_seed(m + n)
    weight = quantize_fp4(torch.randn(n, k, device=cuda_ops, generator=g).half(), fmt)
    x = hard_values(m, k, torch.bfloat16, m + n).clamp(-500, 500)
    got = linear_fp4(x.to(cuda_ops), *weight, fmt)
    xc, xb = oracle.quantize(x.double().numpy(), fmt)
    a = oracle.values(xc, xb, fmt)
    padded = a.shape[1]
    b = dequantize_fp4(*weight, padded, fmt, dtype=torch.float32)
    columns = torch.cat((torch.arange(0, n, 11), torch.arange(n - 130, n))).to(cuda_ops)
    check_product(got[:, columns], a, b[columns].double().cpu().numpy(), torch.bfloat16)
    assert torch.equal(got, matmul_fp4(*quantize_fp4(x.to(cuda_ops), fmt), *weight, fmt, dtype=torch.bfloat16))


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_linear_takes_strided_and_unaligned_rows(cuda_ops, m):
    base = torch.randn(m + 3, 700, device=cuda_ops).half()
    weight = quantize_fp4(torch.randn(256, 640, device=cuda_ops))
    for view in (base[3:, 8:648], base[:m, 1:641], base[:m, :640], base[:1].expand(m, 700)[:, 60:]):
        assert torch.equal(linear_fp4(view, *weight), linear_fp4(view.contiguous(), *weight))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 48, 300])
def test_repeated_calls_give_the_same_bits(cuda_ops, fmt, m):
    x = torch.randn(m, 4096, device=cuda_ops).bfloat16()
    weight = quantize_fp4(torch.randn(520, 4096, device=cuda_ops), fmt)
    first = linear_fp4(x, *weight, fmt)
    for _ in range(5):
        assert torch.equal(linear_fp4(x, *weight, fmt), first)


@pytest.mark.parametrize("fmt", FORMATS)
def test_layers_in_sequence_on_side_streams_and_in_a_graph(cuda_ops, fmt):
    """Two layers as a model runs them -- the second reads what the first writes -- on the current stream,
    on two other streams at once, and replayed from two graphs that run at the same time."""
    torch.manual_seed(0)
    up = MicroscaledLinear.from_float(torch.randn(1024, 512, device=cuda_ops) * 0.05, fmt)
    down = MicroscaledLinear.from_float(torch.randn(384, 1024, device=cuda_ops) * 0.05, fmt)
    for m in (1, 16, 200):
        xs = [torch.randn(m, 512, device=cuda_ops).bfloat16() for _ in range(2)]
        model = lambda x: down(torch.nn.functional.silu(up(x)))  # noqa: E731
        want = [model(x) for x in xs]
        reference = quantize_fp4(torch.nn.functional.silu(up(xs[0])), fmt)
        check_product(want[0], dequantize_fp4(*reference, 1024, fmt, dtype=torch.float32).double().cpu().numpy(),
                      dequantize_fp4(down.codes, down.scales, 1024, fmt, down.tensor_scale, torch.float32).double().cpu().numpy(),
                      torch.bfloat16)
        streams = [torch.cuda.Stream(cuda_ops) for _ in range(2)]
        got = [None, None]
        for i, stream in enumerate(streams):
            stream.wait_stream(torch.cuda.current_stream(cuda_ops))
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got[i] = model(xs[i])
        torch.cuda.synchronize(cuda_ops)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        graphs, outs = [], []
        for i, stream in enumerate(streams):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(model(xs[i]))
            graphs.append(graph)
        xs[0].copy_(xs[1])
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                stream.wait_stream(torch.cuda.current_stream(cuda_ops))
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize(cuda_ops)
        assert torch.equal(outs[0], want[1]) and torch.equal(outs[1], want[1])


def test_empty_outputs_and_refusals(cuda_ops):
    x = torch.ones(4, 64, dtype=torch.float16, device=cuda_ops)
    codes, scales = quantize_fp4(x)
    with pytest.raises(ValueError, match="same device"):
        linear_fp4(x.cpu(), codes, scales)
    with pytest.raises(ValueError, match="same device"):
        matmul_fp4(codes, scales, codes.cpu(), scales.cpu())
    with pytest.raises(ValueError, match="same device"):
        quantize_fp4(x, "nvfp4", torch.ones(1))
    # A row's codes must start on 16 bytes; a view that does not is refused on the host.
    shifted = torch.zeros(codes.numel() + 8, dtype=torch.uint8, device=cuda_ops)[8:].view_as(codes)
    with pytest.raises(RuntimeError, match="aligned"):
        matmul_fp4(shifted, scales, codes, scales)
    assert torch.equal(linear_fp4(x, codes, scales), torch.full((4, 4), 64.0, dtype=torch.float16, device=cuda_ops))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 40, 300])
def test_both_bindings_make_the_same_calls(cuda_ops, fmt, m, monkeypatch):
    """The torch binding and the ctypes path behind it: same bits, same refusals."""
    from lowbitlinear_b200 import _ops

    assert _ops.binding is not None, "csrc/binding.cpp was not built"
    g = on(cuda_ops, factor_of(fmt, 0.02))
    x = torch.randn(m, 200, device=cuda_ops).bfloat16()
    weight = quantize_fp4(torch.randn(300, 200, device=cuda_ops), fmt)

    def everything():
        codes, scales = quantize_fp4(x, fmt, g)
        outputs = [codes, scales, dequantize_fp4(codes, scales, 200, fmt, g, torch.float32),
                   dequantize_fp4(codes, scales, format=fmt, tensor_scale=g),
                   matmul_fp4(codes, scales, *weight, fmt, g, None, torch.bfloat16), linear_fp4(x, *weight, fmt, None, g)]
        outputs.append(quantize_fp4(torch.nn.Parameter(x.float()), fmt, g)[0])
        for bad, error in ((lambda: linear_fp4(x.double(), *weight, fmt), TypeError),
                           (lambda: linear_fp4(x[:, :100], *weight, fmt), ValueError),
                           (lambda: linear_fp4(x, weight[0], weight[1][:1], fmt), ValueError),
                           (lambda: linear_fp4(x[:0], *weight, fmt), ValueError),
                           (lambda: matmul_fp4(codes, scales, *weight, "fp4"), ValueError),
                           (lambda: dequantize_fp4(codes, scales, True, fmt), ValueError),
                           (lambda: dequantize_fp4(codes, scales, 1 << 70, fmt), ValueError),
                           (lambda: dequantize_fp4(codes, scales, 200, fmt, dtype="float"), TypeError),
                           (lambda: quantize_fp4(x, fmt, torch.ones(2, device=cuda_ops)), ValueError),
                           (lambda: quantize_fp4(x, [], g), ValueError)):
            with pytest.raises(error):
                bad()
        return outputs

    with_binding = everything()
    monkeypatch.setattr(_ops, "binding", None)
    for a, b in zip(with_binding, everything()):
        assert torch.equal(a, b) and a.dtype == b.dtype

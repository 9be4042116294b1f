"""Numpy oracle of the microscaled FP4 formats, in 64 bits and by the definitions' borders: a code
is found by comparing magnitudes with the midpoints between neighbouring numbers, never by dividing.
Checker only; the package does not import it."""
import numpy as np

BLOCK = {"mxfp4": 32, "nvfp4": 16}
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([f * 2.0**-9 if p == 0 else (1 + f / 8) * 2.0 ** (p - 7) for p in range(16) for f in range(8)][:127])


def _nearest(values, levels, unit):
    """Index of the level nearest to values / unit (unit broadcasts), ties to the even index."""
    index = np.zeros(values.shape, dtype=np.int64)
    for i in range(len(levels) - 1):
        border = (levels[i] + levels[i + 1]) / 2 * unit
        index += (values > border) | ((values == border) & (i % 2 == 1))
    return index


def quantize(x, fmt, factor=None):
    """float64 array holding FP16 / BF16 / FP32 values -> (codes [R, padded K], scale bytes [R, blocks])."""
    rows, k = x.shape
    block = BLOCK[fmt]
    padded = np.zeros((rows, (k + 31) // 32 * 32))
    padded[:, :k] = x
    blocks = padded.reshape(rows, -1, block)
    size = np.abs(blocks)
    amax = size.max(-1)
    bad = ~np.isfinite(size).all(-1)
    size = np.where(bad[..., None], 0.0, size)
    amax = np.where(bad, 0.0, amax)
    if fmt == "mxfp4":
        exponent = np.maximum(np.frexp(np.where(amax > 0, amax, 1.0))[1] - 3, -127)
        byte = np.where(amax > 0, exponent + 127, 0)
        step = np.exp2(byte - 127.0)
        byte = np.where(bad, 255, byte)
    else:
        g = np.float32(1.0 if factor is None else factor)
        if not (2.0**-64 <= g <= 2.0**64):
            bad, g = np.ones_like(bad), np.float32(1.0)
        six_g = float(np.float32(6.0) * g)
        byte = np.where(bad, 127, _nearest(amax, E4M3, six_g))
        step = (E4M3[np.where(bad, 0, byte)].astype(np.float32) * g).astype(np.float64)
    code = _nearest(size, E2M1, step[..., None])
    code = np.where(step[..., None] > 0, code, 0) | (np.signbit(blocks).astype(np.int64) << 3)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(rows, -1).astype(np.uint8), byte.astype(np.uint8)


def pack(codes):
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpack(packed):
    return np.stack((packed & 15, packed >> 4), -1).reshape(packed.shape[0], -1)


def tile(byte):
    """Scale bytes [R, blocks] -> tiles, byte by byte."""
    rows, blocks = byte.shape
    out = np.zeros(((rows + 127) // 128, (blocks + 3) // 4, 32, 4, 4), dtype=np.uint8)
    r, j = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    out[r // 128, j // 4, r % 32, r % 128 // 32, j % 4] = byte
    return out


def steps(byte, fmt, factor=None):
    if fmt == "mxfp4":
        return np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    value = np.where(byte & 127 == 127, np.nan, E4M3[np.minimum(byte & 127, 126)]) * np.where(byte >= 128, -1.0, 1.0)
    g = np.float32(1.0 if factor is None else factor)
    return (value.astype(np.float32) * g).astype(np.float64)


def values(codes, byte, fmt, factor=None):
    """float64 [R, padded K]: code * step, the step rounded to FP32 as stored arithmetic has it."""
    number = E2M1[codes & 7] * np.where(codes >= 8, -1.0, 1.0)
    rows = codes.shape[0]
    return (number.reshape(rows, -1, BLOCK[fmt]) * steps(byte, fmt, factor)[..., None]).reshape(rows, -1)

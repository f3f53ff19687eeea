"""The 4-bit floating-point formulas in 64 bits, from their definitions (no GPU, none of the library's code)."""
import numpy as np
import torch

TABLE = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
TABLE = np.concatenate([TABLE, -TABLE])
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # half a step of a value of 1 to 2


def up(n, m):
    return -(-n // m) * m


def blocks_of(x):
    """x [m][k] (numpy, f32 values) as [m][blocks][32], zeros behind."""
    m, k = x.shape
    out = np.zeros((m, up(k, 32)), x.dtype)
    out[:, :k] = x
    return out.reshape(m, -1, 32)


def ref_codes(x):
    """(code numbers [m][k up to 32], scale bytes [m][k / 32 up to 4]) of x (CPU tensor) along its rows."""
    b = blocks_of(x.float().numpy())
    amax = np.abs(b).max(axis=-1)
    e = amax.view(np.uint32).astype(np.int64) >> 23
    byte = np.where(np.isfinite(amax), np.maximum(e, 2) - 2, 255)
    with np.errstate(all="ignore"):
        v = np.ldexp(b.astype(np.float64), 127 - np.where(byte == 255, 0, byte)[..., None])
        mag = np.where(np.isfinite(v), np.abs(v), 0.0)
        # to nearest, a tie to the code of even number
        code = np.abs(mag[..., None] - TABLE[:8]).argmin(axis=-1)
        tie = (code < 7) & (mag * 2 == TABLE[:8][code] + TABLE[:8][np.minimum(code + 1, 7)])
        code = np.where(tie & (code % 2 == 1), code + 1, code)
    code = np.where(byte[..., None] == 255, 0, code + 8 * np.signbit(b))
    pad = np.zeros((x.shape[0], up(byte.shape[1], 4)), np.uint8)
    pad[:, :byte.shape[1]] = byte
    return code.reshape(x.shape[0], -1).astype(np.uint8), pad


def pack(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def values(code, byte):
    """What code numbers and scale bytes stand for, in f64; a NaN under a scale of 255."""
    n = code.shape[-1] // 32
    s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(np.int64) - 127))
    return TABLE[code] * np.repeat(s[..., :n], 32, axis=-1)


def random_codes(rng, m, k, lo=120, hi=132):
    """Every code alike, scales of 2^(lo - 127) to 2^(hi - 127), 255 behind the row's blocks: what lies there has no say."""
    code = rng.integers(0, 16, (m, k)).astype(np.uint8)
    byte = np.full((m, up(k, 128) // 32), 255, np.uint8)
    byte[:, :k // 32] = rng.integers(lo, hi, (m, k // 32))
    return code, byte


def product_bound(a, b, y, dtype, slices=16):
    """How far y = a b^T may be off: a block's sum is exact, each block enters through one f32 rounding, the slices of K
    and their join through `slices` more, each relative to the sum of the magnitudes; half a step of the output type; and
    the smallest f32 number for results below the normal ones."""
    mag = np.abs(a) @ np.abs(b).T
    return (a.shape[1] / 32 + slices) * 2.0 ** -24 * mag + HALF[dtype] * np.abs(y) + 2.0 ** -133

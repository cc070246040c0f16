"""The microscaled formats from their definition (OCP MX), in 64 bits: what drama3/mx.py's quantizer, values and
products are checked against."""
import numpy as np

BLOCK = 32
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _e4m3():
    """e4m3's non-negative finite values, code 0 .. 126: four exponent bits biased by 7, three mantissa bits."""
    c = np.arange(127)
    e, m = c >> 3, c & 7
    return np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10))


E4M3 = _e4m3()


def grid(bits):
    return E2M1 if bits == 4 else E4M3


def element(v, bits):
    """Codes of float64 values: the nearest of the format's magnitudes, a tie to the even code, beyond the largest that one;
    the sign in the top bit."""
    g = grid(bits)
    a = np.abs(v)
    high = np.searchsorted(g, a).clip(max=len(g) - 1)
    low = (high - 1).clip(min=0)
    down, up = a - g[low], g[high] - a
    code = np.where((down < up) | ((down == up) & (low % 2 == 0)), low, high)
    return code | (np.signbit(v).astype(np.int64) << (bits - 1))


def quantize(x, bits):
    """(codes [R, C], scale codes [R, C / 32]) of rows x [R, C], one element a byte. The elements of a block whose scale
    is NaN are 0."""
    block = np.asarray(x, np.float64).reshape(x.shape[0], -1, BLOCK)
    amax = np.abs(block).max(axis=-1)
    bad = ~np.isfinite(amax)
    amax = np.where(bad, 0.0, amax)
    _, e = np.frexp(amax)  # amax in [2^(e - 1), 2^e)
    scale = np.where(amax == 0, 0, np.clip(e - 1 - (2 if bits == 4 else 8) + 127, 0, 254))
    v = np.where(bad[..., None], 0.0, block) / np.exp2(scale - 127.0)[..., None]
    return element(v, bits).reshape(x.shape).astype(np.uint8), np.where(bad, 255, scale).astype(np.uint8)


def values(codes, scale, bits):
    """float64 values of codes [R, C] (one a byte) and their blocks' scale codes."""
    sign = np.where(codes >> (bits - 1), -1.0, 1.0)
    magnitude = np.append(grid(bits), np.nan if bits == 8 else [])[codes & ((1 << (bits - 1)) - 1)]
    factor = np.where(scale == 255, np.nan, np.exp2(scale.astype(np.float64) - 127.0))
    return sign * magnitude * np.repeat(factor, BLOCK, axis=-1)


def pack(codes, bits):
    """One code a byte -> as rows hold them."""
    return codes if bits == 8 else codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpack(codes, bits):
    return codes if bits == 8 else np.stack((codes & 15, codes >> 4), axis=-1).reshape(codes.shape[0], -1)

"""Plain 64-bit statements of the operators on rows in few bits (numpy), for their tests."""
import numpy as np
import torch

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
TORCH = {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}
EPS = {0: 2.0 ** -24, 1: 2.0 ** -11, 2: 2.0 ** -8}   # half a step of a rounding, relative to the value


def mx4_encode(x):
    """codes [n][nb * 32] (0 .. 15) and scale bytes [n][nb] of float64 rows."""
    n, d = x.shape
    nb = -(-d // 32)
    v = np.zeros((n, nb, 32))
    v.reshape(n, -1)[:, :d] = x
    fine = np.isfinite(v).all(2)
    v = np.where(fine[:, :, None], v, 0.0)
    top = np.abs(v).max(2)
    _, e = np.frexp(top)                              # top = m 2^e, 1/2 <= m < 1
    e = np.where(top > 0, np.clip(e - 3, -127, 125), -127)
    u = v / np.exp2(e.astype(np.float64))[:, :, None]
    gap = np.abs(np.abs(u)[..., None] - MAGNITUDES)
    # nearest; of two as near ones the even code
    order = gap * 4 + (np.arange(8) & 1) * 1e-9 * (gap == gap.min(-1, keepdims=True))
    mag = np.where(np.abs(u) >= 6.0, 7, np.argmin(order, -1))
    codes = np.where(fine[:, :, None], mag + 8 * np.signbit(u), 0)
    return codes.reshape(n, nb * 32).astype(np.uint8), np.where(fine, e + 127, 255).astype(np.uint8)


def mx4_values(codes, scales, d):
    n, nb = scales.shape
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    v = MAGNITUDES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    return (v.reshape(n, nb, 32) * s[:, :, None]).reshape(n, nb * 32)[:, :d]


def mx4_pack(codes, scales, fill=127):
    """Packed codes and scale bytes as the library lays them out; scale bytes of rows behind n get `fill`."""
    n, nb = scales.shape
    ng, nt = -(-nb // 4), -(-n // 128)
    packed = codes[:, 0::2] | codes[:, 1::2] << 4
    out = np.full(512 * nt * ng, fill, np.uint8)
    r = np.arange(n)[:, None]
    c = np.arange(ng * 4)[None, :]
    at = (r // 128 * ng + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4
    full = np.full((n, ng * 4), 127, np.uint8)
    full[:, :nb] = scales
    out[at] = full
    return packed, out


def mx4_unpack(packed, scales, n, nb):
    codes = np.stack((packed & 15, packed >> 4), 2).reshape(n, nb * 32)
    ng = -(-nb // 4)
    r = np.arange(n)[:, None]
    c = np.arange(nb)[None, :]
    return codes, scales[(r // 128 * ng + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4]


def rms_norm(s, weight, eps):
    """The normalised rows, float64."""
    return s / np.sqrt((s * s).mean(1, keepdims=True) + eps) * weight


def random_mx4(rng, n, d, spread=2):
    """Random codes and scale bytes whose products add up exactly in fp32."""
    nb = -(-d // 32)
    codes = rng.integers(0, 16, (n, nb * 32)).astype(np.uint8)
    codes[:, d:] = 0
    return codes, rng.integers(127 - spread, 128 + spread, (n, nb)).astype(np.uint8)

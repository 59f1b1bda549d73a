"""Plain 64-bit forms of the 8-bit operators: e4m3 codes, 4-bit weight rows, norm, quantiser, rotation."""
from __future__ import annotations

import numpy as np

Q4_0, Q4_1, Q4_K = 2, 3, 12
GROUP_BYTES = {Q4_0: (32, 18), Q4_1: (32, 20), Q4_K: (256, 144)}
LEAST = 2.0 ** -100


def _e4m3_table() -> np.ndarray:
    t = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        t[c] = np.nan if c & 127 == 127 else (-v if c & 128 else v)
    return t


E4M3 = _e4m3_table()


def random_codes(rng, shape) -> np.ndarray:
    """Every finite e4m3 code, the subnormals and zeros of both signs among them."""
    c = rng.integers(0, 127, shape).astype(np.uint8)
    return c | (rng.integers(0, 2, shape).astype(np.uint8) << 7)


def random_weights(rng, w_type: int, out_dim: int, in_dim: int) -> np.ndarray:
    """Rows of blocks with arbitrary codes and finite fp16 scales of both signs (zero and subnormal ones too)."""
    per, size = GROUP_BYTES[w_type]
    raw = rng.integers(0, 256, (out_dim, in_dim // per, size)).astype(np.uint8)
    n_half = 1 if w_type == Q4_0 else 2
    h = (rng.standard_normal((out_dim, in_dim // per, n_half)) * 0.02).astype(np.float16)
    special = rng.random(h.shape)
    h[special < 0.02] = 0.0
    h[(special >= 0.02) & (special < 0.04)] = np.float16(3e-7)
    raw[..., : 2 * n_half] = h.view(np.uint8).reshape(out_dim, in_dim // per, 2 * n_half)
    return raw.reshape(out_dim, -1)


def decode_weights(w_type: int, raw: np.ndarray, in_dim: int):
    """(the float64 weights, and a bound of the magnitudes that a group's sum passes through: the
    codes' part and the offset's part of each weight added up without their signs)."""
    n = raw.shape[0]
    per, size = GROUP_BYTES[w_type]
    b = raw.reshape(n, in_dim // per, size)

    def half(at):
        return np.ascontiguousarray(b[..., at:at + 2]).view(np.float16).astype(np.float64)[..., 0]

    if w_type == Q4_K:
        scales = np.zeros((n, in_dim // 256, 8))
        mins = np.zeros_like(scales)
        for g in range(8):
            if g < 4:
                scales[..., g] = b[..., 4 + g] & 63
                mins[..., g] = b[..., 8 + g] & 63
            else:
                scales[..., g] = (b[..., 8 + g] & 15) | (b[..., g] >> 6) << 4
                mins[..., g] = (b[..., 8 + g] >> 4) | (b[..., 4 + g] >> 6) << 4
        qs = b[..., 16:].reshape(n, -1, 4, 32)
        q = np.stack([qs & 15, qs >> 4], -2).reshape(n, -1, 8, 32).astype(np.float64)
        part = (half(0)[..., None] * scales)[..., None] * q
        off = -(half(2)[..., None] * mins)[..., None] * np.ones(32)
    else:
        qs = b[..., size - 16:]
        q = np.concatenate([qs & 15, qs >> 4], -1).astype(np.float64)
        part = half(0)[..., None] * q
        off = (-8.0 * half(0) if w_type == Q4_0 else half(2))[..., None] * np.ones(32)
    return (part + off).reshape(n, in_dim), (np.abs(part) + np.abs(off)).reshape(n, in_dim)


def norm64(x, residual, weight, eps):
    """(sum as fp32, y in float64 from that sum)."""
    s = x if residual is None else x + residual
    s64 = s.astype(np.float64)
    y = s64 / np.sqrt(np.mean(s64 * s64, -1, keepdims=True) + float(np.float32(eps))) * weight.astype(np.float64)
    return s, y


def check_codes(codes, scale, y, rel):
    """Codes and scales of rows y (float64) that were computed to a relative error `rel`.

    The scale is max(max |y|, 2^-100) / 448 to that error and one rounding of the division.  A code is
    off from y / scale by at most half a step, 2^-4 of a normal value and 2^-10 of a subnormal one, and by what
    the two relative errors and the factor's two roundings move the value before it is rounded."""
    want = np.maximum(np.max(np.abs(y), -1), LEAST) / 448.0
    assert np.all(np.abs(scale - want) <= (rel + 2.0 ** -23) * want)
    v = y / want[:, None]
    slack = (2 * rel + 4 * 2.0 ** -24) * np.abs(v) * 1.1
    got = E4M3[codes]
    assert np.all(np.isfinite(got))
    assert np.all(np.abs(got - v) <= np.maximum(np.abs(v) * 2.0 ** -4, 2.0 ** -10) + slack)


def axis_of_pair(sections, interleaved: bool):
    n, half = len(sections), sum(sections)
    if not interleaved:
        return np.repeat(np.arange(n), sections)
    j = np.arange(half)
    m = j % n
    return np.where(j < n * np.asarray(sections)[m], m, 0)


def rotate64(x, axes, axis, rates, rope_dim, halves: bool, mscale=1.0):
    """x [tokens, heads, d] turned in float64; axes [n_axes, tokens]; and |x0| + |x1| of each value's pair."""
    x = x.astype(np.float64)
    y, mag = x.copy(), np.abs(x)
    half = rope_dim // 2
    j = np.arange(half)
    e0, e1 = (j, j + half) if halves else (2 * j, 2 * j + 1)
    ang = axes[axis].T.astype(np.float64) * rates[None, :]
    c, s = (np.cos(ang) * mscale)[:, None], (np.sin(ang) * mscale)[:, None]
    y[..., e0] = x[..., e0] * c - x[..., e1] * s
    y[..., e1] = x[..., e0] * s + x[..., e1] * c
    mag[..., e0] = mag[..., e1] = (np.abs(x[..., e0]) + np.abs(x[..., e1])) * mscale
    return y, mag

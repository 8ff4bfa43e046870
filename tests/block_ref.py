"""Plain forms in 64 bits (numpy) of the operators over 8-bit blocks and of paged_norm_rotate, shared by their tests."""

import numpy as np

import paged_ref as R

BLOCK = 128


def blocks(n):
    return -(-n // BLOCK)


def quantize(x, rows):
    """Codes (bits) and scales of x (float64 values of its type), block by block."""
    M, K = x.shape
    codes, scales = np.zeros((M, K), np.uint8), np.zeros((-(-M // rows), blocks(K)))
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            at = np.s_[i * rows:(i + 1) * rows, j * BLOCK:(j + 1) * BLOCK]
            part = x[at]
            fine = np.abs(part[np.isfinite(part)])
            s = max(R.f32((fine.max() if fine.size else 0.0) / 448.0), 2.0 ** -126)
            with np.errstate(invalid="ignore", over="ignore"):
                codes[at] = R.encode(R.f32(part * R.f32(1.0 / s)), "e4m3")
            scales[i, j] = s
    return codes, scales


def matmul(a, a_scale, b, b_scale):
    """The product of codes (bits) and their scales, and the sum of its terms' sizes."""
    K = a.shape[1]
    out, size = 0.0, 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        for j in range(blocks(K)):
            k = slice(j * BLOCK, (j + 1) * BLOCK)
            x, y = R.decode(a[:, k], "e4m3"), R.decode(b[:, k], "e4m3")
            f = a_scale[:, j, None].astype(np.float64) * np.repeat(b_scale[:, j].astype(np.float64), BLOCK)[None, :b.shape[0]]
            out = out + (x @ y.T) * f
            size = size + (np.abs(x) @ np.abs(y).T) * np.abs(f)
    return out, size


def most(a, a_scale, b, b_scale):
    """For each result the sum over eights of neighbouring columns of the largest of their terms' sizes."""
    K, out = a.shape[1], np.zeros((a.shape[0], b.shape[0]))
    scale = np.abs(np.repeat(b_scale.astype(np.float64), BLOCK, 0)[:b.shape[0]])
    for k in range(0, K, 8):
        x, y = np.abs(R.decode(a[:, k:k + 8], "e4m3")), np.abs(R.decode(b[:, k:k + 8], "e4m3"))
        terms = x[:, None, 0] * y[None, :, 0]
        for i in range(1, x.shape[1]):
            np.maximum(terms, x[:, None, i] * y[None, :, i], out=terms)
        out += terms * np.abs(a_scale[:, k // BLOCK, None].astype(np.float64)) * scale[None, :, k // BLOCK]
    return out


def rotate(x, weight, cos, sin, pos, eps, interleaved):
    """Rows x [T, H, D] at positions pos, and the size of each result's terms."""
    T, H, D = x.shape
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    r = cos.shape[1]
    z, size = y.copy(), np.abs(y)
    c, s = cos[pos][:, None].astype(np.float64), sin[pos][:, None].astype(np.float64)
    lo, hi = (np.s_[..., 0:2 * r:2], np.s_[..., 1:2 * r:2]) if interleaved else (np.s_[..., :r], np.s_[..., r:2 * r])
    z[lo], z[hi] = y[lo] * c - y[hi] * s, y[hi] * c + y[lo] * s
    size[lo], size[hi] = np.abs(y[lo] * c) + np.abs(y[hi] * s), np.abs(y[hi] * c) + np.abs(y[lo] * s)
    return z, size

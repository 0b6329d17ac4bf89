"""64-bit definitions of the MXFP4 format, the experts on it and the block norms
(numpy), shared by their tests."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
VALUES = np.concatenate([GRID, -GRID])


def quantize(x):
    """(codes, scales) of float64 x [..., K]: the definition, value by value."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    big = np.abs(b).max(-1)
    bad = ~np.isfinite(big)
    _, e = np.frexp(np.where(bad, 1.0, big))
    scale = np.where(big == 0, 0, np.maximum(e - 3 + 127, 0))
    scale = np.where(bad, 255, scale).astype(np.uint8)
    with np.errstate(invalid="ignore"):
        a = np.minimum(np.abs(np.ldexp(np.where(bad[..., None], 0.0, b), 127 - scale.astype(int)[..., None])), 6.0)
    dist = np.abs(a[..., None] - GRID)
    best = dist.min(-1, keepdims=True)
    tie = dist == best                                   # at most two neighbours: prefer the even code
    code = np.where(tie[..., 0::2].any(-1), 2 * tie[..., 0::2].argmax(-1), 2 * tie[..., 1::2].argmax(-1) + 1)
    code = (code | (np.signbit(b) & ~bad[..., None]) * 8).astype(np.uint8).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def dequantize(codes, scales):
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    return VALUES[c] * np.repeat(s, 32, axis=-1)


def ffn_rows(x, g, u, d):
    """(y, bound) of one expert on rows x [n, H] in float64.

    The bound covers what the kernels round: x as two E4M3 pieces (an absolute
    2^-21 of the row's largest value at most), FP32 sums (n 2^-24 of the sum of
    magnitudes), h as two E4M3 pieces (2^-8 of the value, or 2^-21 of the
    largest of 32), and one BF16 rounding (2^-8)."""
    gl, ul = x @ g.T, x @ u.T
    sig = 1 / (1 + np.exp(-gl))
    h = gl * sig * ul
    top = np.abs(x).max(-1, keepdims=True)
    dg = 2.0 ** -21 * top * np.abs(g).sum(-1) + x.shape[1] * 2.0 ** -24 * (np.abs(x) @ np.abs(g).T)
    du = 2.0 ** -21 * top * np.abs(u).sum(-1) + x.shape[1] * 2.0 ** -24 * (np.abs(x) @ np.abs(u).T)
    # |silu'| <= 1.1; a few FP32 roundings in the activation
    dh = 1.1 * dg * (np.abs(ul) + du) + np.abs(gl * sig) * du + 2.0 ** -20 * np.abs(h)
    blocks = np.pad(np.abs(h), ((0, 0), (0, -h.shape[1] % 32))).reshape(h.shape[0], -1, 32).max(-1)
    dh = dh + 2.0 ** -8 * np.abs(h) + 2.0 ** -21 * np.repeat(blocks, 32, axis=1)[:, :h.shape[1]]
    y = h @ d.T
    dy = dh @ np.abs(d).T + h.shape[1] * 2.0 ** -24 * (np.abs(h) @ np.abs(d).T)
    return y, dy + 2.0 ** -8 * (np.abs(y) + dy) + 1e-38


def norm(v, how, weight, eps):
    if how == "none":
        return v
    c = v - v.mean(-1, keepdims=True) if how == "layer" else v
    n = c / np.sqrt((c * c).mean(-1, keepdims=True) + eps)
    return n if weight is None else n * weight


def block_norm(y, residual, *, post="none", post_weight=None, gate=None, gate_act="none", residual_scale=1.0,
               block_scale=1.0, pre="rms", pre_weight=None, eps=1e-6):
    """(stream, normed) in float64."""
    s = residual_scale * residual
    if y is not None:
        z = norm(y, post, post_weight, eps)
        if gate is not None:
            z = z * (1 / (1 + np.exp(-gate)) if gate_act == "sigmoid" else gate)
        s = s + block_scale * z
    return s, norm(s, pre, pre_weight, eps)

"""The 4-bit microscaled form written from its definition in numpy, in 64 bits:
what the tests compare the kernels with."""
import numpy as np
import torch

VALUES = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def encode(x):
    """x float [..., k] -> (codes uint8 [..., ceil(k/32)*32], one a byte, scales
    uint8 [..., ceil(k/32)])."""
    x = np.asarray(x, dtype=np.float64)
    k = x.shape[-1]
    x = np.concatenate([x, np.zeros(x.shape[:-1] + (-k % 32,))], -1).reshape(x.shape[:-1] + (-1, 32))
    top = np.abs(x).max(-1)
    bad = ~np.isfinite(x).all(-1)
    safe = np.where(bad | (top == 0), 1.0, top)
    e = np.floor(np.log2(safe)).astype(np.int64)
    e = np.where(np.ldexp(1.0, e) > safe, e - 1, e)          # log2 rounds
    e = np.where(np.ldexp(1.0, e + 1) <= safe, e + 1, e)
    e = np.where(top == 0, -127, np.maximum(e - 2, -127))
    q = np.abs(np.where(bad[..., None], 0.0, x)) / np.ldexp(1.0, e)[..., None]
    q = np.minimum(q, 6.0)
    d = np.abs(q[..., None] - VALUES)
    low = d.min(-1)
    # of the (at most two) nearest values the one with the even code
    near = d == low[..., None]
    first = near.argmax(-1)
    code = np.where((near.sum(-1) == 2) & (first % 2 == 1), first + 1, first)
    code = code + 8 * (np.signbit(x) & ~bad[..., None])
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    return code.astype(np.uint8).reshape(code.shape[:-2] + (-1,)), scales


def decode(codes, scales):
    """The values, float64 [..., blocks*32]."""
    v = VALUES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    v = v.reshape(v.shape[:-1] + (-1, 32))
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v * s[..., None]).reshape(codes.shape)


def packed(codes):
    """Two codes a byte, the even index low."""
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def rounded(x):
    """The values of the 4-bit form of a tensor [..., k], float64."""
    x = x.detach().cpu().double().numpy()
    return torch.from_numpy(decode(*encode(x))[..., :x.shape[-1]])

"""The paged 4-bit cache and the rotation in numpy, for the tests: the format
in the fp32 steps that define it, the attention in 64 bits."""
import math

import numpy as np

LIMIT = 16384.0
U16 = 2.0 ** -11  # half a step of fp16, relative


def quantize(x):
    """(codes, scale fp16, bias fp16) of fp16 rows [..., dim], 32 channels a group."""
    x = np.clip(np.nan_to_num(x.astype(np.float32), nan=0.0, posinf=LIMIT, neginf=-LIMIT),
                -LIMIT, LIMIT).astype(np.float32)
    x = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    low, high = x.min(-1), x.max(-1)
    scale = ((high - low) / np.float32(15)).astype(np.float16)
    s = scale.astype(np.float32)
    bias = (low - np.float32(16) * s).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        steps = (x - bias.astype(np.float32)[..., None]) / s[..., None]
    codes = np.clip(np.rint(steps) - 16, 0, 15)
    return np.where(s[..., None] > 0, codes, 0.0), scale, bias


def kept(x):
    """The cache's values (fp16) of fp16 rows."""
    codes, scale, bias = quantize(x)
    # exact in 64 bits, so rounded once
    y = (16.0 + codes) * scale.astype(np.float64)[..., None] + bias.astype(np.float64)[..., None]
    return y.astype(np.float16).reshape(x.shape)


def turned(x, positions, freqs, factor, layout):
    """Rows [T, H, dim] rotated in 64 bits, and how far fp16 outputs of the
    fp32 arithmetic may be from them: half a step of fp16 (and of its
    subnormals), and for c, s, two products and a sum of fp32 a half step of
    (|x| + |y|) factor each."""
    x = x.astype(np.float64)
    half = freqs.size
    angle = np.asarray(positions, np.float64)[:, None] * freqs.astype(np.float64)
    c, s = (np.cos(angle) * factor)[:, None], (np.sin(angle) * factor)[:, None]
    a = np.arange(half) * (1 if layout == "half" else 2)
    b = a + (half if layout == "half" else 1)
    want, far = x.copy(), np.zeros_like(x)
    u, v = x[..., a], x[..., b]
    want[..., a], want[..., b] = u * c - v * s, v * c + u * s
    far[..., a] = far[..., b] = (np.abs(u) + np.abs(v)) * factor * 4 * 2.0 ** -24
    far[..., :2 * half] += np.abs(want[..., :2 * half]) * U16 + 2.0 ** -25
    return want, far


def attention(q, k, v, past, scale):
    """Rows q [R, Hq, dim] at positions past + i over keys and values [L, Hkv,
    dim] in 64 bits, and how far fp16 outputs may be from them: half a step of
    fp16; the weights rounded to fp16 in the sum and in its denominator (2
    half steps of sum p |v|); the scores in fp32 (dim products and sums, a half
    step of sum |q k| scale each, in the exponent of both); sums of fp32 over
    the keys and the exponential (2^-21)."""
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    out, far = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim))
    for i in range(rows):
        n = past + i + 1
        for h in range(heads):
            kk, vv = k[:n, h // group], v[:n, h // group]
            x = kk @ q[i, h] * scale
            w = np.exp(x - x.max())
            w /= w.sum()
            out[i, h] = w @ vv
            most = (np.abs(kk) @ np.abs(q[i, h])).max() * abs(scale)
            each = 2 * U16 + 2 * (dim + 8) * 2.0 ** -24 * most + (n + 64) * 2.0 ** -24 + 2.0 ** -21
            far[i, h] = np.abs(out[i, h]) * U16 + 2.0 ** -25 + each * (w @ np.abs(vv))
            far[i, h] += 2.0 ** -32 * (np.abs(vv).sum(0) + n * np.abs(out[i, h]))
    return out, far


def frequencies(rotary, theta, scaling, scale=1.0, original=32768.0, low=1.0, high=32.0):
    out = []
    for i in range(rotary // 2):
        f = theta ** (-2.0 * i / rotary)
        if scaling == "linear":
            f /= scale
        elif scaling == "ntk" and rotary > 2:
            f = (theta * scale ** (rotary / (rotary - 2.0))) ** (-2.0 * i / rotary)
        elif scaling in ("yarn", "bands"):
            keep = min(1.0, max(0.0, (original * f / (2 * math.pi) - low) / (high - low)))
            f = keep * f + (1 - keep) * f / scale
        out.append(f)
    return np.array(out), 0.1 * math.log(scale) + 1 if scaling == "yarn" and scale > 1 else 1.0

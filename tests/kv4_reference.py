"""Plain restatements for 4-bit pages and normed heads, on the CPU, for the tests: codes and scales
from their definition by exhaustive comparison, and norms in the f32 steps their definition names."""
import numpy as np
import torch

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def quantize(x):
    """f32 rows [..., dim] as codes uint8 [..., dim / 2] and exponents uint8 [..., dim / 32]."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore"):
        top = np.abs(g).max(-1)
    bad = ~np.isfinite(g).all(-1)
    e = np.full(top.shape, 1, np.int64)
    for n in range(254, 0, -1):  # the least one that is large enough
        e = np.where(top <= 7 * 2.0 ** (n - 127), n, e)
    y = np.where(bad[..., None], 0.0, g) / 2.0 ** (e[..., None] - 127.0)
    d = np.abs(np.abs(y)[..., None] - VALUES)  # exact: y has 24 bits
    near = d.min(-1, keepdims=True)
    even = np.where(d == near, np.arange(8) % 2, 2)  # ties go to the even code
    code = even.argmin(-1) + 8 * np.signbit(y)
    code = code.reshape(*x.shape).astype(np.uint8)
    return (torch.from_numpy(code[..., 0::2] | (code[..., 1::2] << 4)),
            torch.from_numpy(np.where(bad, 255, e).astype(np.uint8)))


def values64(codes, exponents):
    c, e = codes.numpy(), exponents.numpy().astype(np.float64)
    c = np.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], -1)
    v = np.where(c & 8, -1.0, 1.0) * VALUES[c & 7]
    s = np.where(e == 255, np.nan, 2.0 ** (e - 127))
    return v * np.repeat(s, 32, -1)


def make_pages(num_pages, heads, page, dim, rng, spread=1.0):
    x = rng.normal(0, spread, size=(num_pages, heads, page, dim)).astype(np.float32)
    return quantize(x * np.exp(rng.normal(0, 1, size=(num_pages, heads, page, 1))).astype(np.float32))


def typed(codes, exponents):
    return codes.view(torch.float4_e2m1fn_x2), exponents.view(torch.float8_e8m0fnu)


def norm(x, weight, eps):
    """x [T, heads, D] of any type as f32: x * r * weight, r = f32(1 / sqrt(mean + eps)) from 64 bits."""
    x = x.to(torch.float32).numpy()
    if weight is None:
        return x
    with np.errstate(divide="ignore", invalid="ignore"):
        r = (1.0 / np.sqrt((x.astype(np.float64) ** 2).sum(-1, keepdims=True) / x.shape[-1] + eps)).astype(np.float32)
        return x * r * weight.to(torch.float32).numpy()

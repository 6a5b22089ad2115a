"""Plain 64-bit forms of the linear-layer operators, and their tolerances.

Tolerances, derived from the arithmetic: a product's fp32 sum of K terms is
off by at most K roundings of 2^-23 (the tensor core may truncate) of the sum
of the terms' magnitudes, ``sum_err``; an activation's slope is below 1.13, and
its own fp32 evaluation is off by at most 2^-18 of (|z| + 1); the bf16 output
adds half a step, 2^-8 of the value (values here are far from bf16's
subnormals).
"""

import math

import numpy as np

from oracle import oracle

BF16 = 2.0 ** -8  # torch.finfo(bfloat16).eps / 2
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
_erf = np.vectorize(math.erf, otypes=[np.float64])


def act(z, name):
    if name == "relu":
        return np.maximum(z, 0.0)
    if name == "gelu":
        return 0.5 * z * (1 + _erf(z / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + np.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z / (1 + np.exp(-z))
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).astype(np.float64)
    if name == "gelu":
        return 0.5 * (1 + _erf(z / math.sqrt(2))) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = np.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        p = 1 / (1 + np.exp(-z))
        return p * (1 + z * (1 - p))
    return np.ones_like(z)


def bits(rng, *shape, std=1.0):
    """N(0, std^2) values rounded to bf16, as raw bits."""
    return oracle.f32_to_bf16_bits(rng.standard_normal(shape, dtype=np.float32) * np.float32(std))


def wide(b):
    return oracle.bf16_bits_to_f32(b).astype(np.float64)


def product(a, b):
    """(a @ b, bound on the error of its fp32 sum)."""
    k = a.shape[-1]
    return a @ b, k * 2.0 ** -23 * (np.abs(a) @ np.abs(b))


def close(got_bits, want, err, what):
    """bf16 ``got_bits`` within half a step and ``err`` of ``want``."""
    got = wide(got_bits)
    tol = BF16 * np.abs(want) + (1 + BF16) * err
    off = np.abs(got - want)
    assert np.isfinite(got).all(), f"{what}: not finite"
    worst = np.unravel_index(np.argmax(off - tol), off.shape)
    assert (off <= tol).all(), (f"{what}: {int((off > tol).sum())} of {off.size} off, worst at {worst}: "
                                f"got {got[worst]}, want {want[worst]} +- {tol[worst]}")


def act_err(z, z_err):
    return 1.13 * z_err + 2.0 ** -18 * (np.abs(z) + 1)


def slope_err(z):
    return 2.0 ** -18 * (np.abs(z) + 1) ** 2


def sizes_to_offsets(sizes, first=0):
    return (first + np.concatenate([[0], np.cumsum(sizes)])).astype(np.int32)

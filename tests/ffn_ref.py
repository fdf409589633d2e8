"""Plain 64-bit forms of the feed-forward operators on the host, with the error each stage of the kernels may make.

Everything is row-major with a row per token / channel: x [n, k], w [rows, k], p [n, 2m], c [n, m].
Unit roundoffs are half a step: float 2^-24, half 2^-11, bfloat16 2^-8 relative, and half the smallest subnormal
where a half result is subnormal.
"""
import math

import numpy as np
from scipy.special import erfc

U32 = 2.0 ** -24
UNIT = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
# half the spacing of the type's subnormals (float32 / bfloat16: far below anything here, but the sums of tiny
# products can meet it)
SUBNORMAL = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}
ACTS = ("silu", "gelu", "gelu_tanh", "relu")


def to_bits(x, dtype):
    """float array -> (storage array, the values it holds as float64)."""
    if dtype == "float32":
        s = np.ascontiguousarray(x, dtype=np.float32)
        return s, s.astype(np.float64)
    if dtype == "float16":
        with np.errstate(over="ignore"):
            s = np.ascontiguousarray(x).astype(np.float16)
        return s.view(np.uint16), s.astype(np.float64)
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    s = ((u + np.uint32(0x7FFF) + ((u >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)
    return s, from_bits(s, dtype)


def overflows(got, truth, bound, dtype):
    """Where an infinite result is right: half has nothing between 65504 and infinity, and rounding to nearest gives
    infinity from 65520 on, so a float value of at least 65520 that the bound allows may have become one."""
    if dtype != "float16":
        return np.zeros(got.shape, bool)
    return np.isinf(got) & (np.sign(got) == np.sign(truth)) & (np.abs(truth) + bound >= 65520.0)


def from_bits(s, dtype):
    if dtype == "bfloat16":
        return (s.astype(np.uint32) << np.uint32(16)).view(np.float32).astype(np.float64)
    if dtype == "float16":
        return s.view(np.float16).astype(np.float64)
    return s.astype(np.float64)


def act(g, kind):
    with np.errstate(over="ignore"):
        return _act(g, kind)


def _act(g, kind):
    if kind == "silu":
        return g / (1.0 + np.exp(-g))
    if kind == "gelu":
        return 0.5 * g * erfc(-g / math.sqrt(2.0))
    if kind == "gelu_tanh":
        return g / (1.0 + np.exp(-2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)))
    return np.maximum(g, 0.0)


def slope(g, kind):
    if kind == "silu":
        s = 1.0 / (1.0 + np.exp(-g))
        return s + g * s * (1.0 - s)
    if kind == "gelu":
        return 0.5 * erfc(-g / math.sqrt(2.0)) + g * np.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    if kind == "gelu_tanh":
        z = 2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)
        s = 1.0 / (1.0 + np.exp(-z))
        return s + g * s * (1.0 - s) * 2.0 * math.sqrt(2.0 / math.pi) * (1.0 + 3.0 * 0.044715 * g * g)
    return (g > 0).astype(np.float64)


def steep(g, kind):
    """How much a relative error of the exponential's argument is magnified: |argument| (and its own terms)."""
    if kind == "silu":
        return np.abs(g)
    if kind == "gelu":
        return g * g
    if kind == "gelu_tanh":
        return 2.0 * math.sqrt(2.0 / math.pi) * (np.abs(g) + 0.044715 * np.abs(g) ** 3)
    return np.zeros_like(g)


def act_error(g, kind):
    """Bound of |float act(g) - act(g)| for an exact g.  A handful of roundings of 2^-23 (the hardware's 2^x and
    reciprocal are good to one unit in the last place, the polynomial behind Phi to 4e-7), and the argument's own
    roundings (at most 6 of them) times the magnification.  The reciprocal and the exponential have no subnormal results: a
    factor below 2^-126 becomes 0, and act(g), g times that factor, is then off by up to |g| 2^-126."""
    if kind == "relu":
        return np.zeros_like(g)
    return np.abs(act(g, kind)) * (20.0 + 6.0 * steep(g, kind)) * 2.0 ** -23 + (1.0 + np.abs(g)) * 2.0 ** -126


def slope_error(g, kind):
    """The same for act'(g): every term is at most 1.2 in size where it is not negligible, except that g s (1 - s) z' is
    a product of rounded factors whose s (1 - s) carries an absolute error of 2^-22 times |g z'| <= 20 (beyond |z| of 17
    it vanishes), hence the 100."""
    if kind == "relu":
        return np.zeros_like(g)
    return (100.0 + 12.0 * np.minimum(steep(g, kind), 20.0)) * 2.0 ** -23


def product_error(x, w, k):
    """Bound of a float sum of exact products in any order, k terms: (k + 2) 2^-24 sum |x||w|."""
    return (k + 2) * U32 * (np.abs(x) @ np.abs(w).T)


def rounded(truth, error, dtype):
    """The stored result's bound: the float value's error and one rounding to the type."""
    return error + (np.abs(truth) + error) * UNIT[dtype] + SUBNORMAL[dtype]


def gated(p, p_err, m, kind, dtype):
    """(truth, bound) of act(G) U.  |act'| <= 1.2 for all four, so an error e of G moves act(G) by at most 1.2 e."""
    g, u, eg, eu = p[:, :m], p[:, m:], p_err[:, :m], p_err[:, m:]
    a = act(g, kind)
    ea = 1.2 * eg + act_error(g, kind) + 1.2 * eg * (20.0 + 6.0 * steep(np.abs(g) + eg, kind)) * 2.0 ** -23
    truth = a * u
    err = np.abs(u) * ea + (np.abs(a) + ea) * eu
    err = err + (np.abs(truth) + err) * 2.0 * U32
    return truth, rounded(truth, err, dtype)


def gate_grad(p, dh, m, kind, dtype):
    """(truth, bound) of dP from the stored P and dC."""
    g, u = p[:, :m], p[:, m:]
    s, a = slope(g, kind), act(g, kind)
    dg, du = dh * u * s, dh * a
    eg = np.abs(dh * u) * slope_error(g, kind) + np.abs(dg) * 3.0 * U32
    eu = np.abs(dh) * act_error(g, kind) + np.abs(du) * 2.0 * U32
    truth, err = np.concatenate([dg, du], 1), np.concatenate([eg, eu], 1)
    return truth, rounded(truth, err, dtype)


def quantized(x):
    """Exact quantisation of the rows of x (float64 holding float, half or bfloat16 values): 127 x and the quotient's distance
    from a tie are exact or far above double's rounding, so np.rint (ties to even) of the double quotient is the exact
    answer."""
    largest = np.abs(x).max(axis=1, initial=0.0)
    usable = np.isfinite(largest) & (largest > 0)  # a row of zeros, or with a NaN or an infinity, is all zeros
    q = np.rint(127.0 * np.where(usable[:, None], x, 0.0) / np.where(usable, largest, 1.0)[:, None])
    return q.astype(np.int8), (largest.astype(np.float32) / np.float32(127.0)).astype(np.float32)

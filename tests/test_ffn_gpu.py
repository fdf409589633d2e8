"""GPU tests of the feed-forward operators (include/sbamd_ffn.h) through the Python interface: quantisation, scaled 8-bit
product, gated block in 16 and 8 bits, its gradient, and whole layers made of them.

Every result is compared element by element with the plain 64-bit form of tests/ffn_ref.py inside a bound derived there
from the roundings the kernels make; memory around every output has to stay as it was.
"""
import ctypes as C
import itertools
import math

import numpy as np
import pytest

import sycl_blas_amd as sb
from sycl_blas_amd import _lib, activation_t, helper

import ffn_ref as ref
from common import seeded

pytestmark = pytest.mark.gpu

# kernels to pin: chosen by itself, narrow, 128 x 128 ring, 256 x 256 ring
AUTO, NARROW, RING128, RING256 = (_lib.KERNEL_AUTO,), (_lib.KERNEL_SMALL,), (_lib.KERNEL_LARGE,), (_lib.KERNEL_HUGE,)
FAMILIES = {"narrow": NARROW, "ring128": RING128, "ring256": RING256}
# tiles whole, ragged in one or both directions, smaller than a tile; k of one step, whole steps, with a tail, shorter than a step, odd
FAMILY_SHAPES = [(256, 256, 64), (300, 130, 96), (5, 300, 1000), (520, 70, 40), (129, 257, 31), (257, 513, 333), (64, 1, 2050), (1, 640, 192)]

GUARD = 64  # elements in front of and behind every device matrix
STORE = {"float32": np.float32, "float16": np.uint16, "bfloat16": np.uint16, "int8": np.int8}
FILL = {"float32": np.float32(-12345.0), "float16": np.uint16(0x7BCD), "bfloat16": np.uint16(0x7BCD), "int8": np.int8(-77)}


class Mat:
    """A [rows, cols] row-major matrix on the device with `ld` elements per row, `shift` elements off the allocation's
    alignment, and guard values wherever the matrix is not."""

    def __init__(self, h, dtype, rows, cols, ld=None, shift=0, values=None):
        self.h, self.dtype, self.rows, self.cols = h, dtype, rows, cols
        self.ld = cols if ld is None else ld
        self.start = GUARD + shift
        self.host = np.full(self.start + max(rows, 1) * max(self.ld, 1) + GUARD, FILL[dtype], dtype=STORE[dtype])
        if values is not None:
            self.window(self.host)[...] = values
        self.alloc = helper.allocate(h, dtype, self.host.size)
        h.wait(helper.copy_to_device(h, self.host, self.alloc))
        self.buf = self.alloc + self.start

    def window(self, flat):
        return np.lib.stride_tricks.as_strided(flat[self.start:], (self.rows, self.cols), (self.ld * flat.itemsize, flat.itemsize))

    def get(self):
        """The matrix as stored, after checking that nothing around it changed."""
        out = np.empty_like(self.host)
        self.h.wait(helper.copy_to_host(self.h, self.alloc, out))
        values = self.window(out).copy()
        self.window(out)[...] = self.window(self.host)
        assert (out.view(np.uint8) == self.host.view(np.uint8)).all(), "memory around the matrix was written"
        return values


def vec(h, values):
    return Mat(h, "float32", 1, len(values), values=np.asarray(values, np.float32)[None, :])


def close(got, truth, bound, what, dtype="float32"):
    with np.errstate(invalid="ignore"):
        bad = ~((np.abs(got - truth) <= bound) | ref.overflows(got, truth, bound, dtype))
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, np.abs(got - truth) / bound, 0)), got.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} beyond the bound, worst at {at}: got {got[at]!r}, "
                             f"exact {truth[at]!r}, allowed {bound[at]!r}")


@pytest.fixture()
def h(sb_handle):
    sb_handle.set_kernel(_lib.KERNEL_AUTO)
    yield sb_handle
    sb_handle.set_kernel(_lib.KERNEL_AUTO)


# ------------------------------------------------------------------- quantise
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,m,pad,shift", [(1, 1, 0, 0), (3, 7, 1, 1), (5, 8, 0, 0), (9, 511, 2, 3), (2, 512, 0, 0), (3, 513, 0, 1),
                                           (4, 4096, 0, 0), (3, 4100, 5, 0), (2, 16384, 0, 0), (2, 16391, 1, 2), (3, 40003, 0, 0),
                                           (1000, 64, 0, 0), (257, 130, 6, 1)])
def test_quantize(h, dtype, n, m, pad, shift):
    rng = seeded("quantize", dtype, n, m, pad, shift)
    x = rng.standard_normal((n, m)) * np.exp(3.0 * rng.standard_normal((n, 1)))
    bits, x = ref.to_bits(x, dtype)
    xg = Mat(h, dtype, n, m, m + pad, shift, bits)
    qg = Mat(h, "int8", n, m, m + 2 * pad, shift)
    sg = Mat(h, "float32", 1, n)
    h.wait(sb._quantize(h, m, n, xg.buf, xg.ld, qg.buf, qg.ld, sg.buf))
    q, scale = ref.quantized(x)
    assert (sg.get()[0] == scale).all()
    assert (qg.get() == q).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("m", [40, 700, 9000])
def test_quantize_ties_and_extremes(h, dtype, m):
    """Ties (largest 254 steps: every odd multiple of half a step is one), zeros, subnormals, the largest values, and
    rows with a NaN or an infinity."""
    rng = seeded("quantize ties", dtype, m)
    big = {"float32": 3.4028234663852886e38, "float16": 65504.0, "bfloat16": 3.3895313892515355e38}[dtype]
    small = {"float32": 1e-45, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -133}[dtype]
    rows = [
        np.concatenate([[127.0], (rng.integers(-127, 127, m - 1) + 0.5)]),  # ties: 127 x / 127 is an odd half
        np.concatenate([[-254.0], rng.integers(-127, 128, m - 1)]),         # ties again, half of the integers
        np.zeros(m),
        np.full(m, -0.0),
        np.concatenate([[small], np.zeros(m - 1)]),
        rng.integers(-3, 4, m) * small,
        rng.choice([big, -big, big / 2, 0.0], m),
        np.concatenate([[big], rng.standard_normal(m - 1)]),
    ]
    x = np.stack(rows)
    bits, x = ref.to_bits(x, dtype)
    q, scale = ref.quantized(x)
    odd = np.repeat(bits[:1], 3, axis=0).copy()
    nan, inf = {"float32": (np.nan, np.inf), "float16": (0x7E00, 0x7C00), "bfloat16": (0x7FC0, 0x7F80)}[dtype]
    odd[0, m - 1], odd[1, m // 2], odd[2, 0], odd[2, m - 1] = nan, inf, inf, nan
    xg = Mat(h, dtype, len(rows) + 3, m, values=np.concatenate([bits, odd]))
    qg, sg = Mat(h, "int8", len(rows) + 3, m), Mat(h, "float32", 1, len(rows) + 3)
    h.wait(sb._quantize(h, m, len(rows) + 3, xg.buf, m, qg.buf, m, sg.buf))
    got_q, got_s = qg.get(), sg.get()[0]
    assert (got_s[: len(rows)] == scale).all()
    assert (got_q[: len(rows)] == q).all()
    assert (got_q[len(rows):] == 0).all()
    assert np.isnan(got_s[len(rows)]) and np.isinf(got_s[len(rows) + 1]) and np.isnan(got_s[len(rows) + 2])


def test_quantize_of_nothing(h):
    sg, qg = Mat(h, "float32", 1, 5), Mat(h, "int8", 1, 1)
    h.wait(sb._quantize(h, 0, 5, sg.buf, 0, qg.buf, 0, sg.buf))
    assert (sg.get() == 0).all()
    before = Mat(h, "float32", 1, 5)
    h.wait(sb._quantize(h, 7, 0, before.buf, 7, qg.buf, 7, before.buf))
    assert (before.get() == FILL["float32"]).all()


# ------------------------------------------------------------- scaled product
def int8_operands(rng, n, rows, k):
    return rng.integers(-128, 128, (n, k)).astype(np.int8), rng.integers(-128, 128, (rows, k)).astype(np.int8)


def across(a):
    return np.ascontiguousarray(a.T)


def run_scaled(h, out, n, m, k, ta="t", tb="n", alpha=1.0, beta=0.0, pad=0, shift=0, scales="both", family=AUTO):
    rng = seeded("scaled", out, n, m, k, ta, tb, alpha, beta, pad, shift, scales)
    x, w = int8_operands(rng, n, m, k)
    sx = np.exp(rng.standard_normal(n)).astype(np.float32) if scales != "none" else None
    sw = np.exp(rng.standard_normal(m)).astype(np.float32) if scales == "both" else None
    c_bits, c0 = ref.to_bits(rng.standard_normal((n, m)), out)
    wg = Mat(h, "int8", m, k, k + pad, shift, w) if ta == "t" else Mat(h, "int8", k, m, m + pad, shift, across(w))
    xg = Mat(h, "int8", n, k, k + pad, shift, x) if tb == "n" else Mat(h, "int8", k, n, n + pad, shift, across(x))
    cg = Mat(h, out, n, m, m + pad, shift, c_bits)
    sxg, swg = (None if s is None else vec(h, s) for s in (sx, sw))
    h.set_kernel(*family)
    h.wait(sb._gemm_scaled(h, ta, tb, m, n, k, alpha, wg.buf, wg.ld, swg and swg.buf, xg.buf, xg.ld, sxg and sxg.buf, beta, cg.buf,
                           cg.ld))
    s = (x.astype(np.int64) @ w.astype(np.int64).T).astype(np.float64)
    scaled = s * (1.0 if sx is None else sx.astype(np.float64)[:, None]) * (1.0 if sw is None else sw.astype(np.float64)[None, :])
    alpha32, beta32 = float(np.float32(alpha)), float(np.float32(beta))
    truth = alpha32 * scaled + (beta32 * c0 if beta else 0.0)
    # sum to float, two scales, alpha: four roundings; beta * C and the addition: two more
    err = 4.5 * ref.U32 * np.abs(alpha32 * scaled) + ref.U32 * (np.abs(beta32 * c0) + np.abs(truth)) * 1.1 * (beta != 0)
    close(ref.from_bits(cg.get(), out), truth, ref.rounded(truth, err, out),
          f"scaled {out} n={n} m={m} k={k} {ta}{tb} alpha={alpha} beta={beta} pad={pad} shift={shift} {scales}", out)


@pytest.mark.parametrize("out", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,m,k", [(1, 1, 1), (1, 33, 5), (2, 32, 16), (15, 31, 127), (16, 64, 128), (17, 65, 129), (32, 100, 512),
                                   (33, 257, 1000), (64, 16, 640), (65, 48, 1153), (130, 70, 2048), (300, 513, 333)])
def test_scaled_sizes(h, out, n, m, k):
    run_scaled(h, out, n, m, k)


@pytest.mark.parametrize("family", FAMILIES)
@pytest.mark.parametrize("n,m,k", FAMILY_SHAPES)
def test_scaled_families(h, family, n, m, k):
    for out, pad in (("float32", 0), ("bfloat16", 16), ("float16", 5)):
        run_scaled(h, out, n, m, k, beta=0.5 if pad else 0.0, pad=pad, family=FAMILIES[family])
        assert h.last_kernel() == FAMILIES[family][0]


@pytest.mark.parametrize("family", ["ring128", "ring256"])
@pytest.mark.parametrize("n,m,k", [(300, 500, 4096), (130, 129, 5000), (70, 1030, 3333)])
def test_scaled_cut_along_k(h, family, n, m, k):
    """Few tiles and a long k: the tiles are cut along k and joined; whatever the cut, the integer sum is the same."""
    for out, pad, beta in (("float32", 0, 0.0), ("bfloat16", 0, 0.5), ("float16", 3, 0.0), ("float32", 16, -1.5)):
        run_scaled(h, out, n, m, k, alpha=0.01, beta=beta, pad=pad, family=FAMILIES[family])
        assert h.last_splitk()[0] > 1


@pytest.mark.parametrize("ta,tb", [("t", "n"), ("n", "n"), ("t", "t"), ("n", "t")])
@pytest.mark.parametrize("n,m,k,pad,shift", [(5, 40, 70, 0, 0), (40, 90, 200, 3, 1), (129, 260, 96, 16, 0), (150, 300, 257, 1, 7)])
def test_scaled_layouts(h, ta, tb, n, m, k, pad, shift):
    run_scaled(h, "float32", n, m, k, ta, tb, 0.75, 1.25, pad, shift)


@pytest.mark.parametrize("alpha,beta", [(1.0, 1.0), (-2.5, 0.0), (0.3, -0.7)])
@pytest.mark.parametrize("scales", ["both", "tokens", "none"])
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
def test_scaled_alpha_beta_scales(h, out, alpha, beta, scales):
    run_scaled(h, out, 19, 75, 144, alpha=alpha, beta=beta, scales=scales)


@pytest.mark.parametrize("n", [3, 200])
def test_scaled_k_zero_and_alpha_zero(h, n):
    m = 37
    rng = seeded("scaled zero", n)
    values = rng.standard_normal((n, m)).astype(np.float32)
    one = Mat(h, "int8", 1, 1)
    for beta, k, alpha in ((0.0, 0, 1.0), (2.0, 0, 1.0), (0.5, 9, 0.0), (0.0, 9, 0.0), (1.0, 9, 0.0)):
        start = values if beta else np.full_like(values, np.nan)
        for ta, lda, tb, ldb in (("t", k, "n", k), ("n", m, "t", n)):
            cg = Mat(h, "float32", n, m, m + 3, 0, start)
            h.wait(sb._gemm_scaled(h, ta, tb, m, n, k, alpha, one.buf, lda, None, one.buf, ldb, None, beta, cg.buf, cg.ld))
            assert (cg.get() == np.float32(beta) * values).all(), (beta, k, alpha, ta, tb)


def test_scaled_largest_sums_are_exact(h):
    """k at its limit with all products 16384 and all -16256: the sums reach 2^31 - 2^14 and do not wrap."""
    k, n, m = _lib.I8_MAX_K, 2, 3
    x = np.full((n, k), -128, np.int8)
    w = np.stack([np.full(k, -128, np.int8), np.full(k, 127, np.int8), np.zeros(k, np.int8)])
    xg, wg, cg = Mat(h, "int8", n, k, values=x), Mat(h, "int8", m, k, values=w), Mat(h, "float32", n, m)
    h.wait(sb._gemm_scaled(h, "t", "n", m, n, k, 1.0, wg.buf, k, None, xg.buf, k, None, 0.0, cg.buf, m))
    s = x.astype(np.int64) @ w.astype(np.int64).T
    assert s.max() == k * 16384 < 2 ** 31
    assert (cg.get() == s.astype(np.float32)).all()
    with pytest.raises(NotImplementedError):
        sb._gemm_scaled(h, "t", "n", m, n, k + 1, 1.0, wg.buf, k + 1, None, xg.buf, k + 1, None, 0.0, cg.buf, m)


def test_scaled_poisoned_columns_and_tiny_scales(h):
    """A NaN or infinite scale makes its token NaN and no other; scales whose product underflows do not lose the sum."""
    n, m, k = 6, 50, 64
    rng = seeded("poison")
    x, w = int8_operands(rng, n, m, k)
    x[2] = 0
    x[3] = 0
    sx = np.array([1.0, 1e-30, np.nan, np.inf, 1.0, 0.0], np.float32)
    sw = np.full(m, 1e-20, np.float32)
    xg, wg, cg = Mat(h, "int8", n, k, values=x), Mat(h, "int8", m, k, values=w), Mat(h, "float32", n, m)
    h.wait(sb._gemm_scaled(h, "t", "n", m, n, k, 1e25, wg.buf, k, vec(h, sw).buf, xg.buf, k, vec(h, sx).buf, 0.0, cg.buf, m))
    got = cg.get().astype(np.float64)
    s = (x.astype(np.int64) @ w.astype(np.int64).T).astype(np.float64)
    assert np.isnan(got[2]).all() and np.isnan(got[3]).all() and (got[5] == 0).all()
    for row in (0, 4):
        truth = s[row] * 1e-20 * 1e25
        assert (np.abs(got[row] - truth) <= np.abs(truth) * 6 * ref.U32 + 1e-300).all()


# ---------------------------------------------------------------- gated block
def run_gated(h, dtype, n, m, k, kind, ta="t", tb="n", keep=False, pad=0, shift=0, family=AUTO, size=1.0):
    rng = seeded("gated", dtype, n, m, k, kind, ta, tb, keep, pad, shift)
    xb, x = ref.to_bits(rng.standard_normal((n, k)) * size, dtype)
    wb, w = ref.to_bits(rng.standard_normal((2 * m, k)) * (2.0 / math.sqrt(max(k, 1))), dtype)
    wg = Mat(h, dtype, 2 * m, k, k + pad, shift, wb) if ta == "t" else Mat(h, dtype, k, 2 * m, 2 * m + pad, shift, across(wb))
    xg = Mat(h, dtype, n, k, k + pad, shift, xb) if tb == "n" else Mat(h, dtype, k, n, n + pad, shift, across(xb))
    cg = Mat(h, dtype, n, m, m + pad, shift)
    pg = Mat(h, dtype, n, 2 * m, 2 * m + pad, shift) if keep else None
    h.set_kernel(*family)
    args = (pg.buf, pg.ld) if keep else ()
    h.wait(sb._gated_gemm(h, activation_t[kind], ta, tb, m, n, k, wg.buf, wg.ld, xg.buf, xg.ld, cg.buf, cg.ld, *args))
    p, p_err = x @ w.T, ref.product_error(x, w, k)
    what = f"gated {dtype} {kind} n={n} m={m} k={k} {ta}{tb} pad={pad} shift={shift}"
    truth, bound = ref.gated(p, p_err, m, kind, dtype)
    close(ref.from_bits(cg.get(), dtype), truth, bound, what, dtype)
    if keep:
        close(ref.from_bits(pg.get(), dtype), p, ref.rounded(p, p_err, dtype), what + " P", dtype)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,m,k", [(1, 1, 1), (1, 17, 70), (2, 16, 32), (15, 15, 64), (16, 40, 96), (17, 100, 130), (31, 33, 512),
                                   (48, 64, 1024), (65, 129, 77), (130, 257, 300), (256, 128, 64), (257, 130, 200)])
def test_gated_sizes(h, dtype, n, m, k):
    run_gated(h, dtype, n, m, k, "silu", keep=(n + m) % 2 == 0)


@pytest.mark.parametrize("family", FAMILIES)
@pytest.mark.parametrize("n,m,k", FAMILY_SHAPES)
@pytest.mark.parametrize("ta,tb", [("t", "n"), ("n", "n"), ("t", "t"), ("n", "t")])
def test_gated_families(h, family, n, m, k, ta, tb):
    """Every kernel on every layout: m a multiple of 8 or not decides whether an operand across k is read in place."""
    for dtype, pad, keep in (("bfloat16", 0, True), ("float16", 8, False), ("bfloat16", 3, True)):
        run_gated(h, dtype, n, m, k, "silu", ta, tb, keep, pad, family=FAMILIES[family])


@pytest.mark.parametrize("kind", ref.ACTS)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n", [6, 140])
def test_gated_activations(h, dtype, kind, n):
    run_gated(h, dtype, n, 70, 96, kind, size=3.0)


@pytest.mark.parametrize("ta,tb", [("t", "n"), ("n", "n"), ("t", "t"), ("n", "c")])
@pytest.mark.parametrize("n,m,k,pad,shift", [(5, 40, 70, 0, 0), (40, 96, 200, 3, 1), (136, 264, 96, 8, 0), (150, 300, 257, 1, 5)])
def test_gated_layouts(h, ta, tb, n, m, k, pad, shift):
    run_gated(h, "bfloat16", n, m, k, "gelu_tanh", ta, tb, True, pad, shift)


@pytest.mark.parametrize("n", [3, 150])
def test_gated_k_zero(h, n):
    """A sum over nothing is 0, and so is act(0) * 0, whatever the buffers held."""
    m = 21
    cg, pg, one = Mat(h, "float16", n, m), Mat(h, "float16", n, 2 * m), Mat(h, "float16", 1, 1)
    h.wait(sb._gated_gemm(h, activation_t.silu, "t", "n", m, n, 0, one.buf, 0, one.buf, 0, cg.buf, m, pg.buf, 2 * m))
    assert (ref.from_bits(cg.get(), "float16") == 0).all() and (ref.from_bits(pg.get(), "float16") == 0).all()


@pytest.mark.parametrize("n", [2, 140])
def test_gated_keeps_nan_and_infinity_in_their_token(h, n):
    m, k = 36, 80
    rng = seeded("gated nan", n)
    xb, x = ref.to_bits(rng.standard_normal((n, k)), "bfloat16")
    wb, w = ref.to_bits(rng.standard_normal((2 * m, k)), "bfloat16")
    xb[n - 1, k - 1] = 0x7FC0  # NaN
    xg, wg, cg = Mat(h, "bfloat16", n, k, values=xb), Mat(h, "bfloat16", 2 * m, k, values=wb), Mat(h, "bfloat16", n, m)
    for kind in ref.ACTS:
        h.wait(sb._gated_gemm(h, activation_t[kind], "t", "n", m, n, k, wg.buf, k, xg.buf, k, cg.buf, m))
        got = ref.from_bits(cg.get(), "bfloat16")
        assert np.isnan(got[n - 1]).all() and np.isfinite(got[: n - 1]).all(), kind


def run_gated_scaled(h, out, n, m, k, kind, ta="t", tb="n", pad=0, shift=0, scales=True, family=AUTO):
    rng = seeded("gated scaled", out, n, m, k, kind, ta, tb, pad, shift, scales)
    x, w = int8_operands(rng, n, 2 * m, k)
    sx = (np.exp(0.5 * rng.standard_normal(n)) / 75.0).astype(np.float32)
    sw = (np.exp(0.5 * rng.standard_normal(2 * m)) / (75.0 * math.sqrt(max(k, 1)))).astype(np.float32)
    if not scales:
        sx = (sx * 0 + 2.0 ** -14).astype(np.float32)
    wg = Mat(h, "int8", 2 * m, k, k + pad, shift, w) if ta == "t" else Mat(h, "int8", k, 2 * m, 2 * m + pad, shift, across(w))
    xg = Mat(h, "int8", n, k, k + pad, shift, x) if tb == "n" else Mat(h, "int8", k, n, n + pad, shift, across(x))
    cg = Mat(h, out, n, m, m + pad, shift)
    swg, sxg = vec(h, sw) if scales else None, vec(h, sx)
    h.set_kernel(*family)
    h.wait(sb._gated_gemm_scaled(h, activation_t[kind], ta, tb, m, n, k, wg.buf, wg.ld, swg and swg.buf, xg.buf, xg.ld, sxg.buf,
                                 cg.buf, cg.ld))
    s = (x.astype(np.int64) @ w.astype(np.int64).T).astype(np.float64)
    p = s * sx.astype(np.float64)[:, None] * (sw.astype(np.float64)[None, :] if scales else 1.0)
    truth, bound = ref.gated(p, 3.5 * ref.U32 * np.abs(p), m, kind, out)
    close(ref.from_bits(cg.get(), out), truth, bound, f"gated i8 {out} {kind} n={n} m={m} k={k} {ta}{tb} pad={pad} shift={shift}", out)


@pytest.mark.parametrize("out", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,m,k", [(1, 1, 3), (1, 40, 256), (16, 17, 127), (33, 64, 130), (64, 100, 1000), (130, 257, 512), (300, 70, 64)])
def test_gated_scaled_sizes(h, out, n, m, k):
    run_gated_scaled(h, out, n, m, k, "silu")


@pytest.mark.parametrize("family", FAMILIES)
@pytest.mark.parametrize("n,m,k", FAMILY_SHAPES)
def test_gated_scaled_families(h, family, n, m, k):
    for out, pad in (("float32", 0), ("bfloat16", 16), ("float16", 5)):
        run_gated_scaled(h, out, n, m, k, "gelu_tanh", pad=pad, family=FAMILIES[family])


@pytest.mark.parametrize("kind", ref.ACTS)
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
def test_gated_scaled_activations(h, out, kind):
    run_gated_scaled(h, out, 35, 70, 96, kind, scales=kind != "relu")


@pytest.mark.parametrize("kind", ref.ACTS)
def test_activation_over_its_whole_range(h, kind):
    """act(g) in float for g from -12 to 12 and far beyond: k = 1, the gate's sum is an integer and its scale makes g, the other
    half is 1.  Elementwise inside the relative bound, small values far on the negative side included."""
    steps = np.concatenate([np.linspace(-12.0, 12.0, 4001), np.linspace(-60.0, 60.0, 95)]).astype(np.float32)
    m = steps.size
    x, w = np.ones((1, 1), np.int8), np.ones((2 * m, 1), np.int8)
    xg, wg, c = Mat(h, "int8", 1, 1, values=x), Mat(h, "int8", 2 * m, 1, values=w), Mat(h, "float32", 1, m)
    swg = vec(h, np.concatenate([steps, np.ones(m, np.float32)]))
    h.wait(sb._gated_gemm_scaled(h, activation_t[kind], "t", "n", m, 1, 1, wg.buf, 1, swg.buf, xg.buf, 1, None, c.buf, m))
    g = steps.astype(np.float64)[None, :]
    close(c.get().astype(np.float64), ref.act(g, kind), ref.act_error(g, kind) + 2 * ref.U32 * np.abs(ref.act(g, kind)), kind)


@pytest.mark.parametrize("ta,tb", [("t", "n"), ("n", "n"), ("t", "t"), ("n", "t")])
@pytest.mark.parametrize("n,m,k,pad,shift", [(5, 40, 70, 0, 0), (40, 96, 200, 3, 1), (136, 264, 96, 16, 0)])
def test_gated_scaled_layouts(h, ta, tb, n, m, k, pad, shift):
    run_gated_scaled(h, "float16", n, m, k, "gelu", ta, tb, pad, shift)


# ------------------------------------------------------------------- gradient
def run_grad(h, dtype, n, m, k, kind, ta="t", tb="n", pad=0, shift=0, beta_a=0.0, beta_b=0.0, in_place=False, want="ab", family=AUTO,
             pad_w=None, pad_x=None):
    rng = seeded("grad", dtype, n, m, k, kind, ta, tb, pad, shift, beta_a, beta_b, in_place, want)
    xb, x = ref.to_bits(rng.standard_normal((n, k)), dtype)
    wb, w = ref.to_bits(rng.standard_normal((2 * m, k)) / math.sqrt(max(k, 1)), dtype)
    pb, p = ref.to_bits(rng.standard_normal((n, 2 * m)) * 2.0, dtype)
    db, dh = ref.to_bits(rng.standard_normal((n, m)), dtype)
    daw, da0 = ref.to_bits(rng.standard_normal((2 * m, k)), dtype)
    dbx, db0 = ref.to_bits(rng.standard_normal((n, k)), dtype)

    pad_w, pad_x = pad if pad_w is None else pad_w, pad if pad_x is None else pad_x

    def weights(values):
        return Mat(h, dtype, 2 * m, k, k + pad_w, shift, values) if ta == "t" else Mat(h, dtype, k, 2 * m, 2 * m + pad_w, shift, across(values))

    def tokens(values):
        return Mat(h, dtype, n, k, k + pad_x, shift, values) if tb == "n" else Mat(h, dtype, k, n, n + pad_x, shift, across(values))

    wg, xg = weights(wb), tokens(xb)
    pg = Mat(h, dtype, n, 2 * m, 2 * m + pad, shift, pb)
    dcg = Mat(h, dtype, n, m, m + pad, shift, db)
    dpg = pg if in_place else Mat(h, dtype, n, 2 * m, 2 * m + 2 * pad, shift)
    dag = weights(daw) if "a" in want else None
    dbg = tokens(dbx) if "b" in want else None
    h.set_kernel(*family)
    h.wait(sb._gated_gemm_grad(h, activation_t[kind], ta, tb, m, n, k, wg.buf if dbg else None, wg.ld, xg.buf if dag else None, xg.ld,
                               pg.buf, pg.ld, dcg.buf, dcg.ld, dpg.buf, dpg.ld, beta_a, dag and dag.buf, wg.ld, beta_b,
                               dbg and dbg.buf, xg.ld))
    what = f"grad {dtype} {kind} n={n} m={m} k={k} {ta}{tb} pad={pad} shift={shift}"
    dp, dp_bound = ref.gate_grad(p, dh, m, kind, dtype)
    close(ref.from_bits(dpg.get(), dtype), dp, dp_bound, what + " dP", dtype)
    got_a = got_b = None
    for name, out, other, stored, beta, start in (("a", dag, x, ta != "t", beta_a, da0), ("b", dbg, w, tb != "n", beta_b, db0)):
        if out is None:
            continue
        left = dp.T if name == "a" else dp
        bound_left = dp_bound.T if name == "a" else dp_bound
        truth = left @ other
        terms = left.shape[1]
        sums = np.abs(left) @ np.abs(other) + bound_left @ np.abs(other)
        err = bound_left @ np.abs(other) + (terms + 2) * ref.U32 * sums
        if beta:
            truth = truth + beta * start
            err = err + ref.U32 * (2.2 * np.abs(beta * start) + 1.1 * np.abs(truth))
        got = ref.from_bits(out.get(), dtype)
        got = got.T if stored else got
        close(got, truth, ref.rounded(truth, err, dtype), what + f" d{name.upper()} beta={beta}", dtype)
        if name == "a":
            got_a = got
        else:
            got_b = got
    return got_a, got_b


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,m,k", [(1, 1, 1), (1, 9, 40), (7, 8, 16), (16, 33, 65), (40, 100, 72), (129, 64, 128), (300, 130, 96),
                                   (64, 257, 33)])
def test_grad_sizes(h, dtype, n, m, k):
    run_grad(h, dtype, n, m, k, "silu")


@pytest.mark.parametrize("kind", ref.ACTS)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_grad_activations(h, dtype, kind):
    run_grad(h, dtype, 33, 40, 24, kind)


@pytest.mark.parametrize("ta,tb", [("t", "n"), ("n", "n"), ("t", "t"), ("n", "c")])
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (3, 1)])
def test_grad_layouts(h, ta, tb, pad, shift):
    run_grad(h, "bfloat16", 72, 40, 56, "gelu", ta, tb, pad, shift, in_place=pad == 0)


@pytest.mark.parametrize("family", FAMILIES)
@pytest.mark.parametrize("ta,tb", [("t", "n"), ("n", "n"), ("t", "t"), ("n", "t")])
@pytest.mark.parametrize("n,m,k", [(256, 128, 256), (1104, 304, 136), (72, 700, 264), (600, 36, 48), (2500, 20, 40)])
def test_grad_families(h, family, n, m, k, ta, tb):
    """Products on every kernel, with their sums cut along the long side (1104 tokens, 1400 rows of P) and not; 36 and 20
    channels and 2500 tokens leave rows that do not come in whole 16-byte pieces."""
    run_grad(h, "bfloat16", n, m, k, "silu", ta, tb, beta_a=0.5 if m > 100 else 0.0, family=FAMILIES[family])
    run_grad(h, "float16", n, m, k, "gelu_tanh", ta, tb, pad=8, beta_b=1.0 if m > 100 else 0.0, family=FAMILIES[family])


@pytest.mark.parametrize("pad_w,pad_x", [(0, 3), (3, 0), (3, 3)])
@pytest.mark.parametrize("ta,tb", [("t", "n"), ("n", "n"), ("t", "t")])
@pytest.mark.parametrize("n,m,k", [(200, 34, 72), (1104, 302, 136)])
def test_grad_products_share_the_scratch_area(h, n, m, k, ta, tb, pad_w, pad_x):
    """dP's rows are not whole 16-byte pieces, so one product reads a padded copy of it in the handle's scratch area, while
    the other, whose second operand is misaligned, has both of its operands repacked into the same area (parameter bit 0 of the
    16-bit back end asks for that at any size): neither may take the other's place.  Twice, with the area grown the second time."""
    own = sb.SB_Handle(0)
    try:
        for tokens in (n // 2 // 8 * 8, n, n):
            run_grad(own, "bfloat16", tokens, m, k, "silu", ta, tb, family=(_lib.KERNEL_AUTO, 1), pad_w=pad_w, pad_x=pad_x)
    finally:
        own.close()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_grad_accumulates_and_leaves_out(h, dtype):
    run_grad(h, dtype, 50, 24, 40, "silu", beta_a=1.0, beta_b=0.5)
    run_grad(h, dtype, 50, 24, 40, "silu", want="a")
    run_grad(h, dtype, 50, 24, 40, "silu", want="b", in_place=True)
    run_grad(h, dtype, 50, 24, 40, "silu", want="")


@pytest.mark.parametrize("kind", ref.ACTS)
def test_grad_far_out(h, kind):
    """P up to the type's largest values: no NaN where the formula has none (0 * infinity inside the slope), dP = dC * U
    for large gates and 0 for very negative ones."""
    far = np.array([30.0, 200.0, 3e4, 6e4, -30.0, -200.0, -3e4, -6e4, 0.0, -0.0])
    m, n = len(far), 2
    p = np.concatenate([np.tile(far, (n, 1)), np.ones((n, m))], 1)
    pb, p = ref.to_bits(p, "float16")
    db, dh = ref.to_bits(np.full((n, m), 0.5), "float16")
    pg, dcg, dpg = Mat(h, "float16", n, 2 * m, values=pb), Mat(h, "float16", n, m, values=db), Mat(h, "float16", n, 2 * m)
    h.wait(sb._gated_gemm_grad(h, activation_t[kind], "t", "n", m, n, 1, None, 0, None, 0, pg.buf, 2 * m, dcg.buf, m, dpg.buf, 2 * m,
                               0.0, None, 0, 0.0, None, 0))
    got = ref.from_bits(dpg.get(), "float16")
    assert np.isfinite(got).all()
    with np.errstate(over="ignore"):
        dp, bound = ref.gate_grad(p, dh, m, kind, "float16")
    dp, bound = np.nan_to_num(dp), np.nan_to_num(bound, posinf=0.0)
    close(got, dp, bound + 2.0 ** -24, f"far {kind}")


@pytest.mark.parametrize("kind", ref.ACTS)
def test_grad_of_products_beyond_float(h, kind):
    """bfloat16 dC and U whose product no float holds, under slopes that are 0 or small: the infinity must not meet the slope."""
    gates = np.array([-200.0, -40.0, -1e30, 0.0, -60.0, -0.0, 3.0, -25.0])
    m, n = len(gates), 3
    u = np.array([1e20, -3e30, 2e38])[:, None] * np.ones((n, m))
    pb, p = ref.to_bits(np.concatenate([np.tile(gates, (n, 1)), u], 1), "bfloat16")
    db, dh = ref.to_bits(np.array([3e18, 2e20, -1e10])[:, None] * np.ones((n, m)), "bfloat16")
    pg, dcg, dpg = Mat(h, "bfloat16", n, 2 * m, values=pb), Mat(h, "bfloat16", n, m, values=db), Mat(h, "bfloat16", n, 2 * m)
    h.wait(sb._gated_gemm_grad(h, activation_t[kind], "t", "n", m, n, 1, None, 0, None, 0, pg.buf, 2 * m, dcg.buf, m, dpg.buf, 2 * m,
                               0.0, None, 0, 0.0, None, 0))
    got = ref.from_bits(dpg.get(), "bfloat16")
    assert not np.isnan(got).any()
    with np.errstate(all="ignore"):
        s = np.where(np.abs(p[:, :m]) < 1e10, ref.slope(np.clip(p[:, :m], -1e10, 1e10), kind), 0.0)  # (all four are 0 at -1e30)
    dg = dh * p[:, m:] * np.nan_to_num(s)
    for i, j in np.ndindex(n, m):
        if s[i, j] == 0:
            assert got[i, j] == 0, (kind, i, j)
        elif abs(s[i, j]) > 0.1:  # the slope is accurate there: in range it has to be right, beyond it an infinity
            assert np.isinf(got[i, j]) if abs(dg[i, j]) > 3.5e38 else abs(got[i, j] / dg[i, j] - 1) < 2.0 ** -7, (kind, i, j)


def test_grad_of_no_tokens_scales_what_is_there(h):
    m, k = 12, 20
    rng = seeded("no tokens")
    bits, start = ref.to_bits(rng.standard_normal((2 * m, k)), "bfloat16")
    none = Mat(h, "bfloat16", 1, 1)
    for beta in (0.0, 1.0, 2.0):
        da = Mat(h, "bfloat16", 2 * m, k, values=bits)
        h.wait(sb._gated_gemm_grad(h, activation_t.silu, "t", "n", m, 0, k, none.buf, k, none.buf, k, none.buf, 2 * m, none.buf, m,
                                   none.buf, 2 * m, beta, da.buf, k, 0.0, none.buf, k))
        assert (ref.from_bits(da.get(), "bfloat16") == beta * start).all()


@pytest.mark.parametrize("kind", ref.ACTS)
def test_gradient_against_differences(h, kind):
    """dA and dB against central differences of the 64-bit block in random directions.  x and w are multiples of 1/4 below 2, k
    is 4: the products are multiples of 1/16 below 16 and P is exact in half precision, so forward and backward pass see
    the very same pre-activations."""
    n, m, k, dtype = 6, 10, 4, "float16"
    rng = seeded("differences", kind)
    x = rng.integers(-7, 8, (n, k)) / 4.0
    w = rng.integers(-7, 8, (2 * m, k)) / 4.0
    if kind == "relu":  # keep the kink out of the differences' way
        while (np.abs(x @ w.T)[:, :m] < 0.01).any():
            w = rng.integers(-7, 8, (2 * m, k)) / 4.0 + 0.0
            x = rng.integers(-7, 8, (n, k)) / 4.0 + 0.25 * (rng.integers(0, 2, (n, k)) * 2 - 1) / 2.0
            x = np.round(x * 8) / 8
    p = x @ w.T
    pb, p16 = ref.to_bits(p, dtype)
    assert (p16 == p).all()
    dhb, dh = ref.to_bits(rng.standard_normal((n, m)), dtype)
    xg, wg = Mat(h, dtype, n, k, values=ref.to_bits(x, dtype)[0]), Mat(h, dtype, 2 * m, k, values=ref.to_bits(w, dtype)[0])
    cg, pg, dcg = Mat(h, dtype, n, m), Mat(h, dtype, n, 2 * m), Mat(h, dtype, n, m, values=dhb)
    dpg, dag, dbg = Mat(h, dtype, n, 2 * m), Mat(h, dtype, 2 * m, k), Mat(h, dtype, n, k)
    a = activation_t[kind]
    sb._gated_gemm(h, a, "t", "n", m, n, k, wg.buf, k, xg.buf, k, cg.buf, m, pg.buf, 2 * m)
    h.wait(sb._gated_gemm_grad(h, a, "t", "n", m, n, k, wg.buf, k, xg.buf, k, pg.buf, 2 * m, dcg.buf, m, dpg.buf, 2 * m, 0.0, dag.buf, k,
                               0.0, dbg.buf, k))
    assert (ref.from_bits(pg.get(), dtype) == p).all()
    da, db = ref.from_bits(dag.get(), dtype), ref.from_bits(dbg.get(), dtype)

    def loss(xx, ww):
        pp = xx @ ww.T
        return float((dh * ref.act(pp[:, :m], kind) * pp[:, m:]).sum())

    dp, dp_bound = ref.gate_grad(p, dh, m, kind, dtype)
    step = 1e-5
    for name, grad, at, left, other in (("dA", da, w, dp.T, x), ("dB", db, x, dp, w)):
        bound_left = dp_bound.T if name == "dA" else dp_bound
        err = bound_left @ np.abs(other) + 100 * ref.U32 * (np.abs(left) @ np.abs(other))
        bound = ref.rounded(left @ other, err, dtype)
        for _ in range(8):
            v = rng.standard_normal(at.shape)
            hi, lo = (loss(x, w + s * step * v) if name == "dA" else loss(x + s * step * v, w) for s in (1, -1))
            # central differences: a third derivative of at most about 1e3 here times step^2, and cancellation of the loss
            slack = 1e3 * step ** 2 * np.abs(v).sum() ** 3 + 1e-15 * 1e3 / step
            assert abs((grad * v).sum() - (hi - lo) / (2 * step)) <= (bound * np.abs(v)).sum() + slack, (kind, name)


@pytest.mark.parametrize("m", [2048, 4096 + 128])
def test_ring_walks_many_tiles(h, m):
    """More tiles than workgroups: every workgroup goes through several, the last ones ragged, with results and P leaving
    while the next tile's operands come in.  Sampled tokens against the 64-bit form."""
    n, k, dtype = 2600, 192, "bfloat16"
    rng = seeded("many tiles", m)
    xb, x = ref.to_bits(rng.standard_normal((n, k)), dtype)
    wb, w = ref.to_bits(rng.standard_normal((2 * m, k)) / math.sqrt(k), dtype)
    xg, wg, cg, pg = Mat(h, dtype, n, k, values=xb), Mat(h, dtype, 2 * m, k, values=wb), Mat(h, dtype, n, m), Mat(h, dtype, n, 2 * m)
    for family in (RING128, RING256):
        for keep in (False, True):
            h.set_kernel(*family)
            args = (pg.buf, 2 * m) if keep else ()
            h.wait(sb._gated_gemm(h, activation_t.silu, "t", "n", m, n, k, wg.buf, k, xg.buf, k, cg.buf, m, *args))
            rows = np.unique(np.concatenate([rng.integers(0, n, 200), [0, 255, 256, n - 1]]))
            p, p_err = x[rows] @ w.T, ref.product_error(x[rows], w, k)
            truth, bound = ref.gated(p, p_err, m, "silu", dtype)
            close(ref.from_bits(cg.get()[rows], dtype), truth, bound, f"many tiles {family} {keep}")
            if keep:
                close(ref.from_bits(pg.get()[rows], dtype), p, ref.rounded(p, p_err, dtype), f"many tiles P {family}")


# ------------------------------------------------------ offsets beyond 32 bits
def test_offsets_beyond_32_bits(h):
    """Leading dimensions that put the second and third row more than 2^31 elements away from the first."""
    ld, n, m, k = (1 << 30) + 16, 4, 40, 96
    rng = seeded("far rows")
    x, w = int8_operands(rng, n, 2 * m, k)
    far = helper.allocate(h, "int8", ld * (n - 1) + k)
    out = helper.allocate(h, "float16", ld * (n - 1) + m)
    back = np.empty((n, m), np.uint16)
    try:
        for i in range(n):
            helper.copy_to_device(h, x[i], far + i * ld, k)
        wg = Mat(h, "int8", 2 * m, k, values=w)
        s = (x.astype(np.int64) @ w.astype(np.int64).T).astype(np.float64)
        scale = vec(h, np.full(n, 2.0 ** -12, np.float32))
        h.wait(sb._gated_gemm_scaled(h, activation_t.silu, "t", "n", m, n, k, wg.buf, k, None, far, ld, scale.buf, out, ld))
        for i in range(n):
            h.wait(helper.copy_to_host(h, out + i * ld, back[i], m))
        truth, bound = ref.gated(s * 2.0 ** -12, 3.5 * ref.U32 * np.abs(s) * 2.0 ** -12, m, "silu", "float16")
        close(ref.from_bits(back, "float16"), truth, bound, "far rows")
        # and quantised from there
        q, sc = Mat(h, "int8", n, m), Mat(h, "float32", 1, n)
        h.wait(sb._quantize(h, m, n, out, ld, q.buf, m, sc.buf))
        want_q, want_s = ref.quantized(ref.from_bits(back, "float16"))
        assert (q.get() == want_q).all() and (sc.get()[0] == want_s).all()
    finally:
        helper.deallocate(far)
        helper.deallocate(out)


# ----------------------------------------------------------------- whole layers
@pytest.mark.parametrize("n", [1, 5, 160])
def test_serving_layer_in_8_bits(h, n):
    """quantise -> gated block -> quantise -> down projection, as a serving loop runs them on one stream with nothing waited
    for in between; each stage against the 64-bit form of what the stage before it left."""
    d, f, dtype = 192, 272, "bfloat16"
    rng = seeded("serving", n)
    xb, x = ref.to_bits(rng.standard_normal((n, d)) * np.exp(rng.standard_normal((n, 1))), dtype)
    w1b, w1 = ref.to_bits(rng.standard_normal((2 * f, d)) / math.sqrt(d), dtype)
    w2b, w2 = ref.to_bits(rng.standard_normal((d, f)) / math.sqrt(f), dtype)
    xg, w1g, w2g = (Mat(h, dtype, *v.shape, values=b) for b, v in ((xb, x), (w1b, w1), (w2b, w2)))
    # the weights' channels are rows here: quantised once by the same call
    q1, s1, q2, s2 = Mat(h, "int8", 2 * f, d), Mat(h, "float32", 1, 2 * f), Mat(h, "int8", d, f), Mat(h, "float32", 1, d)
    sb._quantize(h, d, 2 * f, w1g.buf, d, q1.buf, d, s1.buf)
    sb._quantize(h, f, d, w2g.buf, f, q2.buf, f, s2.buf)
    qx, sx, hid = Mat(h, "int8", n, d), Mat(h, "float32", 1, n), Mat(h, dtype, n, f)
    qh, sh, y = Mat(h, "int8", n, f), Mat(h, "float32", 1, n), Mat(h, dtype, n, d)
    sb._quantize(h, d, n, xg.buf, d, qx.buf, d, sx.buf)
    sb._gated_gemm_scaled(h, activation_t.silu, "t", "n", f, n, d, q1.buf, d, s1.buf, qx.buf, d, sx.buf, hid.buf, f)
    sb._quantize(h, f, n, hid.buf, f, qh.buf, f, sh.buf)
    h.wait(sb._gemm_scaled(h, "t", "n", d, n, f, 1.0, q2.buf, f, s2.buf, qh.buf, f, sh.buf, 0.0, y.buf, d))
    for qm, sm, v in ((q1, s1, w1), (q2, s2, w2), (qx, sx, x), (qh, sh, ref.from_bits(hid.get(), dtype))):
        q, s = ref.quantized(v)
        assert (qm.get() == q).all() and (sm.get()[0] == s).all()

    def scaled(qa, sa, qb, sb_):
        return (qa.get().astype(np.int64) @ qb.get().astype(np.int64).T) * sa.get()[0].astype(np.float64)[:, None] * sb_.get()[0].astype(np.float64)

    p = scaled(qx, sx, q1, s1)
    truth, bound = ref.gated(p, 3.5 * ref.U32 * np.abs(p), f, "silu", dtype)
    close(ref.from_bits(hid.get(), dtype), truth, bound, "hidden")
    out = scaled(qh, sh, q2, s2)
    close(ref.from_bits(y.get(), dtype), out, ref.rounded(out, 4.5 * ref.U32 * np.abs(out), dtype), "output")


def test_training_layer_in_bf16(h):
    """Forward with P kept, down projection, then the backward pass of the whole layer for a given gradient of its output:
    dH = W2^T dY, dW2 = dY H^T on the framework's products, the block's gradients on top."""
    n, d, f, dtype = 96, 64, 80, "bfloat16"
    rng = seeded("training")
    xb, x = ref.to_bits(rng.standard_normal((n, d)), dtype)
    w1b, w1 = ref.to_bits(rng.standard_normal((2 * f, d)) / math.sqrt(d), dtype)
    w2b, w2 = ref.to_bits(rng.standard_normal((d, f)) / math.sqrt(f), dtype)
    dyb, dy = ref.to_bits(rng.standard_normal((n, d)), dtype)
    xg, w1g, w2g, dyg = (Mat(h, dtype, *v.shape, values=b) for b, v in ((xb, x), (w1b, w1), (w2b, w2), (dyb, dy)))
    hid, p, y = Mat(h, dtype, n, f), Mat(h, dtype, n, 2 * f), Mat(h, "float32", n, d)
    sb._gated_gemm(h, activation_t.silu, "t", "n", f, n, d, w1g.buf, d, xg.buf, d, hid.buf, f, p.buf, 2 * f)
    sb._gemm(h, "t", "n", d, n, f, 1.0, w2g.buf, f, hid.buf, f, 0.0, y.buf, d)
    # dH (f x n) = W2^T (f x d) dY (d x n), float, then rounded to the type by the host as a trainer's cast would
    dhf = Mat(h, "float32", n, f)
    h.wait(sb._gemm(h, "n", "n", f, n, d, 1.0, w2g.buf, f, dyg.buf, d, 0.0, dhf.buf, f))
    dhb, dh = ref.to_bits(dhf.get(), dtype)
    close(dhf.get().astype(np.float64), dy @ w2, ref.product_error(dy, w2.T, d) + 1e-30, "dH")
    dhg, dp, dw1, dx = Mat(h, dtype, n, f, values=dhb), Mat(h, dtype, n, 2 * f), Mat(h, dtype, 2 * f, d), Mat(h, dtype, n, d)
    h.wait(sb._gated_gemm_grad(h, activation_t.silu, "t", "n", f, n, d, w1g.buf, d, xg.buf, d, p.buf, 2 * f, dhg.buf, f, dp.buf, 2 * f,
                               0.0, dw1.buf, d, 0.0, dx.buf, d))
    ps = ref.from_bits(p.get(), dtype)
    pe = x @ w1.T
    close(ps, pe, ref.rounded(pe, ref.product_error(x, w1, d), dtype), "P")
    truth, bound = ref.gate_grad(ps, dh, f, "silu", dtype)
    for got, left, other, b in ((dw1, truth.T, x, bound.T), (dx, truth, w1, bound)):
        t = left @ other
        err = b @ np.abs(other) + (left.shape[1] + 2) * ref.U32 * ((np.abs(left) + b) @ np.abs(other))
        close(ref.from_bits(got.get(), dtype), t, ref.rounded(t, err, dtype), "layer gradient")
    hs = ref.from_bits(hid.get(), dtype)
    close(y.get().astype(np.float64), hs @ w2.T, ref.product_error(hs, w2, f) + 1e-30, "Y")


# ------------------------------------------------------------ streams and graphs
def test_two_handles_at_once(h):
    """Two handles (two streams) run different calls that both need the repack area: each has its own."""
    n, m, k = 130, 200, 160
    other = sb.SB_Handle(0)
    try:
        jobs = []
        for i, hh in enumerate((h, other)):
            rng = seeded("two handles", i)
            x, w = int8_operands(rng, n, m, k)
            jobs.append((hh, x, w, Mat(hh, "int8", k, m, values=across(w)), Mat(hh, "int8", k, n, values=across(x)), Mat(hh, "float32", n, m)))
        for _ in range(20):
            for hh, x, w, wg, xg, cg in jobs:
                sb._gemm_scaled(hh, "n", "t", m, n, k, 1.0, wg.buf, m, None, xg.buf, n, None, 0.0, cg.buf, m)
        for hh, x, w, wg, xg, cg in jobs:
            hh.wait()
            assert (cg.get() == (x.astype(np.int64) @ w.astype(np.int64).T).astype(np.float32)).all()
    finally:
        for job in jobs:
            for mat in job[3:]:
                helper.deallocate(mat.alloc)
        other.close()


def test_captured_layer_replays(h):
    """The serving chain captured into a HIP graph on a handle's own stream and replayed on new inputs."""
    hip = C.CDLL("libamdhip64.so")
    n, d, f = 3, 128, 96
    hh = sb.SB_Handle(0)
    graph, graph_exec = C.c_void_p(), C.c_void_p()
    lib = _lib.load()
    rng = seeded("captured")
    x0 = rng.standard_normal((n, d)).astype(np.float32)
    w = rng.integers(-128, 128, (2 * f, d)).astype(np.int8)
    xg, wg = Mat(hh, "float32", n, d, values=x0), Mat(hh, "int8", 2 * f, d, values=w)
    q, s, c = Mat(hh, "int8", n, d), Mat(hh, "float32", 1, n), Mat(hh, "float32", n, f)

    def calls():
        assert lib.sbamd_squantize_i8(hh._h, d, n, xg.buf.ptr, d, q.buf.ptr, d, s.buf.ptr) == _lib.OK
        assert lib.sbamd_i8sgated_gemm(hh._h, _lib.ACT_GELU, b"t", b"n", f, n, d, wg.buf.ptr, d, None, q.buf.ptr, d, s.buf.ptr, c.buf.ptr,
                                       f) == _lib.OK

    try:
        calls()
        hh.wait()
        stream = C.c_void_p(hh.get_stream())
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        calls()
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0 and graph.value
        assert hip.hipGraphInstantiate(C.byref(graph_exec), graph, None, None, 0) == 0
        for i in range(4):
            x = (rng.standard_normal((n, d)) * 0.05).astype(np.float32)
            hh.wait(helper.copy_to_device(hh, x, xg.buf, x.size))
            xg.window(xg.host)[...] = x
            assert hip.hipGraphLaunch(graph_exec, stream) == 0
            hh.wait()
            qw, sw = ref.quantized(x.astype(np.float64))
            p = (qw.astype(np.int64) @ w.astype(np.int64).T) * sw.astype(np.float64)[:, None]
            truth, bound = ref.gated(p, 3.5 * ref.U32 * np.abs(p), f, "gelu", "float32")
            close(c.get().astype(np.float64), truth, bound, f"replay {i}")
            calls()  # eager work between the replays
            hh.wait()
            close(c.get().astype(np.float64), truth, bound, f"eager {i}")
    finally:
        if graph_exec.value:
            hip.hipGraphExecDestroy(graph_exec)
        if graph.value:
            hip.hipGraphDestroy(graph)
        hh.wait()
        for mat in (xg, wg, q, s, c):
            helper.deallocate(mat.alloc)
        hh.close()


def test_captured_call_keeps_its_scratch(h):
    """A call that repacks an operand and one that cuts its product along k, captured into a graph; a later, bigger call
    outgrows the scratch they were captured with; the graph still replays right."""
    hip = C.CDLL("libamdhip64.so")
    n, m, k = 200, 300, 2048
    hh = sb.SB_Handle(0)
    graph, graph_exec = C.c_void_p(), C.c_void_p()
    rng = seeded("captured scratch")
    x, w = int8_operands(rng, n, m, k)
    xg, wg = Mat(hh, "int8", n, k, values=x), Mat(hh, "int8", k, m, values=across(w))
    c = Mat(hh, "float32", n, m)
    big_x, big_w = int8_operands(rng, 2 * n, 4 * m, 2 * k)
    big = [Mat(hh, "int8", 2 * n, 2 * k, values=big_x), Mat(hh, "int8", 2 * k, 4 * m, values=across(big_w)), Mat(hh, "float32", 2 * n, 4 * m)]
    want = (x.astype(np.int64) @ w.astype(np.int64).T).astype(np.float32)
    hh.set_kernel(*RING128)

    def call():
        assert _lib.load().sbamd_i8sgemm(hh._h, b"n", b"n", m, n, k, 1.0, wg.buf.ptr, m, None, xg.buf.ptr, k, None, 0.0, c.buf.ptr,
                                         m) == _lib.OK

    try:
        call()  # the scratch has to exist before the capture
        assert hh.last_splitk()[0] > 1
        hh.wait()
        stream = C.c_void_p(hh.get_stream())
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        call()
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0 and graph.value
        assert hip.hipGraphInstantiate(C.byref(graph_exec), graph, None, None, 0) == 0
        for i in range(4):
            hh.wait(sb._gemm_scaled(hh, "n", "n", 4 * m, 2 * n, 2 * k, 1.0, big[1].buf, 4 * m, None, big[0].buf, 2 * k, None, 0.0,
                                    big[2].buf, 4 * m))
            assert (big[2].get() == (big_x.astype(np.int64) @ big_w.astype(np.int64).T).astype(np.float32)).all()
            filler = helper.allocate(hh, "float32", 1 << 20)  # lands where a freed scratch buffer would have been
            helper.copy_to_device(hh, np.full(1 << 20, np.nan, np.float32), filler)
            hh.wait(helper.copy_to_device(hh, np.zeros((n, m), np.float32), c.buf, n * m))
            assert hip.hipGraphLaunch(graph_exec, stream) == 0
            hh.wait()
            got = np.empty_like(c.host)
            hh.wait(helper.copy_to_host(hh, c.alloc, got))
            assert (c.window(got) == want).all(), f"replay {i}"
            helper.deallocate(filler)
    finally:
        if graph_exec.value:
            hip.hipGraphExecDestroy(graph_exec)
        if graph.value:
            hip.hipGraphDestroy(graph)
        hh.wait()
        for mat in (xg, wg, c, *big):
            helper.deallocate(mat.alloc)
        hh.close()


# -------------------------------------------------------------------- refusals
def test_refusals_leave_the_output(h):
    i8, f = Mat(h, "int8", 4, 8), Mat(h, "float32", 4, 8)
    with pytest.raises(ValueError, match="_TransA"):
        sb._gemm_scaled(h, "x", "n", 4, 4, 4, 1.0, i8.buf, 8, None, i8.buf, 8, None, 0.0, f.buf, 8)
    with pytest.raises(ValueError, match="_TransB"):
        sb._gated_gemm_scaled(h, activation_t.silu, "t", "x", 4, 4, 4, i8.buf, 8, None, i8.buf, 8, None, f.buf, 8)
    with pytest.raises(ValueError):
        sb._gated_gemm_scaled(h, 17, "t", "n", 4, 4, 4, i8.buf, 8, None, i8.buf, 8, None, f.buf, 8)
    with pytest.raises(ValueError):
        sb._gemm_scaled(h, "t", "n", 4, 4, 9, 1.0, i8.buf, 8, None, i8.buf, 8, None, 0.0, f.buf, 8)
    with pytest.raises(ValueError):
        sb._quantize(h, 8, 4, f.buf, 7, i8.buf, 8, f.buf)
    assert (f.get() == FILL["float32"]).all() and (i8.get() == FILL["int8"]).all()

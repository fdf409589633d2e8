"""The feed-forward ring kernel where a workgroup goes through several tiles, and the gradient's products term by term.

Operands are small whole numbers, so every sum is exact in float (below 2^24) whatever its order, and the stored result is the
exact one rounded once: results are compared bit by bit over the whole matrix, and a term too many, too few or read too early shows.
"""
import numpy as np
import pytest

import sycl_blas_amd as sb
from sycl_blas_amd import _lib, activation_t

import ffn_ref as ref
from common import seeded
from test_ffn_gpu import FAMILIES, NARROW, RING128, RING256, Mat, across, vec

pytestmark = pytest.mark.gpu

UNITS = 256  # workgroups of the 256 x 256 ring that are resident at once; twice as many of the 128 x 128 one


@pytest.fixture()
def h(sb_handle):
    sb_handle.set_kernel(_lib.KERNEL_AUTO)
    yield sb_handle
    sb_handle.set_kernel(_lib.KERNEL_AUTO)


def whole(rng, top, *shape):
    return rng.integers(-top, top + 1, shape).astype(np.float32)


def bits(x, dtype):
    return ref.to_bits(x, dtype)[0]


def same(got, want, what):
    """Equal bit by bit, but for the sign of a zero: -0 and 0 are the same number, and where a half result is a product rounded
    once the compiler adds a 0 to it, which makes -0 + 0 = 0 of a zero product and nothing of any other."""
    if got.dtype == np.uint16:
        got, want = (np.where(v == 0x8000, np.uint16(0), v) for v in (got, want))
    bad = got != want
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} differ, first at {np.unravel_index(np.argmax(bad), bad.shape)}"


# k: nine steps of 32 (the fewest whose first trip counts the stores behind the loads), ten with a tail, eight (none), more
@pytest.mark.parametrize("k", [288, 333, 256, 544])
@pytest.mark.parametrize("family,n,m", [(RING256, 2600, 4224), (RING128, 1300, 4160)])
@pytest.mark.parametrize("dtype,keep", [("bfloat16", False), ("bfloat16", True), ("float16", False)])
def test_gated_tiles_in_turn(h, dtype, keep, family, n, m, k):
    tiles = (-(-n // 256) * -(-m // 128)) if family is RING256 else (-(-n // 128) * -(-m // 64))
    assert tiles > UNITS * (1 if family is RING256 else 2)
    rng = seeded("gated tiles", dtype, keep, n, m, k)
    x, w = whole(rng, 1, n, k), whole(rng, 1, 2 * m, k)
    pre = x @ w.T + 0.0
    assert np.abs(pre).max() ** 2 < 2 ** 24
    pad = -k % 8  # rows in whole 16-byte pieces, so that the ring reads the operands where they are
    xg, wg = Mat(h, dtype, n, k, k + pad, values=bits(x, dtype)), Mat(h, dtype, 2 * m, k, k + pad, values=bits(w, dtype))
    cg, pg = Mat(h, dtype, n, m), Mat(h, dtype, n, 2 * m)
    h.set_kernel(*family)
    args = (pg.buf, pg.ld) if keep else ()
    for kind in ("relu", "relu", "silu"):
        h.wait(sb._gated_gemm(h, activation_t[kind], "t", "n", m, n, k, wg.buf, wg.ld, xg.buf, xg.ld, cg.buf, cg.ld, *args))
        assert h.last_kernel() == family[0]
        if kind == "relu":
            same(cg.get(), bits(np.maximum(pre[:, :m], 0) * pre[:, m:], dtype), "C")
        if keep:
            same(pg.get(), bits(pre, dtype), "P")
    by_ring = cg.get()
    h.set_kernel(*NARROW)  # the same sums, exact, and the same activation code
    h.wait(sb._gated_gemm(h, activation_t.silu, "t", "n", m, n, k, wg.buf, wg.ld, xg.buf, xg.ld, cg.buf, cg.ld))
    same(by_ring, cg.get(), "silu on the ring and on the narrow kernel")


@pytest.mark.parametrize("family,n,m", [(RING256, 4200, 4480), (RING128, 2100, 4160)])
@pytest.mark.parametrize("k", [576, 650])
@pytest.mark.parametrize("out,beta", [("float32", 0.0), ("float16", 0.0), ("bfloat16", 0.0), ("float32", 2.0), ("bfloat16", 2.0)])
def test_scaled_tiles_in_turn(h, out, beta, family, n, m, k):
    """8-bit products, each token and channel with a scale of its own (a power of two, so nothing is rounded but the result):
    the scales go from tile to tile with the operands."""
    rng = seeded("scaled tiles", out, beta, n, m, k)
    x, w = whole(rng, 3, n, k), whole(rng, 3, m, k)
    sx, sw = np.exp2(rng.integers(-3, 4, n)).astype(np.float32), np.exp2(rng.integers(-3, 4, m)).astype(np.float32)
    c0 = whole(rng, 20, n, m) if beta else np.zeros((n, m), np.float32)
    pad = -k % 16
    xg, wg = Mat(h, "int8", n, k, k + pad, values=x.astype(np.int8)), Mat(h, "int8", m, k, k + pad, values=w.astype(np.int8))
    cg = Mat(h, out, n, m, values=bits(c0, out))
    h.set_kernel(*family)
    h.wait(sb._gemm_scaled(h, "t", "n", m, n, k, 0.5, wg.buf, wg.ld, vec(h, sw).buf, xg.buf, xg.ld, vec(h, sx).buf, beta, cg.buf, cg.ld))
    assert h.last_kernel() == family[0] and h.last_splitk()[0] == 1
    scaled = np.float32(0.5) * (x @ w.T + 0.0) * sx[:, None] * sw[None, :]
    same(cg.get(), bits(scaled + np.float32(beta) * c0, out), f"{out} beta {beta}")


@pytest.mark.parametrize("family,n,m", [(RING256, 2600, 4224), (RING128, 1300, 4160)])
@pytest.mark.parametrize("out", ["float32", "float16", "bfloat16"])
def test_gated_scaled_tiles_in_turn(h, out, family, n, m):
    k = 650
    rng = seeded("gated scaled tiles", out, n, m)
    x, w = whole(rng, 2, n, k), whole(rng, 2, 2 * m, k)
    sx, sw = np.exp2(rng.integers(-2, 3, n)).astype(np.float32), np.exp2(rng.integers(-2, 3, 2 * m)).astype(np.float32)
    xg, wg = Mat(h, "int8", n, k, k + 6, values=x.astype(np.int8)), Mat(h, "int8", 2 * m, k, k + 6, values=w.astype(np.int8))
    cg = Mat(h, out, n, m)
    pre = (x @ w.T + 0.0) * sx[:, None] * sw[None, :]
    h.set_kernel(*family)
    for kind in ("relu", "gelu"):
        h.wait(sb._gated_gemm_scaled(h, activation_t[kind], "t", "n", m, n, k, wg.buf, wg.ld, vec(h, sw).buf, xg.buf, xg.ld, vec(h, sx).buf,
                                     cg.buf, cg.ld))
        assert h.last_kernel() == family[0]
        if kind == "relu":
            same(cg.get(), bits(np.maximum(pre[:, :m], 0) * pre[:, m:], out), out)
    by_ring = cg.get()
    h.set_kernel(*NARROW)
    h.wait(sb._gated_gemm_scaled(h, activation_t.gelu, "t", "n", m, n, k, wg.buf, wg.ld, vec(h, sw).buf, xg.buf, xg.ld, vec(h, sx).buf, cg.buf,
                                 cg.ld))
    same(by_ring, cg.get(), "gelu on the ring and on the narrow kernel")


@pytest.mark.parametrize("out,beta", [("float32", 0.0), ("bfloat16", 0.0), ("float16", 1.0)])
@pytest.mark.parametrize("n,m,k", [(4090, 4300, 4106), (5100, 4200, 9000)])
def test_whole_and_cut_tiles_in_one_launch(h, out, beta, n, m, k):
    """A first round of whole 256 x 256 tiles and a second, of 16 or 84, in pieces along k."""
    tiles = -(-n // 256) * -(-m // 256)
    assert UNITS < tiles < 2 * UNITS
    rng = seeded("whole and cut", out, n, m, k)
    x, w = whole(rng, 3, n, k), whole(rng, 3, m, k)
    c0 = whole(rng, 20, n, m) if beta else np.zeros((n, m), np.float32)
    pad = -k % 16
    xg, wg = Mat(h, "int8", n, k, k + pad, values=x.astype(np.int8)), Mat(h, "int8", m, k, k + pad, values=w.astype(np.int8))
    cg = Mat(h, out, n, m, values=bits(c0, out))
    h.set_kernel(*RING256)
    h.wait(sb._gemm_scaled(h, "t", "n", m, n, k, 0.5, wg.buf, wg.ld, None, xg.buf, xg.ld, None, beta, cg.buf, cg.ld))
    assert h.last_kernel() == RING256[0] and h.last_splitk()[0] > 1
    same(cg.get(), bits(np.float32(0.5) * (x @ w.T + 0.0) + np.float32(beta) * c0, out), out)


# ------------------------------------------------------------------- gradient
def exact_grad(h, dtype, n, m, k, ta="t", tb="n", pad=0, shift=0, beta_a=0.0, beta_b=0.0, want="ab", family=RING256, top=2, check_cut=None,
               repeat=1, in_place=False):
    """ReLU and whole numbers: dP is exact, and so are the sums behind dA and dB."""
    rng = seeded("exact gradient", dtype, n, m, k, ta, tb, pad, shift, beta_a, beta_b, want)
    x, w, p, dh = (whole(rng, top, *s) for s in ((n, k), (2 * m, k), (n, 2 * m), (n, m)))
    da0, db0 = whole(rng, 9, 2 * m, k), whole(rng, 9, n, k)
    dp = np.concatenate([dh * p[:, m:] * (p[:, :m] > 0), dh * np.maximum(p[:, :m], 0)], 1)

    def weights(v):
        return Mat(h, dtype, 2 * m, k, k + pad, shift, bits(v, dtype)) if ta == "t" else Mat(h, dtype, k, 2 * m, 2 * m + pad, shift, across(bits(v, dtype)))

    def tokens(v):
        return Mat(h, dtype, n, k, k + pad, shift, bits(v, dtype)) if tb == "n" else Mat(h, dtype, k, n, n + pad, shift, across(bits(v, dtype)))

    wg, xg = weights(w), tokens(x)
    pg = Mat(h, dtype, n, 2 * m, 2 * m + pad, shift, bits(p, dtype))
    dcg, dpg = Mat(h, dtype, n, m, m + pad, shift, bits(dh, dtype)), Mat(h, dtype, n, 2 * m, 2 * m + pad, shift)
    dpg = pg if in_place else dpg
    h.set_kernel(*family)
    for _ in range(repeat):
        dag, dbg = weights(da0) if "a" in want else None, tokens(db0) if "b" in want else None
        h.wait(sb._gated_gemm_grad(h, activation_t.relu, ta, tb, m, n, k, wg.buf, wg.ld, xg.buf, xg.ld, pg.buf, pg.ld, dcg.buf, dcg.ld, dpg.buf,
                                   dpg.ld, beta_a, dag and dag.buf, wg.ld, beta_b, dbg and dbg.buf, xg.ld))
        if check_cut is not None:
            assert (h.last_splitk()[0] > 1) == check_cut
        # (+ 0: a product's -0 and a sum's 0 are the same number)
        same(ref.from_bits(dpg.get(), dtype) + 0.0, dp + 0.0, "dP")
        for name, out, left, other, turned, beta, start in (("dA", dag, dp.T, x, ta != "t", beta_a, da0), ("dB", dbg, dp, w, tb != "n", beta_b, db0)):
            if out is not None:
                truth = left @ other + np.float32(beta) * start
                assert np.abs(left).max() * np.abs(other).max() * left.shape[1] < 2 ** 24
                got = ref.from_bits(out.get(), dtype)
                same((got.T if turned else got) + 0.0, ref.to_bits(truth, dtype)[1] + 0.0, f"{name} {ta}{tb} beta {beta}")


@pytest.mark.parametrize("family", FAMILIES)
@pytest.mark.parametrize("ta,tb", [("t", "n"), ("n", "n"), ("t", "t"), ("n", "t")])
@pytest.mark.parametrize("n,m,k", [(256, 128, 256), (1104, 304, 136), (72, 700, 264), (600, 36, 48), (2500, 20, 40), (1119, 273, 100),
                                   (33, 17, 31)])
def test_grad_counts_every_term(h, family, n, m, k, ta, tb):
    exact_grad(h, "bfloat16", n, m, k, ta, tb, beta_a=0.5 if m > 100 else 0.0, family=FAMILIES[family])
    exact_grad(h, "float16", n, m, k, ta, tb, pad=8, beta_b=1.0 if m > 100 else 0.0, family=FAMILIES[family])
    exact_grad(h, "bfloat16", n, m, k, ta, tb, pad=3, shift=1, family=FAMILIES[family])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("ta,tb", [("t", "n"), ("n", "t")])
def test_grad_whole_and_cut_tiles_in_one_launch(h, dtype, ta, tb):
    """dA has 17 x 16 tiles of 256 x 256, a sum over 2208 tokens; dB 16 x 9, a sum over 4352 rows of P."""
    n, m, k = 2208, 2176, 4096
    exact_grad(h, dtype, n, m, k, ta, tb, want="a", top=1, check_cut=True)
    exact_grad(h, dtype, n, m, k, ta, tb, top=1, repeat=2)


@pytest.mark.parametrize("family", FAMILIES)
@pytest.mark.parametrize("ta,tb", [("t", "n"), ("n", "t")])
@pytest.mark.parametrize("n,m,k,pad", [(1104, 302, 136, 0), (77, 29, 40, 0), (520, 130, 64, 6)])
def test_grad_in_place_of_p(h, family, n, m, k, pad, ta, tb):
    """dP over P where the products read a padded copy of it (2m and its rows no multiple of 8) and where they do not."""
    exact_grad(h, "bfloat16", n, m, k, ta, tb, pad=pad, family=FAMILIES[family], in_place=True)
    exact_grad(h, "float16", n, m, k, ta, tb, pad=pad, family=FAMILIES[family], in_place=True, want="b")


def test_grad_tiles_in_turn(h):
    """Four tiles and more for each workgroup, dA over 333 tokens and dB over 352 rows of P."""
    exact_grad(h, "bfloat16", 333, 4352, 4104, want="a", family=RING256, check_cut=False, beta_a=1.0)
    exact_grad(h, "bfloat16", 333, 4352, 4104, want="a", family=RING256, check_cut=False)
    exact_grad(h, "float16", 4200, 176, 4608, want="b", family=RING256, check_cut=False)
    exact_grad(h, "bfloat16", 333, 4352, 2100, want="a", family=RING128, check_cut=False)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("n,m,k", [(1119, 2730, 1000), (4096, 128, 128), (2208, 2176, 1024)])
def test_grad_repeats_bit_by_bit(h, dtype, n, m, k):
    """Sums have a fixed order: the same call on the same operands gives the same bits."""
    rng = seeded("repeats", dtype, n, m, k)
    mats = [Mat(h, dtype, r, c, values=bits(rng.standard_normal((r, c)) * s, dtype)) for r, c, s in
            ((2 * m, k, 0.05), (n, k, 1.0), (n, 2 * m, 1.0), (n, m, 0.01))]
    wg, xg, pg, dcg = mats
    dpg, dag, dbg = Mat(h, dtype, n, 2 * m), Mat(h, dtype, 2 * m, k), Mat(h, dtype, n, k)
    first = None
    for _ in range(3):
        h.wait(sb._gated_gemm_grad(h, activation_t.gelu, "t", "n", m, n, k, wg.buf, k, xg.buf, k, pg.buf, 2 * m, dcg.buf, m, dpg.buf, 2 * m,
                                   0.0, dag.buf, k, 0.0, dbg.buf, k))
        now = [g.get() for g in (dpg, dag, dbg)]
        first = first or now
        assert all((a == b).all() for a, b in zip(first, now))

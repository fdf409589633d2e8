"""Feed-forward operators with more items than one row of workgroups holds (HIP refuses 2^32 or more threads along an axis):
sampled columns, the last ones among them, against the plain 64-bit form of tests/ffn_ref.py, and the memory behind the
last one unchanged."""
import numpy as np
import pytest

import sycl_blas_amd as sb
from sycl_blas_amd import _lib, activation_t, helper

import ffn_ref as ref
from common import seeded

pytestmark = pytest.mark.gpu

STORE = {"float32": np.float32, "float16": np.uint16, "bfloat16": np.uint16, "int8": np.int8}
TAIL = 64  # elements behind every output


class Pool:
    """Device buffers of one test, freed at its end."""

    def __init__(self):
        self.h = sb.SB_Handle(0)
        self.bufs = []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.h.wait()
        for b in self.bufs:
            helper.deallocate(b)
        self.h.close()  # and its scratch

    def empty(self, dtype, count, byte=0x2A):
        b = helper.allocate(self.h, dtype, count)
        self.bufs.append(b)
        assert _lib.load().sbamd_memset(self.h._h, b.ptr, byte, count * b.itemsize) == _lib.OK
        return b

    def random(self, dtype, count, seed, lo=-2.0, hi=5.0):
        b = self.empty(dtype, count)
        helper.fill_uniform(self.h, b, count, seed, lo, hi)
        return b

    def read(self, buf, at, count):
        out = np.empty(count, STORE[buf.dtype])
        self.h.wait(helper.copy_to_host(self.h, buf + at, out))
        return out

    def values(self, buf, at, count):
        bits = self.read(buf, at, count)
        return bits.astype(np.float64) if buf.dtype == "int8" else ref.from_bits(bits, buf.dtype)

    def untouched(self, buf, at):
        return (self.read(buf, at, TAIL).view(np.uint8) == 0x2A).all()


def sampled(rng, n, around=()):
    at = set(int(i) for i in rng.integers(0, n, 30)) | {0, 1, 2, n - 1, n - 2, n - 3}
    for a in around:
        at |= {a - 1, a, a + 1}
    return sorted(i for i in at if 0 <= i < n)


@pytest.mark.parametrize("m,n", [(1, (1 << 26) + 3), (513, (1 << 24) + 5), (4097, (1 << 22) + 5)])
def test_quantize_many_columns(m, n):
    rng = seeded("many columns", m, n)
    with Pool() as p:
        x = p.random("bfloat16", m * n, 7)
        q, s = p.empty("int8", m * n + TAIL), p.empty("float32", n + TAIL)
        p.h.wait(sb._quantize(p.h, m, n, x, m, q, m, s))
        for j in sampled(rng, n, (n // 2,)):
            want_q, want_s = ref.quantized(p.values(x, j * m, m)[None, :])
            assert (p.read(q, j * m, m) == want_q[0]).all() and p.read(s, j, 1)[0] == want_s[0], j
        assert p.untouched(q, m * n) and p.untouched(s, n)


@pytest.mark.parametrize("out", ["float32", "float16", "bfloat16"])
def test_scaled_alpha_zero_of_many_elements(out):
    """C <- beta C on 5 * 2^30 elements, all three types."""
    m, n, beta = 5, 1 << 30, 0.5
    rng = seeded("many elements", out)
    with Pool() as p:
        c = p.empty(out, m * n + TAIL)
        helper.fill_uniform(p.h, c, m * n, 11)
        at = sampled(rng, n, (n // 2, (1 << 32) // m))
        before = {j: p.values(c, j * m, m) for j in at}
        one = p.empty("int8", 64)
        p.h.wait(sb._gemm_scaled(p.h, "t", "n", m, n, 8, 0.0, one, 8, None, one, 8, None, beta, c, m))
        for j in at:
            assert (p.values(c, j * m, m) == ref.to_bits(beta * before[j], out)[1]).all(), j
        assert p.untouched(c, m * n)


@pytest.mark.parametrize("family", [_lib.KERNEL_SMALL, _lib.KERNEL_LARGE])
def test_scaled_of_many_tokens(family):
    """2^30 tokens of one element: the narrow kernel's workgroups, and the copy that pads such rows for the ring (64 GB)."""
    n = (1 << 30) + 70
    rng = seeded("many tokens", family)
    with Pool() as p:
        x, w = p.empty("int8", n, 3), p.empty("int8", 64, 2)
        s = p.random("float32", n, 5)
        c = p.empty("float16", n + TAIL)
        p.h.set_kernel(family)
        p.h.wait(sb._gemm_scaled(p.h, "t", "n", 1, n, 1, 1.0, w, 1, None, x, 1, s, 0.0, c, 1))
        assert p.h.last_kernel() == family
        for j in sampled(rng, n - 64, (n // 2, n // 4)) + [n - 64]:
            truth = 6.0 * p.values(s, j, 64)
            got = p.values(c, j, 64)
            assert (np.abs(got - truth) <= ref.rounded(truth, 3.0 * ref.U32 * np.abs(truth), "float16")).all(), j
        assert p.untouched(c, n)


def test_gated_of_many_channels():
    m = (1 << 28) + 37
    rng = seeded("many channels")
    with Pool() as p:
        x, w = p.empty("int8", 64, 1), p.empty("int8", 2 * m, 1)
        s = p.random("float32", 2 * m, 6)
        c = p.empty("float32", m + TAIL)
        p.h.set_kernel(_lib.KERNEL_SMALL)
        p.h.wait(sb._gated_gemm_scaled(p.h, activation_t.silu, "t", "n", m, 1, 1, w, 1, s, x, 1, None, c, m))
        for j in sampled(rng, m - 64, (m // 2,)) + [m - 64]:
            g = np.concatenate([p.values(s, j, 64), p.values(s, m + j, 64)])[None, :]
            truth, bound = ref.gated(g, 3.5 * ref.U32 * np.abs(g), 64, "silu", "float32")
            assert (np.abs(p.values(c, j, 64) - truth[0]) <= bound[0]).all(), j
        assert p.untouched(c, m)


def test_grad_of_many_tokens():
    """dP of 2^32 tokens of one channel, in place of P."""
    m, n = 1, (1 << 32) + 9
    rng = seeded("many gradients")
    with Pool() as p:
        pre = p.empty("bfloat16", 2 * n + TAIL)
        helper.fill_uniform(p.h, pre, 2 * n, 8)
        dc = p.random("bfloat16", n, 9)
        at = sampled(rng, n - 32, (n // 2,)) + [n - 32]
        before = {j: p.values(pre, 2 * j, 64).reshape(32, 2) for j in at}
        p.h.wait(sb._gated_gemm_grad(p.h, activation_t.silu, "t", "n", m, n, 1, None, 0, None, 0, pre, 2, dc, 1, pre, 2, 0.0, None, 0, 0.0,
                                     None, 0))
        for j in at:
            truth, bound = ref.gate_grad(before[j], p.values(dc, j, 32)[:, None], m, "silu", "bfloat16")
            assert (np.abs(p.values(pre, 2 * j, 64).reshape(32, 2) - truth) <= bound).all(), j
        assert p.untouched(pre, 2 * n)

"""The feed-forward entry points without a GPU: header, library and binding agree, and every refusal of the host code
holds under sanitizers (tests/host_san/ffn_logic.cpp over the stand-in HIP runtime)."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

import sycl_blas_amd as sb
from sycl_blas_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HOST_SAN = os.path.join(ROOT, "tests", "host_san")


def test_header_symbols_are_exported_and_bound():
    text = open(os.path.join(ROOT, "include", "sbamd_ffn.h")).read()
    plain = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = sorted(set(re.findall(r"\b(sbamd_[a-z0-9_]+)\s*\(", plain)))
    assert len(names) == 13
    lib = ctypes.CDLL(_lib.LIB_PATH)
    for name in names:
        assert hasattr(lib, name), f"{name} is declared but not exported"
    assert sorted(_lib.FFN_SIGNATURES) == names
    # argument counts of the prototypes
    for name, args in re.findall(r"int (sbamd_[a-z0-9_]+)\(([^;]*?)\);", plain, flags=re.S):
        assert len(args.split(",")) == len(_lib.FFN_SIGNATURES[name][1]), name
    for constant, value in (("SBAMD_ACT_SILU", _lib.ACT_SILU), ("SBAMD_ACT_GELU", _lib.ACT_GELU),
                            ("SBAMD_ACT_GELU_TANH", _lib.ACT_GELU_TANH), ("SBAMD_ACT_RELU", _lib.ACT_RELU)):
        assert re.search(rf"\b{constant} = {value}\b", text)
    assert f"#define SBAMD_I8_MAX_K {_lib.I8_MAX_K}" in text


def test_null_handle_is_rejected():
    lib = _lib.load()
    assert lib.sbamd_bquantize_i8(None, 1, 1, None, 1, None, 1, None) == _lib.INVALID_HANDLE
    assert lib.sbamd_i8sgemm(None, b"t", b"n", 1, 1, 1, 1.0, None, 1, None, None, 1, None, 0.0, None, 1) == _lib.INVALID_HANDLE
    assert lib.sbamd_bgated_gemm(None, 0, b"t", b"n", 1, 1, 1, None, 1, None, 1, None, 1, None, 0) == _lib.INVALID_HANDLE


def test_element_types_are_checked_before_the_call():
    class NoHandle:
        _h = None

        def depends_on(self, deps):
            raise AssertionError("a refused call must not reach the stream")

    def buf(dtype):
        return sb.DeviceBuffer.from_pointer(64, dtype, 64)

    h, f, i, b, d = NoHandle(), buf("float32"), buf("int8"), buf("bfloat16"), buf("float64")
    silu = sb.activation_t.silu
    for call in (
        lambda: sb._quantize(h, 1, 1, d, 1, i, 1, f),
        lambda: sb._quantize(h, 1, 1, b, 1, b, 1, f),
        lambda: sb._quantize(h, 1, 1, b, 1, i, 1, b),
        lambda: sb._gemm_scaled(h, "t", "n", 1, 1, 1, 1.0, b, 1, f, i, 1, f, 0.0, f, 1),
        lambda: sb._gemm_scaled(h, "t", "n", 1, 1, 1, 1.0, i, 1, f, b, 1, f, 0.0, f, 1),
        lambda: sb._gemm_scaled(h, "t", "n", 1, 1, 1, 1.0, i, 1, b, i, 1, f, 0.0, f, 1),
        lambda: sb._gemm_scaled(h, "t", "n", 1, 1, 1, 1.0, i, 1, f, i, 1, f, 0.0, i, 1),
        lambda: sb._gated_gemm(h, silu, "t", "n", 1, 1, 1, f, 1, f, 1, f, 1),
        lambda: sb._gated_gemm(h, silu, "t", "n", 1, 1, 1, b, 1, b, 1, f, 1),
        lambda: sb._gated_gemm(h, silu, "t", "n", 1, 1, 1, b, 1, b, 1, b, 1, f, 2),
        lambda: sb._gated_gemm_scaled(h, silu, "t", "n", 1, 1, 1, i, 1, f, i, 1, i, f, 1),
        lambda: sb._gated_gemm_grad(h, silu, "t", "n", 1, 1, 1, b, 1, b, 1, f, 2, b, 1, b, 2, 0.0, b, 1, 0.0, b, 1),
        lambda: sb._gated_gemm_grad(h, silu, "t", "n", 1, 1, 1, b, 1, b, 1, b, 2, b, 1, b, 2, 0.0, f, 1, 0.0, b, 1),
        lambda: sb.helper.fill_uniform(h, i, 1, 1),
    ):
        with pytest.raises(TypeError):
            call()


CALLS = r"""
#include "portblas_compat.hpp"
template <typename T>
void layer(blas::SB_Handle& h) {
  using blas::activation_t;
  auto x = blas::make_sycl_iterator_buffer<T>(h, 64), y = blas::make_sycl_iterator_buffer<T>(h, 64);
  auto q = blas::make_sycl_iterator_buffer<int8_t>(h, 64);
  auto s = blas::make_sycl_iterator_buffer<float>(h, 64);
  const float* ones = nullptr;
  auto ev = blas::_quantize(h, 4, 4, x, 4, q, 4, s);
  ev = blas::_gemm_scaled(h, 't', 'n', 4, 4, 4, 1.0f, q, 4, s, q, 4, ones, 0.0f, y, 4, ev);
  blas::_gated_gemm_scaled(h, activation_t::gelu, 't', 'n', 2, 4, 4, q, 4, s, q, 4, s, y, 2, ev);
}
template <typename T>
void training(blas::SB_Handle& h) {
  using blas::activation_t;
  auto w = blas::make_sycl_iterator_buffer<T>(h, 64), x = w, c = w, p = w, dw = w, dx = w;
  T* none = nullptr;
  auto ev = blas::_gated_gemm(h, activation_t::silu, 't', 'n', 2, 4, 4, w, 4, x, 4, c, 2, p + 8, 4);
  blas::_gated_gemm(h, activation_t::silu, 't', 'n', 2, 4, 4, w, 4, x.get(), 4, c, 2, none, 0, ev);
  blas::_gated_gemm_grad(h, activation_t::silu, 't', 'n', 2, 4, 4, w, 4, x, 4, p, 4, c, 2, p, 4, 0.0f, dw, 4, 1.0f, none, 4, ev);
}
int main() {
  blas::SB_Handle h(0);
  layer<float>(h);
  layer<blas::half_t>(h);
  layer<blas::bfloat16_t>(h);
  training<blas::half_t>(h);
  training<blas::bfloat16_t>(h);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_cpp_interface_compiles_for_every_type(tmp_path):
    source = tmp_path / "calls.cpp"
    source.write_text(CALLS)
    run = subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(source)],
                         capture_output=True, text=True)
    assert run.returncode == 0, run.stderr[-3000:]


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc") or shutil.which("make") is None, reason="needs hipcc and make")
def test_host_logic_refuses_and_accepts_under_asan_and_ubsan():
    build = subprocess.run(["make", "-C", HOST_SAN, "-j8", "build/ffn_logic"], capture_output=True, text=True)
    assert build.returncode == 0, build.stdout[-3000:] + build.stderr[-3000:]
    run = subprocess.run(["make", "-C", HOST_SAN, "run-ffn"], capture_output=True, text=True, timeout=300)
    out = run.stdout + run.stderr
    assert run.returncode == 0, out[-6000:]
    assert "ERROR: AddressSanitizer" not in out and "runtime error:" not in out and "LeakSanitizer" not in out, out[-6000:]
    assert " 0 expectations failed" in out

"""The draft verification's weights e^((l - m) / T) on the CPU: verify_weight.h, the header
the kernels use, built for the host (its one GPU instruction, ldexp, is exact on
both) and compared with 80-bit exponentials.

The exponential states 4e-14 of the value. A weight adds the rounding of its exponent
t = (l - m) c: c = log2 e / T is off by 2 half units (the constant's and the quotient's), the
product by one more, so t by 3 2^-53 |t| and the weight by ln 2 times that; the
difference of two f32 numbers rounds by another 2^-53 where they lie 2^29 apart."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "qwen3asr.rs_amd", "csrc")
F32 = np.finfo(np.float32)

SOURCE = r"""
#include <math.h>
#include <stdint.h>
#include <string.h>
static double __builtin_amdgcn_ldexp(double v, int n) { return ldexp(v, n); }
static float __uint_as_float(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
static uint32_t __float_as_uint(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
#include "verify_weight.h"
extern "C" void exp2s(const double* t, double* out, int64_t n) {
  for (int64_t i = 0; i < n; ++i) out[i] = vpa::exp2_nonpos(t[i]);
}
// of each logit: its weight, and the exponent that is formed for it (0: none is)
extern "C" void weights(float max, float temp, const float* l, double* out, double* t, int64_t n) {
  const vpa::Scale s(max, temp);
  for (int64_t i = 0; i < n; ++i) {
    t[i] = s.odd ? 0.0 : s.exponent(l[i]);
    out[i] = t[i] < -2147483648.0 ? NAN : s.weight(l[i]);
  }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None or not os.path.exists("/opt/rocm/include/hip/hip_runtime.h"):
        pytest.skip("g++ or the HIP headers not found")
    d = tmp_path_factory.mktemp("weight")
    (d / "weight.cpp").write_text(SOURCE)
    subprocess.run([gxx, "-O2", "-std=c++20", "-ffp-contract=off", "-shared", "-fPIC",
                    "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{CSRC}",
                    str(d / "weight.cpp"), "-o", str(d / "weight.so")], check=True)
    lib = ctypes.CDLL(str(d / "weight.so"))
    p = ctypes.c_void_p
    lib.exp2s.argtypes = [p, p, ctypes.c_int64]
    lib.weights.argtypes = [ctypes.c_float, ctypes.c_float, p, p, p, ctypes.c_int64]
    return lib


def weights(lib, top, temp, logits):
    l = np.ascontiguousarray(logits, np.float32)
    out, t = np.empty(l.size), np.empty(l.size)
    lib.weights(top, temp, l.ctypes.data, out.ctypes.data, t.ctypes.data, l.size)
    return out, t


def test_exponential_keeps_its_stated_error(lib):
    rng = np.random.default_rng(0)
    half = np.arange(-1020, 1) - 0.5  # the polynomial's ends
    t = np.concatenate([-1020 * rng.random(400000), -2 * rng.random(200000), half,
                        np.nextafter(half, -np.inf), np.nextafter(half, 0), np.arange(-1020.0, 1)])
    t = t[t <= 0]
    out = np.empty_like(t)
    lib.exp2s(t.ctypes.data, out.ctypes.data, t.size)
    want = np.exp2(t.astype(np.longdouble))
    assert np.max(np.abs(out / want - 1)) < 4e-14
    assert np.all(out[t == np.rint(t)] == np.exp2(t[t == np.rint(t)]))


def test_small_results_of_the_exponential(lib):
    """Below the normal numbers half a unit more, below all numbers 0."""
    t = np.concatenate([np.linspace(-1074.9, -1020, 20001), [-1076.0, -2000.0, -1e9, -2147483648.0]])
    out = np.empty_like(t)
    lib.exp2s(t.ctypes.data, out.ctypes.data, t.size)
    want = np.exp2(t.astype(np.longdouble))
    assert np.all(np.abs(out - want) <= 4e-14 * want + np.longdouble(2) ** -1075)
    assert np.all(out[-4:] == 0)


TEMPS = [1e-45, 1e-39, 1e-30, 1e-16, 1e-9, 1e-6, 1e-3, 0.3, 1.0, 7.5, 1e4, 1e15, 1e29, 1e30, 1e33,
         3e38, np.inf]
TOPS = [0.0, 1e-45, -1e-45, 1e-38, 0.1, -0.1, 1.0, -2.0, 10.0, -10.0, 3e4, -6.5e4, 1e9, 1e30, -1e30, 1e38,
        -3.3895314e38, 3.3895314e38, float(F32.max), float(F32.min)]


@pytest.mark.parametrize("temp", TEMPS)
def test_weights(lib, temp):
    """Maxima of every size against logits one step, a temperature, and everything below
    them; no exponent leaves the range that the exponential converts."""
    temp = float(np.float32(temp))
    for top in TOPS:
        top = np.float32(top)
        with np.errstate(over="ignore", invalid="ignore"):
            near = top - np.float32(temp) * np.linspace(0, 900, 91, dtype=np.float32)
            steps = [top]
            for _ in range(40):
                steps.append(np.nextafter(steps[-1], np.float32(-np.inf)))
            l = np.concatenate([near, steps, top - np.float32(2.0) ** np.arange(-149, 128, dtype=np.float32),
                                [-F32.max, np.float32(-3.3895314e38), -65504.0]]).astype(np.float32)
        l = l[(l <= top) & np.isfinite(l)]
        got, t = weights(lib, top, temp, l)
        assert not np.isnan(got).any(), "an exponent below -2^31"
        real = max(np.log2(np.e) / np.float64(temp), 1e-30) if temp > 0 else np.inf
        exact = (l.astype(np.longdouble) - np.longdouble(top)) * np.longdouble(real)
        want = np.exp2(np.maximum(exact, -5000))
        tol = want * (4e-14 + 4 * 2.0 ** -53 * 0.7 * np.minimum(-exact, 5000)) + np.longdouble(2) ** -1074
        assert np.all(np.abs(got - want) <= tol), (top, temp)
        assert got[l == top].min() == 1.0
        none, _ = weights(lib, top, temp, [-np.inf, np.nan])
        assert none.tolist() == [0.0, 0.0]


@pytest.mark.parametrize("temp", [1e-39, 1.0, np.inf])
def test_maxima_that_only_their_equals_share(lib, temp):
    lowest = float(-F32.max)
    got, _ = weights(lib, np.inf, temp, [np.inf, F32.max, 0.0, -np.inf, np.nan])
    assert got.tolist() == [1, 0, 0, 0, 0]
    got, _ = weights(lib, lowest, temp, [lowest, -np.inf, np.nan])
    assert got.tolist() == [1, 0, 0]
    got, _ = weights(lib, -np.inf, temp, [-np.inf, np.nan])
    assert got.tolist() == [0, 0]

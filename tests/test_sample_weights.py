"""CPU tests of the sampler's weights: csrc/sample_weights.hpp, which the kernels include, compiled for the host and compared
with the definition in extended precision."""
from __future__ import annotations

import ctypes
import importlib
import subprocess

import numpy as np
import pytest

from conftest import PKG

REST = 1023            # the bin of the tokens without weight
GREEDY = np.float32(1e-10)

SOURCE = r"""
#include "sample_weights.hpp"
extern "C" void weigh(const float* l, const float* largest, const float* t, int n, int32_t* bin, int32_t* off) {
    for (int i = 0; i < n; ++i) {
        const nvg::Weight w = nvg::weigh(l[i], nvg::scale_of(largest[i], t[i]));
        bin[i] = w.bin;
        off[i] = w.off;
    }
}
"""


@pytest.fixture(scope="module")
def weigh(tmp_path_factory):
    build = importlib.import_module("inference_systems_amd.build")
    try:
        hipcc = build.hipcc()
    except RuntimeError as exc:
        pytest.skip(str(exc))
    folder = tmp_path_factory.mktemp("weights")
    source, library = folder / "weights.cpp", folder / "libweights.so"
    source.write_text(SOURCE)
    proc = subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-O2", "-std=c++17", "-fPIC", "-shared",
                           f"-I{build.CSRC}", str(source), "-o", str(library)], capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr
    call = ctypes.CDLL(str(library)).weigh

    def run(logits, largest, t):
        """(bins, offsets) of logits in rows of these largest logits and temperatures."""
        l, b, t = (np.ascontiguousarray(x, dtype=np.float32) for x in np.broadcast_arrays(logits, largest, t))
        bins, offs = np.empty(l.size, np.int32), np.empty(l.size, np.int32)
        f, i = ctypes.POINTER(ctypes.c_float), ctypes.POINTER(ctypes.c_int32)
        call(*(x.ctypes.data_as(f) for x in (l, b, t)), l.size, bins.ctypes.data_as(i), offs.ctypes.data_as(i))
        return bins, offs
    return run


def temperatures(g, n):
    t = np.exp(g.uniform(np.log(1.0e-10), np.log(1.0e-6), n)).astype(np.float32)
    wide = np.exp(g.uniform(np.log(1.0e-10), np.log(3.0e38), n)).astype(np.float32)
    near = g.uniform(0.05, 3.0, n).astype(np.float32)
    t = np.choose(g.integers(0, 3, n), [t, wide, near])
    return np.maximum(t, np.nextafter(GREEDY, np.float32(1)))


def logits(g, n):
    """Of both signs, 32 and 16 bits, ordinary ones and ones of any size."""
    x = np.where(g.random(n) < 0.5, g.uniform(-30, 30, n), np.exp(g.uniform(np.log(1e-30), np.log(3.3e38), n)) * g.choice([-1, 1], n))
    x = x.astype(np.float32)
    bf16 = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
    return np.where(g.random(n) < 0.3, bf16, x)


@pytest.mark.parametrize("seed", range(4))
def test_the_largest_logit_has_weight(weigh, seed):
    g = np.random.default_rng(seed)
    x, t = logits(g, 400000), temperatures(g, 400000)
    bins, offs = weigh(x, x, t)
    assert (bins == 0).all()
    assert (np.abs(offs) <= 1600000000).all()


def below(g, x, t):
    """Logits below x, most of them by up to 70 octaves of weight, some next to it."""
    down = np.exp(g.uniform(np.log(1e-6), np.log(70.0), x.size)) * np.log(2.0) * t.astype(np.float64)
    with np.errstate(over="ignore"):
        y = (x.astype(np.float64) - down).astype(np.float32)
    for steps in (1, 2, 3):
        pick = g.random(x.size) < 0.1
        near = x
        for _ in range(steps):
            near = np.nextafter(near, np.float32(-np.inf))
        y = np.where(pick, near, y)
    return np.minimum(np.maximum(y, np.float32(-3.4e38)), x)


def octaves16(x, y, t):
    """How far y's weight is below x's, in 1/16 octaves, in extended precision."""
    return (x.astype(np.longdouble) - y.astype(np.longdouble)) * np.longdouble(16) / np.log(np.longdouble(2)) / t.astype(np.longdouble)


@pytest.mark.parametrize("seed", range(4))
def test_bins_follow_the_definition(weigh, seed):
    """A token's bin is its distance from the largest logit's, each rounded: off by less than 1, and beyond the bins only
    what is that far down."""
    g = np.random.default_rng(100 + seed)
    x, t = logits(g, 400000), temperatures(g, 400000)
    y = below(g, x, t)
    bins, _ = weigh(y, x, t)
    want = np.minimum(octaves16(x, y, t), REST)
    # Each rounding takes a half; a product in 32 bits, up to 2^14, is off by 2^-9 in front of it.
    assert (np.abs(bins - want) <= 1.0 + 2.0 ** -8).all()


def test_bins_do_not_fall_with_the_logit(weigh):
    g = np.random.default_rng(7)
    for t in (1.5e-10, 1e-9, 1e-8, 1e-3, 0.7, 1.0, 40.0, 1e6):
        for top in (-3e5, -700.0, -3.0, 0.0, 1.0, 9.7, 709.8, 16384.0, 4e6, 1e20):
            x = np.float32(top)
            y = np.sort(below(g, np.full(20000, x), np.full(20000, t, np.float32)))[::-1]
            bins, _ = weigh(y, x, np.float32(t))
            assert (np.diff(bins) >= 0).all(), (t, top)


@pytest.mark.parametrize("seed", range(6))
def test_weights_are_good_to_2_to_the_minus_32(weigh, seed):
    """Weights as shares of the largest logit's.  Within its bin each is off by less than 8 units of 2^-36: one for each of
    the two terms' cuts to a whole number; from the remainder up to 2^-9 of the product 0.25 for its term's rounding and
    0.17 for its own; 1 for the sum's rounding at 2^24 units; from the square term, up to 1.7e7 units, 0.5 each for the
    coefficient and the polynomial, 1 for the square and 1.95 for twice its argument's rounding; 0.02 for the 6th power.
    A weight is 0.978 of its bin's at least, so two of them are off by less than 2 * 8 * 2^-36 = 2^-32 (7.4 / 0.978 is
    below 8).  Above T = 2^100 the second float of c is denormal, off by up to 2^-150; times the 2^129 that two logits may
    lie apart, times ln 2 / 16, that is 2^-25.5 more."""
    g = np.random.default_rng(200 + seed)
    n = 300000
    x, t = logits(g, n), temperatures(g, n)
    if seed % 2:   # ordinary rows, where products are in 32 bits; next to half a bin, where most is off
        x, t = g.uniform(-40, 40, n).astype(np.float32), g.uniform(0.1, 3.0, n).astype(np.float32)
    y = below(g, x, t)
    bins, offs = weigh(y, x, t)
    _, top_offs = weigh(x, x, t)
    ld = np.longdouble
    part = (ld(1) + offs.astype(ld) * ld(2.0) ** -36) / (ld(1) + top_offs.astype(ld) * ld(2.0) ** -36)
    down = octaves16(x, y, t)
    has = bins < REST
    most = np.where(t[has] <= 2.0 ** 100, ld(2.0) ** -32, ld(2.0) ** -25)
    error = np.abs(part[has] * np.exp2((down[has] - bins[has]) / ld(16)) - 1)
    assert has.mean() > 0.3 and (error < most).all(), float((error / most).max())

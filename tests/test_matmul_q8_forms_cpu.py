"""The choice of a form and of a split of k (csrc/matmul_q8_forms.h), compiled for
the CPU: what a form cannot take is never chosen, and the sizes of the GPU tests
go to the kernels that they are there for."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from matmul_q8_sizes import SIZES

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xdna.cpp_amd", "csrc")
SRC = r"""
#include "matmul_q8_forms.h"
extern "C" int c_choose(int cus, int m, int n, int k, int64_t xs, int64_t ws) {
    const mi355x::MatmulChoice c = mi355x::choose_matmul(cus, m, n, k, xs, ws);
    return static_cast<int>(c.form) * 100 + c.splits;
}
"""
FORMS = ["few16", "few16wide", "few32", "few32wide", "far", "64x64", "64x128", "128x128", "256x128", "256x256"]


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    d = tmp_path_factory.mktemp("forms")
    (d / "forms.cpp").write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover",
                    f"-I{CSRC}", str(d / "forms.cpp"), "-o", str(d / "forms.so")], check=True)
    f = ctypes.CDLL(str(d / "forms.so")).c_choose
    f.argtypes = [ctypes.c_int] * 4 + [ctypes.c_int64] * 2

    def of(m, n, k, xs=None, ws=None, cus=256):
        c = f(cus, m, n, k, k if xs is None else xs, k if ws is None else ws)
        return FORMS[c // 100], c % 100

    return of


def test_sizes_of_the_gpu_tests(choose):
    for name, sizes in SIZES.items():
        form, _, parts = name.partition(" in ")
        for size in sizes:
            assert choose(*size) == (form, int(parts or 1)), size


@pytest.mark.parametrize("cus", [32, 64, 256, 304])
def test_only_what_a_form_can_take(choose, cus):
    rng = np.random.default_rng(cus)
    for _ in range(5000):
        m, n = (int(2 ** rng.uniform(0, 24)) for _ in range(2))
        k = 16 * int(2 ** rng.uniform(0, 13))
        form, splits = choose(m, n, k, cus=cus)
        assert form != "far" and form.startswith("few") == (m <= 32)
        if form.startswith("few"):
            assert splits == 1 and (m <= 16 or not form.startswith("few16"))
            continue
        bm, bn = map(int, form.split("x"))
        tiles = -(-m // bm) * -(-n // bn)
        assert 1 <= splits <= -(-k // 128)
        if form == "256x256":
            assert m >= 256 and n >= 256 and splits == 1
        if splits > 1:  # a counter for each tile, room for each part
            assert tiles <= 1024 and tiles * splits * bm * bn * 4 <= 64 << 20


def test_rows_far_apart_take_no_tile(choose):
    far = (1 << 23) + 16
    for m in (33, 300, 5000):
        assert choose(m, 5000, 2064, xs=1 << 23, ws=1 << 23)[0] not in ("far",)
        assert choose(m, 5000, 2064, xs=far) == ("far", 1) and choose(m, 5000, 2064, ws=far) == ("far", 1)
    assert choose(1, 5000, 2064, xs=far, ws=far) == ("few16", 1)

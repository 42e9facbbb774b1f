"""Where the recurrence's lanes read (csrc/glr_place.h), lane by lane on the host: every offset from its wave's base is
the distance in memory, for sequences that are apart, that overlap and that are one and the same."""
import ctypes
import os
import shutil
import subprocess

import pytest

import fhtest

SOURCE = r"""
#include "glr_place.h"
using namespace fhc::seq;
// the live lanes whose address is not the element's, over all waves of columns of v channels; -1: the waves' first one
extern "C" int64_t wrong_lanes(uint32_t b, uint32_t d, uint32_t v, int64_t bs, uint32_t elem, int64_t* worst) {
    const bool near = near_sequences(b, d, bs, elem);
    const uint32_t per = d / v, groups = near ? per : (per + 63) / 64 * 64;
    int64_t wrong = 0;
    *worst = 0;
    for (uint64_t w = 0; w < (uint64_t)b * groups; w += 64) {
        const uint32_t b0 = w / groups, first = (w - (uint64_t)b0 * groups) * v;
        const uint32_t c0 = base_channel(near && b > 1, first);
        const int64_t base = b0 * bs * elem + (int64_t)c0 * elem;
        for (uint32_t l = 0; l < 64; l++) {
            const uint32_t lb = (w + l) / groups, ch = (w + l - (uint64_t)lb * groups) * v;
            if (lb >= b || ch >= d) continue;
            const int64_t got = base + lane_offset(lb, ch, b0, c0, bs * elem, elem);  // extended without a sign
            const int64_t off = got - (lb * bs + ch) * elem;
            if (off) wrong++, *worst = off;
        }
    }
    return wrong;
}
"""


@pytest.fixture(scope="module")
def place(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host compiler")
    at = tmp_path_factory.mktemp("place")
    (at / "place.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(fhtest.ROOT, "flyhigh-engine_amd", "csrc"),
                    str(at / "place.cpp"), "-o", str(at / "place.so")], check=True)
    f = ctypes.CDLL(str(at / "place.so")).wrong_lanes
    f.restype = ctypes.c_int64
    f.argtypes = [ctypes.c_uint32] * 3 + [ctypes.c_int64, ctypes.c_uint32, ctypes.POINTER(ctypes.c_int64)]

    def check(b, d, v, bs, elem):
        worst = ctypes.c_int64()
        n = f(b, d, v, bs, elem, worst)
        assert n == 0, f"{n} lanes of {b} x {d} are read elsewhere, by {worst.value} bytes (sequences {bs} apart)"

    return check


@pytest.mark.parametrize("d", [1, 2, 7, 48, 64, 65, 100, 128, 192, 320, 1532, 2048, 2049])
@pytest.mark.parametrize("b", [1, 2, 4, 67])
def test_lanes_read_their_elements(place, b, d):
    for elem in (2, 4):
        for v in (1, 2) if d % 2 == 0 else (1,):
            for bs in (0, 1, d // 2, d - 1, d, d + 3, 5 * d, (1 << 24) // elem - 1, (1 << 24) // elem, 1 << 40, -d,
                       -(1 << 33)):
                place(b, d, v, bs, elem)


def test_widest_rows(place):
    """Rows whose last channel lies past 2^31 bytes, one of them or two, apart and shared."""
    for b, d, bs in ((1, (1 << 23) + 6, 0), (2, (1 << 23) + 6, 0), (2, (1 << 23) + 6, 1 << 35)):
        place(b, d, 2, bs, 1 << 9)  # an element of 512 bytes stands for 128 times the channels

"""The search for the lowest key that min-p leaves, on the host: the kernel's own header, compiled with the host compiler."""
import ctypes as C
import math
import os
import random
import shutil
import struct
import subprocess

import pytest

from simplicial_attention_b200 import build

SOURCE = r"""
#include "sa2_sample_keys.h"
#include <math.h>
#include <string.h>

static float logit_of(uint32_t key, int bf16) {
    if (bf16) key = key << 16 | (key & 0x8000u ? 0u : 0xffffu);
    const uint32_t u = key & 0x80000000u ? key ^ 0x80000000u : ~key;
    float v;
    memcpy(&v, &u, 4);
    return v;
}
extern "C" int stays(uint32_t key, float best, double least, double inv_t, int bf16) {
    return ((double)logit_of(key, bf16) - (double)best) * inv_t >= least;
}
extern "C" uint32_t search(uint32_t best_key, uint32_t near, float best, double least, double inv_t, int bf16, int *looked) {
    *looked = 0;
    return sa2::sample::first_key(best_key, near, [&](uint32_t k) {
        ++*looked;
        return stays(k, best, least, inv_t, bf16) != 0;
    });
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    folder = tmp_path_factory.mktemp("keys")
    (folder / "keys.cpp").write_text(SOURCE)
    out = str(folder / "keys.so")
    subprocess.run([shutil.which("g++") or "g++", "-shared", "-fPIC", "-O1", "-I", build.CSRC, str(folder / "keys.cpp"), "-o", out], check=True)
    lib = C.CDLL(out)
    lib.search.restype = C.c_uint32
    lib.search.argtypes = [C.c_uint32, C.c_uint32, C.c_float, C.c_double, C.c_double, C.c_int, C.POINTER(C.c_int)]
    lib.stays.argtypes = [C.c_uint32, C.c_float, C.c_double, C.c_double, C.c_int]
    return lib


def _key(v, bf16):
    u = struct.unpack("<I", struct.pack("<f", v + 0.0))[0]
    k = (~u if u & 0x80000000 else u | 0x80000000) & 0xFFFFFFFF
    return k >> 16 if bf16 else k


def _rounded(v, bf16):
    v = struct.unpack("<f", struct.pack("<f", v))[0]
    return struct.unpack("<f", struct.pack("<I", struct.unpack("<I", struct.pack("<f", v))[0] & 0xFFFF0000))[0] if bf16 else v


def _search(lib, best, temperature, min_p, bf16):
    best, inv_t, least = _rounded(best, bf16), 1.0 / temperature, math.log(min(min_p, 1.0))
    about = best + least * temperature
    near = _key(_rounded(about, False), bf16) if abs(about) < 3.4e38 else 0
    looked, top = C.c_int(), _key(best, bf16)
    got = lib.search(top, near, best, least, inv_t, bf16, C.byref(looked))
    assert got <= top and lib.stays(got, best, least, inv_t, bf16)
    assert got == 0 or not lib.stays(got - 1, best, least, inv_t, bf16)
    return looked.value


# the floor lies at a logit of about 0, where neighbouring numbers are no longer told apart next to the best one
@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("best, temperature, min_p", [(5.0, 1.0, math.exp(-5)), (1.0, 1 / math.log(2), 0.5), (7.0, 0.7, math.exp(-10)), (1.0, 1.0, math.exp(-1)),
                                                      (64.0, 8.0, math.exp(-8)), (0.0, 1.0, 1.0), (-3.0, 1.0, 1.0), (1e-45, 1.0, 1.0), (3e38, 1e38, math.exp(-3))])
def test_floors_at_zero(lib, best, temperature, min_p, bf16):
    assert _search(lib, best, temperature, min_p, bf16) <= 64


@pytest.mark.parametrize("bf16", [0, 1])
def test_floors_anywhere(lib, bf16):
    rng = random.Random(5)
    for _ in range(2000):
        best = rng.choice((1, -1)) * math.exp(rng.uniform(-20, 20))
        temperature, min_p = math.exp(rng.uniform(-10, 10)), math.exp(-rng.uniform(0, 40))
        assert _search(lib, best, temperature, min_p, bf16) <= 64
        # the settings for which the floor is at 0 to the last bits
        assert _search(lib, abs(best), temperature, max(math.exp(-abs(_rounded(best, bf16)) / temperature), 1e-300), bf16) <= 64


def test_any_guess(lib):
    looked = C.c_int()
    for near in (0, 1, 0x7FFFFFFF, 0x80000000, 0x80000001, _key(4.999, 0), _key(5.0, 0), 0xFFFFFFFF):
        got = lib.search(_key(5.0, 0), near, 5.0, -1.0, 1.0, 0, C.byref(looked))
        assert got == _key(4.0, 0) and looked.value <= 64

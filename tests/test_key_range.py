"""The threshold search of the page selection in whole numbers, on the CPU: the
kernel's own range arithmetic (csrc/key_range.h, compiled here) with a plain
histogram gives the threshold that sorting gives, in at most four rounds, also
where scores of minus infinity put the last bin within a bin's width of 0."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "iris-kernel_b200", "csrc")
SOURCE = """
#include "key_range.h"
using iris::KeyRange;
extern "C" int rounds() { return iris::kRangeRounds; }
extern "C" void bins_of(uint32_t low, uint32_t high, int shift, const uint32_t* keys, int n, int32_t* bin) {
  const KeyRange r = {low, high};
  for (int i = 0; i < n; ++i) bin[i] = r.holds(keys[i]) ? static_cast<int32_t>(r.bin(keys[i], shift)) : -1;
}
extern "C" void narrowed(uint32_t* low, uint32_t* high, uint32_t index, int shift) {
  KeyRange r = {*low, *high};
  r.narrow(index, shift);
  *low = r.low, *high = r.high;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    cxx = os.environ.get("CXX", "g++")
    if shutil.which(cxx) is None:
        pytest.skip("no C++ compiler")
    at = tmp_path_factory.mktemp("key_range")
    (at / "r.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-std=c++17", "-shared", "-fPIC", "-I", CSRC, str(at / "r.cpp"), "-o", str(at / "r.so")],
                   check=True)
    return ctypes.CDLL(str(at / "r.so"))


def _ordered(x):
    """fp32 -> unsigned with the same order, as the scores are stored."""
    u = (np.asarray(x, np.float32) + np.float32(0)).view(np.uint32)
    return np.where(u >> 31, ~u, u | np.uint32(0x80000000)).astype(np.uint32)


def _search(lib, keys, need):
    """(threshold, how many equal to it are wanted): keys above it are taken."""
    low, high = ctypes.c_uint32(int(keys.min())), ctypes.c_uint32(int(keys.max()))
    bins = np.empty(len(keys), np.int32)
    for _ in range(lib.rounds()):
        assert low.value <= high.value
        shift = max((high.value - low.value).bit_length() - 8, 0)
        lib.bins_of(low, high, shift, keys.ctypes.data_as(ctypes.c_void_p), len(keys),
                    bins.ctypes.data_as(ctypes.c_void_p))
        assert bins.max() < 256
        counts = np.bincount(bins[bins >= 0], minlength=256)
        index = int(np.argmax(np.cumsum(counts) >= need))
        need -= int(counts[:index].sum())
        lib.narrowed(ctypes.byref(low), ctypes.byref(high), index, shift)
        if counts[index] == need:
            return low.value - 1, 0
        if shift == 0:
            return low.value, need
    raise AssertionError("the search has not ended")


INF = np.float32(np.inf)
SETS = {
    "few large among -inf": np.concatenate([np.full(297, -INF), np.ones(3)]),
    "inf among -inf": np.concatenate([np.full(297, -INF), np.full(3, INF)]),
    "all there is": np.concatenate([np.full(60, -INF), np.full(60, INF), np.linspace(-3e38, 3e38, 80), np.zeros(30)]),
    "next to -inf": np.concatenate([np.full(50, -INF), -3.4e38 * (1 - np.arange(50) / 1e5), [1e-30, 2.0, INF]]),
    "small numbers": np.random.default_rng(0).standard_normal(300) * 1e-40,
    "ordinary": np.random.default_rng(1).standard_normal(300),
    "one": np.full(20, 0.25),
}


@pytest.mark.parametrize("name", SETS)
def test_threshold_for_every_budget(lib, name):
    keys = _ordered(SETS[name])
    down = np.sort(keys.astype(np.int64))[::-1]
    for need in range(1, len(keys)):
        thr, equal = _search(lib, keys, need)
        above = int((keys > thr).sum())
        assert above + equal == need and equal <= int((keys == thr).sum())
        assert set(down[:above].tolist()) == set(keys[keys > thr].tolist())


def test_threshold_among_random_keys(lib):
    rng = np.random.default_rng(2)
    for _ in range(200):
        bits = rng.integers(1, 33)
        keys = rng.integers(0x007fffff, 0x007fffff + min(2 ** int(bits), 0xff000000), 64).astype(np.uint32)
        need = int(rng.integers(1, 64))
        thr, equal = _search(lib, keys, need)
        assert int((keys > thr).sum()) + equal == need and equal <= int((keys == thr).sum())

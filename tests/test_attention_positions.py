"""The plan of the attention over the pages (csrc/attn_plan.hpp), compiled by itself: the first position that any
part asks the block table for, before a row's limit is known, fits 32 bits whatever a table row holds."""

import ctypes
import os
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "cq-pretrain_amd" / "csrc"
SOURCE = """
#include "attn_plan.hpp"
extern "C" void plan(int64_t N, int kv, int group, int D, int most, int64_t capacity, int window, int64_t* out) {
  const cqgdn::AttendPlan p = cqgdn::attend_plan(N, kv, group, D, most, capacity, window);
  out[0] = p.tiles;
  out[1] = p.splits;
  out[2] = p.per;
  out[3] = cqgdn::kWaves;
  out[4] = cqgdn::kStep;
  out[5] = cqgdn::kMaxSplits;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = os.environ.get("CXX", "g++")
    if shutil.which(cxx) is None:
        pytest.skip("no C++ compiler")
    where = tmp_path_factory.mktemp("plan")
    (where / "plan.cpp").write_text(SOURCE)
    lib = where / "plan.so"
    subprocess.run([cxx, "-O1", "-std=c++17", "-shared", "-fPIC", f"-I{CSRC}", str(where / "plan.cpp"), "-o", str(lib)],
                   check=True, capture_output=True, text=True)
    f = ctypes.CDLL(str(lib)).plan

    def call(N, kv, group, D, most, capacity, window=0):
        out = (ctypes.c_int64 * 6)()
        f(ctypes.c_int64(N), kv, group, D, most, ctypes.c_int64(capacity), window, out)
        return dict(zip(("tiles", "splits", "per", "waves", "step", "most"), out))

    return call


ROOM = 2 ** 31 - 1 - 1024  # positions that can be seen


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("columns,page", [(40000, 65536), (65536, 65536), (2 ** 31 - 1, 65536), (2 ** 27, 16),
                                          (2 ** 27 - 64, 16), (2 ** 31 - 1, 16), (32768, 65536), (4096, 16), (1, 16), (0, 16)])
def test_the_parts_positions_fit_32_bits(plan, D, columns, page):
    for N, kv, group, most in ((1, 1, 1, 1), (1, 4, 4, 1), (3, 8, 1, 2), (64, 4, 4, 1), (1, 1, 16, 3), (5000, 8, 8, 1)):
        p = plan(N, kv, group, D, most, columns * page)
        assert not p["tiles"] and 1 <= p["splits"] <= p["most"]
        last = ((p["splits"] - 1) * p["per"] + p["waves"] - 1) * p["step"]
        assert last <= 2 ** 31 - 1, (N, kv, p)
        # and the parts cover what can be seen
        assert p["splits"] * p["per"] * p["step"] >= min(columns * page, ROOM)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_windows_take_no_more_parts_than_the_workspace_is_for(plan, D):
    for capacity in (16, 1000, 100000, 40000 * 65536):
        for N, most in ((1, 1), (64, 1), (1, 4), (1, 300), (7, 60)):
            whole = plan(N, 4, 4, D, most, capacity)["splits"]
            for window in (1, 100, 5000, 2 ** 31 - 1):
                p = plan(N, 4, 4, D, most, capacity, window)
                assert 1 <= p["splits"] <= whole

"""Index arithmetic of the kernels of few rows (csrc/attn_rows_plan.hpp), compiled for the host."""
import ctypes
import subprocess
from pathlib import Path

import pytest


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    csrc = Path(__file__).resolve().parent.parent / "hybrid-model-factory_amd" / "csrc"
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text('''
#include "attn_rows_plan.hpp"
using namespace hmx::attn::rows;
extern "C" int half16(int b, int e, int t, int w, int h) { return half_row<4, 16>(b, e, t, w, h); }
extern "C" int half32(int b, int e, int t, int w, int h) { return half_row<4, 32>(b, e, t, w, h); }
''')
    subprocess.run(["g++", "-std=c++17", "-O1", "-fwrapv", "-shared", "-fPIC", f"-I{csrc}", "-o",
                    str(d / "plan.so"), str(d / "plan.cpp")], check=True)
    return ctypes.CDLL(str(d / "plan.so"))


@pytest.mark.parametrize("KT", [16, 32])
@pytest.mark.parametrize("end", [1, 16, 17, 700, 1 << 20, (1 << 31) - 8192, (1 << 31) - 8191, (1 << 31) - 272, (1 << 31) - 257])
def test_rows_asked_for_ahead_lie_in_the_table(plan, KT, end):
    """64 halves past a share's last turn too, at the most keys that a table row may hold."""
    f, NH = getattr(plan, f"half{KT}"), KT // 16
    for beg in {0, max(end - 64, 0) & ~63, max(end - 100000, 0) & ~63}:
        turns = -(-(end - beg) // (4 * KT))
        for turn in {0, 1, turns // 2, *range(max(turns - 2, 0), turns + 64 // NH + 2), turns + 2 * (64 // NH)}:
            for wave in range(4):
                for half in range(NH):
                    assert f(beg, end, turn, wave, half) == min(beg + (turn * 4 + wave) * KT + 16 * half, (end - 1) // 16 * 16)

"""CPU checks of what the host side keeps per device (csrc/per_device.h), compiled alone with a query that fails at first."""

from __future__ import annotations

import pathlib
import re
import subprocess

CSRC = pathlib.Path(__file__).resolve().parents[1] / "lczero_triton_b200" / "csrc"

PROGRAM = r"""
#include "per_device.h"
#include <cstdio>
static lc0b200::PerDeviceNumber kept;  // as beside a launch: zeros
int main() {
  int asked = 0;
  auto fails = [&] { ++asked; return 0; };
  auto gives = [&] { ++asked; return 168; };
  std::printf("%d ", lc0b200::ask_once(kept, 3, fails));
  std::printf("%d ", lc0b200::ask_once(kept, 3, gives));
  std::printf("%d ", lc0b200::ask_once(kept, 3, fails));
  std::printf("%d ", lc0b200::ask_once(kept, 4, fails));
  std::printf("%d ", lc0b200::ask_once(kept, 4, gives));
  std::printf("%d\n", asked);
}
"""


def test_a_failed_query_is_not_kept_and_devices_are_asked_apart(tmp_path) -> None:
    (tmp_path / "program.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", "-o", str(tmp_path / "program"),
                    str(tmp_path / "program.cpp")], check=True)
    out = subprocess.run([str(tmp_path / "program")], capture_output=True, text=True, check=True).stdout.split()
    #                fails, kept,  kept,  fails, kept, queries: the third call asks nothing
    assert out == ["0", "168", "168", "0", "168", "4"]


def test_the_pair_tile_asks_per_device_and_falls_back() -> None:
    text = (CSRC / "gemm_fp8.cu").read_text()
    assert not re.search(r"static const int\s+launch_regs", text), "one answer for all devices and for ever"
    split = text[text.index("PerDeviceNumber"):]
    split = split[:split.index("ceil_div_ll(g.m, kBM * CTAS)")]
    assert re.search(r"== 0\) return LC0B200_ERR_CUDA;", split), "a query that failed is an error of the device"
    assert re.search(r"< T::kLaunchRegs\) return launch<128, 1, ACT>\(g, stream\);", split)

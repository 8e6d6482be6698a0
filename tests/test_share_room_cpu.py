"""Joining the shares of a request's keys within the launch: no counter serves two steps, on devices of any number of compute units."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hecbench_amd", "csrc")
# As the kernels go about it: of more than kJoin shares every kTeam are joined by the last of them, counted where the first one's place is; then
# what is left, `unit` shares each, likewise.
PROGRAM = """
#include <cstdio>
#include <set>
#include "attend.h"
int main() {
  for (int cus = 1; cus <= 2048; ++cus)
    for (int heads : {1, 2, 3, 8}) {
      std::set<int64_t> counters;
      int64_t n = share_room(cus, heads), unit = 1;
      if (n < 1) return printf("%d units, %d heads: no share", cus, heads), 1;
      for (; n > kJoin; n = (n + kTeam - 1) / kTeam, unit *= kTeam)
        for (int64_t team = 0; team * kTeam < n; ++team)
          if (!counters.insert(team * kTeam * unit).second) return printf("%d units, %d heads: counter %d twice", cus, heads, (int)(team * kTeam * unit)), 1;
    }
  return 0;
}
"""


def test_no_counter_twice(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    source, program = tmp_path / "room.hip", tmp_path / "room"
    source.write_text(PROGRAM)
    subprocess.run([hipcc, "-w", "-O1", "-std=c++17", "--offload-host-only", "-I", CSRC, str(source), "-o", str(program)], check=True, timeout=300)
    run = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout

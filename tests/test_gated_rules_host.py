"""Where weight gradients of 16 bits go past the caches, asked of the rule on the host."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
MIB = 1 << 20

PROGRAM = """
#include "%s/unit_amd/csrc/gated.hpp"
#include <cstdio>
int main(int argc, char **argv) {
  for (int i = 1; i + 2 < argc; i += 3) printf("%%d", (int)unit::dw_past_caches(strtoull(argv[i], 0, 10), strtoull(argv[i + 1], 0, 10), atoi(argv[i + 2])));
}
"""


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_weight_gradients_past_the_caches(tmp_path):
    src, exe = tmp_path / "rule.hip", tmp_path / "rule"
    src.write_text(PROGRAM % ROOT)
    subprocess.check_call([HIPCC, "-std=c++17", "-O1", "--offload-arch=gfx950", "--offload-host-only", "-w", str(src), "-o", str(exe)])
    cases = [  # dw, bytes moved, pre-activations kept
        (40 * MIB, 90 * MIB, 0, 1), (40 * MIB - 1, 600 * MIB, 0, 0), (40 * MIB - 1, 600 * MIB, 1, 0), (40 * MIB, 280 * MIB - 1, 1, 0), (40 * MIB, 280 * MIB, 1, 1),
        (128 * MIB, 268 * MIB, 1, 0), (1 << 34, 1 << 36, 1, 1)]
    got = subprocess.check_output([str(exe), *(str(v) for c in cases for v in c[:3])], text=True)
    assert got == "".join(str(c[3]) for c in cases)

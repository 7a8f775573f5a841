"""Which MXFP4 products of few rows take the kernel that reaches its scales by 32-bit offsets, asked of its rule on the host: no device, no
weights."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

PROGRAM = """
#include "%s/unit_amd/csrc/grouped_split.hpp"
#include <cstdio>
// rows, groups, N (of the result), halves -> whether the product is of few rows
int main(int argc, char **argv) {
  for (int i = 1; i + 3 < argc; i += 4) {
    unit::GroupedParams p{};
    const int sizes = 0;
    p.sizes = &sizes, p.rows = atoi(argv[i]), p.groups = atoi(argv[i + 1]), p.n = atoi(argv[i + 2]);
    printf("%%d", (int)unit::grouped_split_pays(p, atoi(argv[i + 3])));
  }
}
"""


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_the_scales_of_all_groups_are_within_32_bits(tmp_path):
    """Four bytes a row, the second plane behind all rows of the first, sixteen rows at a time: 4 (rows + 16) bytes lie in a descriptor of
    2^31 - 1."""
    src = tmp_path / "rule.hip"
    src.write_text(PROGRAM % ROOT)
    exe = tmp_path / "rule"
    subprocess.check_call([HIPCC, "-std=c++17", "-O1", "--offload-arch=gfx950", "--offload-host-only", "-w", str(src), "-o", str(exe)])
    cases = [(1, 1 << 16, 4096, 1, 1), (1, 1 << 16, 4096, 2, 0), (1, (1 << 16) - 1, 4096, 2, 1), (1, 1 << 17, 4096, 1, 0), (1, (1 << 17) - 1, 4096, 1, 1),
             (1, 1 << 17, 4096, 2, 0), (1, 1 << 20, 512, 1, 0), (1, 1 << 20, 256, 2, 0), (16, 64, 512, 2, 1), (17, 64, 512, 2, 0), (1, 1 << 20, 255, 2, 1), (1, 1, (1 << 22), 1, 0),
             (1, (1 << 29) // 24, 24, 1, 0), (1, (1 << 29) // 24 - 1, 24, 1, 1), (1, (1 << 29) // 24 - 1, 12, 2, 1), (1, (1 << 29) // 24, 12, 2, 0)]
    assert all(4 * (c[1] * c[2] * c[3] + 16) <= (1 << 31) - 1 for c in cases if c[4])
    got = subprocess.check_output([str(exe), *(str(v) for c in cases for v in c[:4])], text=True)
    assert got == "".join(str(c[4]) for c in cases)

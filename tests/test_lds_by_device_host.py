"""More than 64 KiB of LDS is granted to a kernel device by device: asked for once on each, with the runtime's two calls replaced."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

PROGRAM = """
#include <hip/hip_runtime.h>
#include <cstdio>
static int device = 0, granted[128], refuse = 0;
static hipError_t device_now(int *d) { return *d = device, hipSuccess; }
static hipError_t grant(const void *, hipFuncAttribute, int) { return refuse ? hipErrorInvalidValue : (++granted[device], hipSuccess); }
#define hipGetDevice device_now
#define hipFuncSetAttribute grant
#include "%s/unit_amd/csrc/grouped.hpp"
namespace unit { char *error_buf() { static char text[256]; return text; } }
int main() {
  unsigned long long allowed = 0;
  const int order[] = {0, 0, 1, 0, 1, 63, 63, 1, 70, 70};
  for (int d : order) {
    device = d;
    if (unit::allow_lds("test", nullptr, &allowed)) return 1;
  }
  printf("%%d %%d %%d %%d", granted[0], granted[1], granted[63], granted[70]);
  device = 2, refuse = 1;
  if (!unit::allow_lds("test", nullptr, &allowed)) return 2;
  refuse = 0;
  if (unit::allow_lds("test", nullptr, &allowed)) return 3;
  printf(" %%d", granted[2]);
}
"""


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_every_device_grants_once(tmp_path):
    src, exe = tmp_path / "lds.hip", tmp_path / "lds"
    src.write_text(PROGRAM % ROOT)
    subprocess.check_call([HIPCC, "-std=c++17", "-O1", "--offload-arch=gfx950", "--offload-host-only", "-w", str(src), "-o", str(exe)])
    assert subprocess.check_output([str(exe)], text=True) == "1 1 1 2 1"

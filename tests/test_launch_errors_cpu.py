"""What a launch that fails on the host returns through the native entry points: never 0."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "gcore_b200" / "ops" / "csrc"

# A runtime whose launches fail with an error that the next question takes off, or with one that no question shows.
PROGRAM = r"""
#include <cuda_runtime.h>
static cudaError_t pending = cudaSuccess, result = cudaSuccess;
static bool shown = true;
static cudaError_t fake_last() { const cudaError_t e = pending; pending = cudaSuccess; return e; }
template <typename... T>
static cudaError_t fake_launch(const cudaLaunchConfig_t*, void (*)(T...), T...) { pending = shown ? result : cudaSuccess; return result; }
#define cudaGetLastError fake_last
#define cudaLaunchKernelEx fake_launch
#include "host_utils.h"
__global__ void nothing(int) {}
static int one() { return gk::launch_ex(cudaLaunchConfig_t{}, nothing, 1); }
static int two() { return gk::launch_waiting(nothing, 1, 32, static_cast<cudaStream_t>(nullptr), 1); }
int main() {
  for (int (*launch)() : {one, two}) {
    result = cudaSuccess;
    printf("%d ", launch());
    result = cudaErrorInvalidConfiguration;
    printf("%d %d ", launch(), gk::launch_status());
    shown = false;
    printf("%d ", launch());
    shown = true;
  }
  return 0;
}
"""


def test_a_failed_launch_is_reported(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        pytest.skip("needs nvcc")
    (tmp_path / "t.cu").write_text(PROGRAM)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", str(CSRC), "-o", str(tmp_path / "t"),
                    str(tmp_path / "t.cu")], check=True, capture_output=True)
    out = subprocess.run([str(tmp_path / "t")], check=True, capture_output=True, text=True).stdout
    assert out.split() == ["0", "9", "0", "9"] * 2   # cudaErrorInvalidConfiguration is 9


def test_the_status_is_asked_once():
    """The first question takes the error off the runtime; the answer to a second one would be that all is well."""
    for f in sorted(CSRC.glob("*.cu")):
        for line in f.read_text().splitlines():
            assert line.count("launch_status()") <= 1, (f.name, line.strip())

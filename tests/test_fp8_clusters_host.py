"""How many clusters fit is asked on every device, and a query that failed is made again (csrc/gemm_fp8.cu: clusters_that_fit): the function as the
source has it, over a runtime of which the number of devices and what it answers are given."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
RUNTIME = r"""
#include <atomic>
#include <cstdio>
#include <cstdlib>
#define __global__
struct dim3 { unsigned x, y, z; dim3(unsigned a = 1, unsigned b = 1, unsigned c = 1) : x(a), y(b), z(c) {} };
enum { cudaSuccess = 0, cudaLaunchAttributeClusterDimension = 4, cudaFuncAttributeMaxDynamicSharedMemorySize = 8 };
struct cudaLaunchAttribute { int id; struct { struct { unsigned x, y, z; } clusterDim; } val; };
struct cudaLaunchConfig_t { dim3 gridDim, blockDim; size_t dynamicSmemBytes; void* stream; cudaLaunchAttribute* attrs; unsigned numAttrs; };
static int device = 0, fails = 0, asked = 0;
static int cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
template <typename F> static int cudaFuncSetAttribute(F, int, int) { return cudaSuccess; }
template <typename F> static int cudaOccupancyMaxActiveClusters(int* n, F, cudaLaunchConfig_t* c) {
  ++asked;
  if (fails) return 2;
  *n = (device == 1 ? 66 : 74) * (c->dynamicSmemBytes < 120000 ? 4 : 2) / c->attrs[0].val.clusterDim.x;
  return cudaSuccess;
}
static int cudaGetLastError() { return 0; }
static int num_sms() { return 100; }
constexpr int FL_MAX_SPLITS = 8;
"""
MAIN = r"""
int main() {
  const int whole = F8_WHOLE_SM, half = F8_HALF_SM;
  auto is = [](int have, int want, const char* what) { if (have != want) { std::printf("%s: %d, not %d\n", what, have, want); std::exit(1); } };
  fails = 1;
  is(clusters_that_fit(2, whole, 384), 50, "by SMs where the query fails");
  fails = 0;
  is(clusters_that_fit(2, whole, 384), 74, "asked again behind a failure");
  is(clusters_that_fit(2, half, 192), 148, "two CTAs to an SM");
  device = 1;
  is(clusters_that_fit(2, whole, 384), 66, "another device");
  device = 0;
  is(clusters_that_fit(2, whole, 384), 74, "the first again");
  const int before = asked;
  is(clusters_that_fit(2, half, 192), 148, "kept");
  is(asked, before, "asked once");
  device = 5000;
  is(clusters_that_fit(2, whole, 384), 74, "a device beyond the list");
  std::puts("fine");
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_clusters_of_each_device(tmp_path):
    with open(os.path.join(ROOT, "llmq_b200", "csrc", "gemm_fp8.cu")) as f:
        source = f.read()
    part = re.search(r"__global__ void fp8_probe_kernel\(\) \{\}.*?\nstatic int clusters_that_fit\(.*?\n}\n", source, re.S).group(0)
    (tmp_path / "t.cpp").write_text(RUNTIME + part + MAIN)
    subprocess.run(["g++", "-std=c++17", "-o", str(tmp_path / "t"), str(tmp_path / "t.cpp")], check=True, capture_output=True, text=True)
    r = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout

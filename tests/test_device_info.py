"""device_info.cuh without a GPU: the shared-memory limit of a kernel that two threads launch with different sizes, against
a stand-in for the CUDA runtime whose cudaFuncSetAttribute can be held up."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

RUNTIME = r"""
#pragma once
#include <chrono>
#include <thread>
typedef int cudaError_t;
enum { cudaSuccess = 0 };
enum { cudaDevAttrMaxSharedMemoryPerMultiprocessor, cudaDevAttrMaxSharedMemoryPerBlockOptin, cudaDevAttrMultiProcessorCount };
enum { cudaFuncAttributeMaxDynamicSharedMemorySize };
static int g_limit = 49152, g_calls = 0;
inline int cudaGetDevice(int* d) { *d = 0; return 0; }
inline int cudaGetLastError() { return 0; }
inline int cudaDeviceGetAttribute(int* v, int, int) { *v = 232448; return 0; }
template <class K>
int cudaFuncSetAttribute(K, int, int bytes) {
    g_limit = bytes;
    g_calls++;
    if (bytes == 230000) std::this_thread::sleep_for(std::chrono::milliseconds(400));  // the larger one returns last
    return 0;
}
"""

MAIN = r"""
#include <cstdio>
#include "device_info.cuh"
void kern() {}
int main() {
    static std::atomic<int> granted[kMaxDevices];
    (void)device_info();
    std::thread a([] { ensure_smem(kern, 230000, granted); });
    std::this_thread::sleep_for(std::chrono::milliseconds(100));
    std::thread b([] { ensure_smem(kern, 200000, granted); });
    a.join();
    b.join();
    // what a later launch of 230 000 bytes finds
    ensure_smem(kern, 230000, granted);
    printf("%d %d %d\n", g_limit, (int)granted[0], g_calls);
    return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_two_threads_ask_for_different_sizes(tmp_path):
    (tmp_path / "cuda_runtime.h").write_text(RUNTIME)
    (tmp_path / "main.cpp").write_text(MAIN)
    exe = str(tmp_path / "main")
    subprocess.run(["g++", "-std=c++17", "-pthread", "-I", str(tmp_path), "-I", os.path.join(ROOT, "mantle_b200", "csrc"),
                    str(tmp_path / "main.cpp"), "-o", exe], check=True)
    limit, granted, calls = map(int, subprocess.run([exe], check=True, capture_output=True, text=True, timeout=20).stdout.split())
    assert limit == granted == 230000 and calls == 1

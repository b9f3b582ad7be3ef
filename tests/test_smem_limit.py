"""A kernel's shared-memory limit under two host threads: what is recorded is never more than what is set."""

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "reflex_b200", "csrc")

# The driver's calls are stood in for; the first caller's is slow to come back.
PROGRAM = r"""
#include "smem_limit.h"
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
static std::atomic<int> set{0}, calls{0};
extern "C" cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int v) {
    set = v;
    if (calls++ == 0) std::this_thread::sleep_for(std::chrono::milliseconds(300));
    return cudaSuccess;
}
int main() {
    static rfx::SmemLimit limit;
    std::thread a([] { limit.raise((const void*)main, 150000); });
    std::this_thread::sleep_for(std::chrono::milliseconds(100));
    std::thread b([] { limit.raise((const void*)main, 60000); });
    a.join(), b.join();
    std::printf("%d %d\n", (int)set, limit.have[0]);
}
"""


def test_two_threads_with_different_sizes(tmp_path):
    from reflex_b200.csrc.build import find_nvcc

    include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(find_nvcc()))), "include")
    if not shutil.which("g++") or not os.path.exists(os.path.join(include, "cuda_runtime_api.h")):
        pytest.skip("no host compiler, or no headers")
    source, binary = tmp_path / "limit.cpp", tmp_path / "limit"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-pthread", "-I", CSRC, "-I", include, str(source), "-o", str(binary)], check=True,
                   timeout=120)
    attribute, recorded = map(int, subprocess.run([str(binary)], check=True, capture_output=True, text=True, timeout=60).stdout.split())
    assert attribute >= recorded == 150000

"""The limit of dynamic shared memory that a kernel's launches share: two threads that raise it to different sizes
must not leave it at the smaller one.  Compiled for the host, with a stand-in for the runtime call that holds
the larger request back until the smaller one has been made (or is found to wait for it)."""

import os
import shutil
import subprocess

import pytest

from morphottention_b200.build import CUDA_HOME, CSRC

PROGRAM = r"""
#include <chrono>
#include <cstdio>
#include <thread>
#include "host_common.h"

static std::atomic<int> attribute{48 * 1024}, calls{0};
static std::atomic<bool> large_in{false}, small_done{false};

extern "C" cudaError_t CUDARTAPI cudaFuncSetAttribute(const void*, cudaFuncAttribute, int bytes) {
    ++calls;
    attribute = bytes;
    if (bytes == 200 * 1024) {  // the other thread may run now
        large_in = true;
        for (int i = 0; i < 300 && !small_done; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
    }
    return cudaSuccess;
}

int main() {
    static morpho::SharedLimit limit;
    const void* kernel = nullptr;
    std::thread large([&] { limit.raise(kernel, 0, 200 * 1024); });
    std::thread small([&] {
        while (!large_in) std::this_thread::yield();
        limit.raise(kernel, 0, 100 * 1024);
        small_done = true;
    });
    large.join();
    small.join();
    limit.raise(kernel, 0, 150 * 1024);  // a launch between the two sizes
    std::printf("%d", attribute.load());
    if (attribute < 150 * 1024) return 1;
    const int before = calls;
    limit.raise(kernel, 0, 200 * 1024);
    limit.raise(kernel, 0, 1024);
    if (calls != before) return 2;         // no further calls
    limit.raise(kernel, 1, 64 * 1024);     // another device has its own limit
    return calls == before + 1 ? 0 : 3;
}
"""


def test_two_threads_raise_one_limit(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    (tmp_path / "limit.cpp").write_text(PROGRAM)
    exe = str(tmp_path / "limit")
    subprocess.run([compiler, "-std=c++17", "-pthread", "-I", CSRC, "-I", os.path.join(CUDA_HOME, "include"),
                    str(tmp_path / "limit.cpp"), "-o", exe], check=True)
    assert subprocess.run([exe], timeout=60).returncode == 0

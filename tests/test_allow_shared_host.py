"""Two threads ask for shared memory for one kernel, by the header's own code over a runtime that is not there (no GPU)."""
import subprocess

from nnis_b200.csrc import build

PROGRAM = r"""
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdio.h>
#include <unistd.h>
#include <atomic>
#include <thread>
static std::atomic<int> granted{0};
static cudaError_t device_0(int* d) { *d = 0; return cudaSuccess; }
static cudaError_t grant(int bytes) {
    if (bytes < 1000) usleep(300000);  // (the smaller request arrives last)
    granted = bytes;
    return cudaSuccess;
}
#define cudaGetDevice(d) device_0(d)
#define cudaFuncSetAttribute(kernel, attribute, bytes) grant(bytes)
#include "common.cuh"
static void kernel(int) {}
int main() {
    static std::atomic<int> held[16];
    std::thread small([&] { nnis::allow_shared(kernel, 500, held); });
    usleep(50000);
    std::thread large([&] { nnis::allow_shared(kernel, 2000, held); });
    small.join();
    large.join();
    printf("%d\n", granted.load());
    return nnis::allow_shared(kernel, 700, held) == cudaSuccess && granted == 2000 ? 0 : 1;
}
"""


def test_the_larger_request_of_two_threads_stands(tmp_path):
    source, program = tmp_path / "ask.cu", tmp_path / "ask"
    source.write_text(PROGRAM)
    subprocess.run([build.find_nvcc(), *build.ARCH_FLAGS, "-std=c++17", "-I", build.HERE, "-o", str(program), str(source),
                    "-lpthread"], check=True, capture_output=True, timeout=300)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, f"{done.stdout.strip()} bytes stand"

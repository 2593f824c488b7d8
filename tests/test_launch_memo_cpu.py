"""The memo of shared-memory opt-ins against a fake driver: api.cu compiled into a small program without a GPU."""
import subprocess

import pytest

from rgd_triton_b200 import build

PROGRAM = r"""
#include <cstdio>
#include <map>
#include <utility>
#include "common.cuh"

static int device = 0, calls = 0;
static bool fails = false;
static std::map<std::pair<int, const void *>, int> limit;       // as the driver keeps it: the last value set

static cudaError_t fake_get_device(int *dev) { *dev = device; return cudaSuccess; }
static cudaError_t fake_set(const void *kernel, cudaFuncAttribute, int bytes) {
    ++calls;
    if (fails) return cudaErrorInvalidValue;
    limit[{device, kernel}] = bytes;
    return cudaSuccess;
}
#define cudaGetDevice fake_get_device
#define cudaFuncSetAttribute fake_set
#include "api.cu"

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

int main() {
    int a, b;
    const void *ka = &a, *kb = &b;
    auto ask = [](const void *k, size_t bytes) { return rgd::ensure_dyn_smem(k, bytes); };
    CHECK(ask(ka, 100000) == 0 && limit[std::make_pair(0, ka)] == 100000);
    CHECK(ask(ka, 60000) == 0 && limit[std::make_pair(0, ka)] >= 60000);
    CHECK(ask(ka, 100000) == 0 && limit[std::make_pair(0, ka)] >= 100000);      // a smaller request takes nothing back
    CHECK(ask(ka, 150000) == 0 && limit[std::make_pair(0, ka)] == 150000);
    const int before = calls;
    CHECK(ask(ka, 150000) == 0 && ask(ka, 100000) == 0 && calls == before);      // answered without the driver
    CHECK(ask(kb, 70000) == 0 && limit[std::make_pair(0, kb)] == 70000);
    device = 1;
    CHECK(ask(ka, 60000) == 0 && limit[std::make_pair(1, ka)] == 60000 && limit[std::make_pair(0, ka)] == 150000);
    fails = true;
    CHECK(ask(ka, 90000) == RGD_E_CUDA_BASE + (int)cudaErrorInvalidValue);
    fails = false;
    CHECK(ask(ka, 90000) == 0 && limit[std::make_pair(1, ka)] == 90000);         // an error is not remembered
    return 0;
}
"""


def test_a_smaller_request_leaves_the_larger_limit(tmp_path):
    try:
        nvcc = build._nvcc()
    except RuntimeError:
        pytest.skip("no nvcc")
    source, program = tmp_path / "memo.cu", tmp_path / "memo"
    source.write_text(PROGRAM)
    made = subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", f"-I{build.CSRC}", f"-I{build.INCLUDE}",
                           str(source), "-o", str(program)], capture_output=True, text=True)
    assert made.returncode == 0, made.stdout + made.stderr
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout

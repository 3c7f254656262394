"""Barriers of the row kernels, counted on the CPU: the kernel's own source is compiled for the host and run thread by thread, with a
__syncthreads that only counts.  Every thread of a workgroup has to meet the same number, whatever the rows leave over in the last one
(values mean nothing here: a shuffle returns the caller's own)."""
import os
import shutil
import subprocess

import pytest

import adcdiff

CSRC = os.path.join(os.path.dirname(os.path.abspath(adcdiff._lib.__file__)), "csrc")
CLANG = shutil.which("clang++") or "/opt/rocm/llvm/bin/clang++"

COMMON = r"""
#pragma once
#include <math.h>
#include <algorithm>
#include <cstdint>
#define __device__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static
#define ADCDIFF_F32 0
#define ADCDIFF_BF16 1
#define ADCDIFF_OK 0
#define ADCDIFF_E_LAUNCH -3
struct Dim { unsigned x, y, z; };
static Dim threadIdx, blockIdx, gridDim;
static long long met;
static inline void __syncthreads() { ++met; }
template <typename T> static inline T __shfl_xor(T v, int) { return v; }
enum hipError_t { hipSuccess };
enum { hipFuncAttributeMaxDynamicSharedMemorySize };
static inline hipError_t hipGetDevice(int*) { return hipSuccess; }
static inline hipError_t hipFuncSetAttribute(const void*, int, int) { return hipSuccess; }
static inline const char* hipGetErrorString(hipError_t) { return ""; }
namespace adcdiff {
using std::max;
using std::min;
typedef __bf16 bf16_t;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
static inline int fail(int code, const char*, ...) { return code; }
template <int LPG> static inline float lanes_allsum(float x, int) { return x; }
}
"""

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "row_access.h"
namespace adcdiff {
namespace {
%s
template <typename T, RowShape SHAPE, int TPR, int V>
int uneven(int M, int K, unsigned groups) {
    const int Kp = (K + 15) / 16 * 16, threads = quantize_threads<TPR>();
    std::vector<T> x((size_t)M * K, (T)1.0f);
    std::vector<int8_t> q((size_t)M * Kp);
    std::vector<float> scale(M);
    int bad = 0;
    gridDim.x = groups;
    for (unsigned b = 0; b < groups; ++b) {
        long long first = -1;
        for (int t = 0; t < threads; ++t) {
            blockIdx.x = b;
            threadIdx.x = t;
            met = 0;
            quantize_rows_kernel<T, SHAPE, true, TPR, V>(x.data(), K, M, K, Kp, q.data(), Kp, scale.data());
            if (first < 0) first = met;
            bad += met != first;
        }
    }
    return bad;
}
}
}
int main() {
    using namespace adcdiff;
    for (int M : {1, 2, 3, 4, 5, 7, 8})
        for (unsigned groups : {1u, 2u, 4u}) {
            printf("%%d %%d %%d %%d %%d %%d\n", uneven<float, kWhole, 16, 1>(M, 128, groups), uneven<float, kMoved, 64, 1>(M, 509, groups),
                   uneven<float, kWhole, 128, 2>(M, 2048, groups), uneven<bf16_t, kMoved, 128, 2>(M, 1003, groups),
                   uneven<float, kWhole, 256, 2>(M, 4096, groups), uneven<float, kWhole, 512, 2>(M, 8192, groups));
        }
}
"""


@pytest.mark.skipif(not os.path.exists(CLANG), reason="clang++ not available")
def test_row_quantiser(tmp_path):
    source = open(os.path.join(CSRC, "gemm_i8.hip")).read()
    kernel = source[source.index("struct RowScale"):source.index("// rows of any length")]
    (tmp_path / "common.h").write_text(COMMON)
    shutil.copy(os.path.join(CSRC, "row_access.h"), tmp_path)
    (tmp_path / "count.cpp").write_text(PROGRAM % kernel)
    subprocess.run([CLANG, "-std=c++17", "-O1", "-w", str(tmp_path / "count.cpp"), "-o", str(tmp_path / "count")], check=True)
    lines = subprocess.run([str(tmp_path / "count")], check=True, capture_output=True, text=True).stdout.split("\n")[:-1]
    assert len(lines) == 21 and set(lines) == {"0 0 0 0 0 0"}, lines

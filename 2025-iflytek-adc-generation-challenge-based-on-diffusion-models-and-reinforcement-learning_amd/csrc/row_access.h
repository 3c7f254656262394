// Rows held in the registers of a team of threads: loads, stores and sums shared by the row kernels (norms, row quantiser).
#pragma once
#include <atomic>

#include "common.h"

namespace adcdiff {

constexpr int kThreads = 256;   // threads of a row kernel's workgroup: as many teams as fit, or one team where a row needs a wider one
template <int TPR>
constexpr int threads_for() { return TPR >= kThreads ? TPR : kThreads / TPR * TPR; }

template <typename T>
__device__ __forceinline__ float to_f(T v) { return (float)v; }

__device__ __forceinline__ float bf_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Columns of element e of thread t: vectors of 8 consecutive columns where VEC, else single columns TPR apart.
template <bool VEC, int TPR>
__device__ __forceinline__ int column(int t, int e) { return VEC ? ((e >> 3) * TPR + t) * 8 + (e & 7) : e * TPR + t; }

// E elements of the row at p; columns >= D read as 0.
template <typename T, bool VEC, int TPR, int E>
__device__ __forceinline__ void load_row(const T* __restrict__ p, int t, int D, float (&v)[E]) {
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < E / 8; ++j) {
            const int c = (j * TPR + t) * 8;
            if (c < D) {
                if constexpr (sizeof(T) == 2) {
                    const u32x4 w = *reinterpret_cast<const u32x4*>(p + c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) { v[j * 8 + 2 * i] = bf_lo(w[i]); v[j * 8 + 2 * i + 1] = bf_hi(w[i]); }
                } else {
                    const f32x4 a = *reinterpret_cast<const f32x4*>(p + c), b = *reinterpret_cast<const f32x4*>(p + c + 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i) { v[j * 8 + i] = a[i]; v[j * 8 + 4 + i] = b[i]; }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j * 8 + i] = 0.0f;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = e * TPR + t;
            v[e] = c < D ? to_f(p[c]) : 0.0f;
        }
    }
}

template <typename T, bool VEC, int TPR, int E>
__device__ __forceinline__ void store_row(T* __restrict__ p, int t, int D, const float (&v)[E]) {
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < E / 8; ++j) {
            const int c = (j * TPR + t) * 8;
            if (c < D) {
                if constexpr (sizeof(T) == 2) {
                    bf16x8 o;
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = (bf16_t)v[j * 8 + i];
                    *reinterpret_cast<bf16x8*>(p + c) = o;
                } else {
                    f32x4 a, b;
#pragma unroll
                    for (int i = 0; i < 4; ++i) { a[i] = v[j * 8 + i]; b[i] = v[j * 8 + 4 + i]; }
                    *reinterpret_cast<f32x4*>(p + c) = a;
                    *reinterpret_cast<f32x4*>(p + c + 4) = b;
                }
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = e * TPR + t;
            if (c < D) p[c] = (T)v[e];
        }
    }
}

// Eight elements of a row as they stand in memory: loaded without being looked at, so that the loads of a row ahead stay in flight under the
// arithmetic of the row in hand.  Columns as in load_row with E = 8; those >= D read as 0.
template <typename T, bool VEC, int TPR>
struct RawRow {
    static constexpr int N = VEC && sizeof(T) == 2 ? 4 : 8;
    uint32_t r[N];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = 0;
    }
    __device__ __forceinline__ void load(const T* __restrict__ p, int t, int D) {
        if constexpr (VEC) {
            clear();
            if (t * 8 < D) {
#pragma unroll
                for (int i = 0; i < N / 4; ++i) {
                    const u32x4 w = *reinterpret_cast<const u32x4*>(p + t * 8 + 4 * i);
#pragma unroll
                    for (int k = 0; k < 4; ++k) r[4 * i + k] = w[k];
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = e * TPR + t;
                if constexpr (sizeof(T) == 2) r[e] = c < D ? reinterpret_cast<const uint16_t*>(p)[c] : 0;
                else r[e] = c < D ? reinterpret_cast<const uint32_t*>(p)[c] : 0;
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_bit_cast(float, r[e]);
        } else if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = bf_lo(r[i]); v[2 * i + 1] = bf_hi(r[i]); }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = bf_lo(r[e]);
        }
    }
};

// Sums over a team of TPR threads; every thread receives them.  Teams wider than a wave exchange through `red`, whose two halves
// alternate, so one barrier per call is enough (a half is written again only behind the barrier of the call in between).
template <int TPR, int N>
struct TeamSum {
    float* red;
    int half;
    __device__ __forceinline__ explicit TeamSum(float* r) : red(r), half(0) {}
    __device__ __forceinline__ void operator()(float (&s)[N], int tid) {
#pragma unroll
        for (int n = 0; n < N; ++n) s[n] = lanes_allsum<(TPR < 64 ? TPR : 64)>(s[n], 0);
        if constexpr (TPR > 64) {
            constexpr int WAVES = TPR / 64, SLOTS = threads_for<TPR>() / 64;
            float* buf = red + half * SLOTS * N;
            const int wave = tid >> 6;
            if ((tid & 63) == 0) {
#pragma unroll
                for (int n = 0; n < N; ++n) buf[wave * N + n] = s[n];
            }
            __syncthreads();
            const int first = wave / WAVES * WAVES;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                float a = 0.0f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) a += buf[(first + w) * N + n];
                s[n] = a;
            }
            half ^= 1;
        }
    }
};

inline bool type_ok(int dtype) { return dtype == ADCDIFF_F32 || dtype == ADCDIFF_BF16; }
inline int type_size(int dtype) { return dtype == ADCDIFF_BF16 ? 2 : 4; }

// rows on 16-byte boundaries (vector accesses), or absent
inline bool vector_rows(const void* p, long long ld, int size) { return !p || (aligned16(p) && (ld * size & 15) == 0); }

// Lets a kernel use `bytes` of dynamic LDS on the current device; done[device] remembers that it was said
inline int allow_lds(const char* who, const void* kernel, int bytes, std::atomic<bool> (&done)[64]) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess || dev < 0 || dev >= 64) return fail(ADCDIFF_E_LAUNCH, "%s: hipGetDevice: %s (device %d)", who, hipGetErrorString(e), dev);
    if (done[dev].load(std::memory_order_relaxed)) return ADCDIFF_OK;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return fail(ADCDIFF_E_LAUNCH, "%s: hipFuncSetAttribute: %s", who, hipGetErrorString(e));
    done[dev].store(true, std::memory_order_relaxed);
    return ADCDIFF_OK;
}

}  // namespace adcdiff

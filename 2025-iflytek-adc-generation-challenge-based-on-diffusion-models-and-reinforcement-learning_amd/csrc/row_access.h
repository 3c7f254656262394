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

// Thread t of a team owns the eight columns from 8 t on.  Rows start at any element: the memory system takes 16-byte accesses at any address.
//   kWhole: D is a multiple of 8
//   kMoved: it is not, and the last thread with columns moves its eight back to the row's last ones.  It loads and stores what its neighbour does,
//           with the same bits, and own_columns leaves them to the neighbour in sums.  (65536 x 777 bfloat16: forward 98 us, backward 169; all in single elements 129 and 206;
//           vectors with a single-element tail 115 and 237: the tail's branch makes the loads of a row ahead wait.)  Where a row is overwritten in place, neighbours in two waves have to
//           have loaded it before either stores (wave_crossing).
//   kTiny:  D < 8, the first thread has the row in single elements
enum RowShape { kWhole, kMoved, kTiny };
inline RowShape row_shape(int D) { return D % 8 == 0 ? kWhole : D > 8 ? kMoved : kTiny; }
inline bool wave_crossing(int D) { return D > 512 && D % 512 > 0 && D % 512 < 8; }   // the last thread is a wave's first

typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef bf16x8 bf16x8_any __attribute__((aligned(2)));

// first of the eight columns of thread t (8 t < D)
template <RowShape SHAPE>
__device__ __forceinline__ int first_column(int t, int D) { return SHAPE == kMoved ? min(t * 8, D - 8) : t * 8; }

// bit e: element e is this thread's in a sum over the row
template <RowShape SHAPE>
__device__ __forceinline__ unsigned own_columns(int t, int D) {
    const int rest = D - t * 8;
    if (rest <= 0) return 0u;
    if (SHAPE == kWhole || rest >= 8) return 0xffu;
    return SHAPE == kMoved ? 0xffu >> (8 - rest) << (8 - rest) : 0xffu >> (8 - rest);
}

// the eight elements of thread t of the row at p
template <typename T, RowShape SHAPE>
__device__ __forceinline__ void store_row(T* __restrict__ p, int t, int D, const float (&v)[8]) {
    if (t * 8 >= D) return;
    if constexpr (SHAPE == kTiny) {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < D) p[e] = (T)v[e];
    } else {
        T* const q = p + first_column<SHAPE>(t, D);
        if constexpr (sizeof(T) == 2) {
            bf16x8 o;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = (bf16_t)v[i];
            *reinterpret_cast<bf16x8_any*>(q) = o;
        } else {
            *reinterpret_cast<f32x4_any*>(q) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4_any*>(q + 4) = f32x4{v[4], v[5], v[6], v[7]};
        }
    }
}

// The eight elements of thread t as they stand in memory: loaded without being looked at, so that the loads of a row ahead stay in flight under
// the arithmetic of the row in hand.  Elements without a column read as 0.
template <typename T, RowShape SHAPE>
struct RawRow {
    static constexpr int N = sizeof(T) == 2 ? 4 : 8;
    uint32_t r[N];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = 0;
    }
    __device__ __forceinline__ void load(const T* __restrict__ p, int t, int D) {
        clear();
        if (t * 8 >= D) return;
        if constexpr (SHAPE == kTiny) {
#pragma unroll
            for (int e = 0; e < 7; ++e) {
                if (e < D) {
                    if constexpr (sizeof(T) == 2) r[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e & 1));
                    else r[e] = reinterpret_cast<const uint32_t*>(p)[e];
                }
            }
        } else {
            const T* const q = p + first_column<SHAPE>(t, D);
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                const u32x4 w = *reinterpret_cast<const u32x4_any*>(q + 4 * i);
#pragma unroll
                for (int k = 0; k < 4; ++k) r[4 * i + k] = w[k];
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_bit_cast(float, r[e]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = bf_lo(r[i]); v[2 * i + 1] = bf_hi(r[i]); }
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

// The 8-bit integer layer: codes of rows with a scale each (activations by row, weights by channel), and their product
//   out[m, n] = act(a_scale[m] * w_scale[n] * sum_k a[m, k] w[n, k] + bias[n] + residual[m, n]).
// The sum runs on v_mfma_i32_16x16x64_i8 and is exact; what follows is float32 and rounded once.
#include <algorithm>
#include <atomic>

#include "row_access.h"

namespace adcdiff {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_byte __attribute__((aligned(1)));   // global memory takes 16-byte loads at any address

// ------------------------------------------------------------------ codes of rows
// A code is rne(x * 127 / top), exactly.
// bfloat16 rows: x * 127 is exact in float32, and one correction of the product with 1 / top gives the correctly rounded quotient; a half
// is then a half, and no other quotient of two 8-bit significands comes closer to one than 2^-10.  No branch: a value of top / 2, which is
// such a half, stands in every second group of 512 codes.
// float32 rows: t = x * (127 / top) is off by at most 127 * 2^-23 < 1.6e-5, so its rounding can only differ where t lies within that of a
// half; there the quotient is formed in float64, where x * 127 is exact and the division's error is far below the distance of any
// quotient of two float32 numbers from a half (>= 2^-26).  One test for N codes: a wave meets such a value in one group of thirty.
// Rows whose maximum nears overflow or the subnormals (times 127, or 127 / top) take the float64 form throughout.
struct RowScale {
    float top, inv, scale;
    bool none, far;                        // none: a row of zeros, or one with a NaN or an infinity: codes 0
    __device__ __forceinline__ explicit RowScale(uint32_t top_bits) {
        top = __builtin_bit_cast(float, top_bits);
        const bool poison = top_bits >= 0x7f800000u;   // infinity or NaN (NaN's bits are the larger)
        none = poison || top_bits == 0u;
        far = top < 1e-30f || top > 1e36f;
        inv = 127.0f / top;
        scale = poison ? __builtin_nanf("") : top / 127.0f;
    }
    template <bool BF16, int N>
    __device__ __forceinline__ void codes(const float (&x)[N], int (&q)[N]) const {
        bool exact = far;
        const float rtop = BF16 ? 1.0f / top : 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if constexpr (BF16) {
                const float p = x[e] * 127.0f, t = p * rtop;
                q[e] = (int)rintf(fmaf(fmaf(-t, top, p), rtop, t));
            } else {
                const float t = x[e] * inv, r = rintf(t);
                exact |= fabsf(fabsf(t - r) - 0.5f) < 3.1e-5f;
                q[e] = (int)r;
            }
        }
        if (exact) {
            asm volatile("");   // a branch to stay: computed in any case and selected, 65536 x 512 takes 38 us instead of 19
#pragma unroll
            for (int e = 0; e < N; ++e) q[e] = (int)rint((double)x[e] * 127.0 / (double)top);
        }
        if (none) {
#pragma unroll
            for (int e = 0; e < N; ++e) q[e] = 0;
        }
    }
    __device__ __forceinline__ int code(float x) const {   // of either type (rows of more than 8192)
        const float v[1] = {x};
        int q[1];
        codes<false>(v, q);
        return q[0];
    }
};

template <int TPR>
__device__ __forceinline__ uint32_t team_max(uint32_t v, uint32_t* red, int tid) {
#pragma unroll
    for (int m = (TPR < 64 ? TPR : 64) / 2; m > 0; m >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, m));
    if constexpr (TPR > 64) {
        if ((tid & 63) == 0) red[tid >> 6] = v;
        __syncthreads();
        const int first = (tid >> 6) / (TPR / 64) * (TPR / 64);
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) v = max(v, red[first + w]);
        __syncthreads();   // the next row writes red again
    }
    return v;
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// One row per team, held in registers between the maximum and the codes; bound by HBM (65536 x 2048 bfloat16 74 us, 403 MB at 5.4 TB/s; 4096 x 2048
// 7.2 us) and by latency below.  PAIRS: rows of q start on 8-byte boundaries and eight codes are one store, those behind K among them.
template <int TPR>
constexpr int quantize_threads() { return TPR > 64 ? TPR : threads_for<TPR>(); }

template <typename T, RowShape SHAPE, bool PAIRS, int TPR, int V>
__global__ __launch_bounds__(quantize_threads<TPR>()) void quantize_rows_kernel(const T* __restrict__ x, long long ldx, int M, int K, int Kp, int8_t* __restrict__ q,
                                                                           long long ldq, float* __restrict__ scale) {
    constexpr int THREADS = quantize_threads<TPR>(), TEAMS = THREADS / TPR;
    __shared__ uint32_t red[THREADS / 64];
    const int tid = threadIdx.x, t = tid % TPR;
    // a team wider than a wave is alone in its workgroup, so the barriers of the maximum are met by every thread
    for (long long row = (long long)blockIdx.x * TEAMS + tid / TPR; row < M; row += (long long)gridDim.x * TEAMS) {
        float v[V][8];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            RawRow<T, SHAPE> raw;
            raw.load(x + row * ldx, j * TPR + t, K);
            raw.get(v[j]);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, abs_bits(v[j][e]));
        }
        const RowScale s(team_max<TPR>(top, red, tid));
        int8_t* out = q + row * ldq;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * TPR + t) * 8;
            if (c < Kp) {
                int code[8];
                s.template codes<sizeof(T) == 2>(v[j], code);
                uint64_t w = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) w |= (uint64_t)((uint32_t)code[i] & 0xffu) << (8 * i);
                if constexpr (SHAPE == kMoved) {   // the last thread's own columns are the last of its eight
                    if (c < K && c + 8 > K) w >>= 8 * (c + 8 - K);
                }
                if constexpr (PAIRS) {
                    *reinterpret_cast<uint64_t*>(out + c) = w;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (c + i < Kp) out[c + i] = (int8_t)(w >> (8 * i));
                }
            }
        }
        if (t == 0) scale[row] = s.scale;
    }
}

// rows of any length: the row is read twice, the second time out of the cache
template <typename T>
__global__ __launch_bounds__(1024) void quantize_long_rows_kernel(const T* __restrict__ x, long long ldx, int M, int K, int Kp, int8_t* __restrict__ q, long long ldq,
                                                                  float* __restrict__ scale) {
    __shared__ uint32_t red[16];
    for (long long row = blockIdx.x; row < M; row += gridDim.x) {
        const T* in = x + row * ldx;
        uint32_t top = 0;
        for (int c = threadIdx.x; c < K; c += 1024) top = max(top, abs_bits(to_f(in[c])));
        const RowScale s(team_max<1024>(top, red, threadIdx.x));
        int8_t* out = q + row * ldq;
        for (int c = threadIdx.x; c < Kp; c += 1024) out[c] = c < K ? (int8_t)s.code(to_f(in[c])) : (int8_t)0;
        if (threadIdx.x == 0) scale[row] = s.scale;
    }
}

struct QuantizeArgs {
    const void* x;
    long long ldx;
    int M, K, Kp;
    int8_t* q;
    long long ldq;
    float* scale;
};

template <typename T, RowShape SHAPE, bool PAIRS, int TPR, int V>
void launch_quantize(const QuantizeArgs& a, hipStream_t stream) {
    constexpr int threads = quantize_threads<TPR>(), teams = threads / TPR;
    hipLaunchKernelGGL((quantize_rows_kernel<T, SHAPE, PAIRS, TPR, V>), dim3((unsigned)std::min(((long long)a.M + teams - 1) / teams, 1LL << 20)), dim3(threads), 0, stream,
                       static_cast<const T*>(a.x), a.ldx, a.M, a.K, a.Kp, a.q, a.ldq, a.scale);
}

template <typename T, RowShape SHAPE, bool PAIRS>
void quantize_by_width(const QuantizeArgs& a, hipStream_t stream) {
    if (a.Kp <= 128) return launch_quantize<T, SHAPE, PAIRS, 16, 1>(a, stream);
    if constexpr (SHAPE != kTiny) {
        if (a.Kp <= 512) return launch_quantize<T, SHAPE, PAIRS, 64, 1>(a, stream);
        // few rows: the latency of one row counts (32 x 2048: 256 threads 2.5 us, 128 threads 2.8); many: the barriers of wide teams (65536 x 2048: 87, 75 us)
        if (a.Kp <= 2048 && a.M < 2048) return launch_quantize<T, SHAPE, PAIRS, 256, 1>(a, stream);
        if (a.Kp <= 2048) return launch_quantize<T, SHAPE, PAIRS, 128, 2>(a, stream);
        if (a.Kp <= 4096) return launch_quantize<T, SHAPE, PAIRS, 256, 2>(a, stream);
        if (a.Kp <= 8192) return launch_quantize<T, SHAPE, PAIRS, 512, 2>(a, stream);
        hipLaunchKernelGGL((quantize_long_rows_kernel<T>), dim3(std::min(a.M, 1 << 20)), dim3(1024), 0, stream, static_cast<const T*>(a.x), a.ldx, a.M, a.K, a.Kp, a.q,
                           a.ldq, a.scale);
    }
}

template <typename T, bool PAIRS>
void quantize_by_shape(const QuantizeArgs& a, hipStream_t stream) {
    switch (row_shape(a.K)) {
        case kWhole: return quantize_by_width<T, kWhole, PAIRS>(a, stream);
        case kMoved: return quantize_by_width<T, kMoved, PAIRS>(a, stream);
        case kTiny: return quantize_by_width<T, kTiny, PAIRS>(a, stream);
    }
}

struct PitchParams {
    adcdiff_i8_copy c[2];
    unsigned first;   // the second copy's first workgroup
};

__global__ __launch_bounds__(256) void pitch_rows_kernel(const PitchParams p) {
    // sixteen columns per thread: byte loads at any alignment, one 16-byte store
    const bool second = blockIdx.x >= p.first;
    const adcdiff_i8_copy& c = p.c[second];
    const long long per_row = c.ld_dst / 16;
    const long long i = (long long)(blockIdx.x - (second ? p.first : 0u)) * 256 + threadIdx.x;
    if (i >= per_row * c.M) return;
    const long long row = i / per_row, col = (i - row * per_row) * 16;
    const int8_t* s = c.src + row * c.ld_src + col;
    const int n = (int)min(16LL, max(0LL, (long long)c.K - col));
    u32x4 w = {0, 0, 0, 0};
    if (n == 16) {
        w = *reinterpret_cast<const u32x4_byte*>(s);
    } else {
#pragma unroll
        for (int b = 0; b < 15; ++b)
            if (b < n) w[b >> 2] |= (uint32_t)(uint8_t)s[b] << (8 * (b & 3));
    }
    *reinterpret_cast<u32x4*>(c.dst + row * c.ld_dst + col) = w;
}

// ------------------------------------------------------------------ product
struct I8Params {
    const int8_t *a, *w;
    const float *a_scale, *w_scale, *bias;
    const void* residual;
    void* out;
    long long lda, ldw, ldr, ldo;
    int M, N, K, act;
};

// v * sigmoid(v) on the hardware's exp2 and reciprocal (each within one unit in the last place): the argument's rounding adds |v| * 2^-24 relative,
// which the sigmoid's own slope keeps below 2^-23 of |v|; the exact division costs four times the instructions.
__device__ __forceinline__ float silu_fast(float v) {
    return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896f));
}

// The sum times both scales, |sum| < 2^31.  The row's scale first stays finite below 2^96, and a sum is at least 1, so nothing is lost below either (a
// subnormal scale times a whole number is exact until it is normal).  From 2^96 on the output's scale comes first: where that overflows, so does the value.
__device__ __forceinline__ bool far_scale(float sa) { return fabsf(sa) >= 0x1p96f; }

// 16 bytes of a row from column k on, with the bytes at columns >= K cleared.  Rows start on 16-byte boundaries, so a chunk that holds a
// valid byte never leaves the page of that byte: the bytes behind K may be read, and count for nothing.
__device__ __forceinline__ i32x4 load_chunk(const int8_t* __restrict__ row, int k, int K) {
    if (k >= K) return i32x4{0, 0, 0, 0};
    i32x4 v = *reinterpret_cast<const i32x4*>(row + k);
    const int keep = K - k;
    if (keep < 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = keep - 4 * i;
            v[i] = b >= 4 ? v[i] : b <= 0 ? 0 : v[i] & (int)((1u << (8 * b)) - 1u);
        }
    }
    return v;
}

// Eight consecutive outputs of row m from column n on (single elements where the row ends before): their scales, biases and residual (which the
// few-row kernel loads before the sums are there), and the outputs.  Rows may start at any element.
template <typename Out>
struct Finish8 {
    typedef Out Eight __attribute__((ext_vector_type(8)));
    typedef Eight EightAny __attribute__((aligned(sizeof(Out))));
    f32x4 w0, w1, b0, b1;
    float sa;
    Eight r;
    __device__ __forceinline__ void load(const I8Params& p, int m, int n) {
        const Out* res = static_cast<const Out*>(p.residual) + (long long)m * p.ldr + n;
        sa = p.a_scale[m];
        b0 = b1 = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (n + 8 <= p.N) {
            const f32x4_any* pw = reinterpret_cast<const f32x4_any*>(p.w_scale + n);
            w0 = pw[0];
            w1 = pw[1];
            if (p.bias) {
                const f32x4_any* pb = reinterpret_cast<const f32x4_any*>(p.bias + n);
                b0 = pb[0];
                b1 = pb[1];
            }
            if (p.residual) r = *reinterpret_cast<const EightAny*>(res);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const bool in = n + c < p.N, in4 = n + 4 + c < p.N;
                w0[c] = in ? p.w_scale[n + c] : 0.0f;
                w1[c] = in4 ? p.w_scale[n + 4 + c] : 0.0f;
                b0[c] = in && p.bias ? p.bias[n + c] : 0.0f;
                b1[c] = in4 && p.bias ? p.bias[n + 4 + c] : 0.0f;
            }
            if (p.residual) {
#pragma unroll
                for (int c = 0; c < 8; ++c) r[c] = n + c < p.N ? res[c] : (Out)0.0f;
            }
        }
    }
    __device__ __forceinline__ void store(const I8Params& p, int m, int n, const i32x4& lo, const i32x4& hi) const {
        Out* out = static_cast<Out*>(p.out) + (long long)m * p.ldo + n;
        float v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = c < 4 ? fmaf((float)lo[c & 3] * sa, w0[c & 3], b0[c & 3]) : fmaf((float)hi[c & 3] * sa, w1[c & 3], b1[c & 3]);
        const bool far = far_scale(sa);
        if (__builtin_expect(__any(far), 0)) {
            if (far) {
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = c < 4 ? fmaf((float)lo[c & 3] * w0[c & 3], sa, b0[c & 3]) : fmaf((float)hi[c & 3] * w1[c & 3], sa, b1[c & 3]);
            }
        }
        Eight o;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            if (p.residual) v[c] += (float)r[c];
            if (p.act) v[c] = silu_fast(v[c]);
            o[c] = (Out)v[c];
        }
        if (n + 8 <= p.N) {
            *reinterpret_cast<EightAny*>(out) = o;
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (n + c < p.N) out[c] = o[c];
        }
    }
};

// ---- BM x BN tile through a ring of LDS stages ------------------------------------------------------------------------------------
// Eight waves (2 x 4); a stage is 128 columns of the tile's rows, filled by LDS-DMA (64 lanes x 16 bytes = eight rows of 128 bytes per
// instruction).  The chunk c of a row lies at position c ^ ((row >> 1) & 7), applied to the source address, so fragment reads are free of bank
// conflicts.  STAGES - 1 tiles are under way; a stage is refilled behind the barrier that follows the last wait for its reads.  The weights are
// the MFMA's first operand: a lane's four results are consecutive outputs of a row.
// Bound by the waits between its steps, not by one unit (4096 x 2048 x 2048, counters): the matrix cores are busy in 43 % of the CUs' cycles and LDS reads
// take 36 %, while the waves spend 41 % of their time behind a wait or barrier and 34 % ready for an issue slot that another wave has.  A K tile of
// 128 x 128 takes 0.7 us whether one workgroup runs or all do, with the rows' lines in L2 or not (a prefetch into L2 and an order of tiles that shares
// more rows there changed nothing).  So two or three workgroups share a CU (two stages of 32 KiB, three of 16 KiB): each covers the others' barriers and
// epilogues (4096 x 2048 x 2048: 26 us, four stages and one workgroup 32 us, 256 x 128 tiles 27 us).
template <typename Out, int BM, int BN, int STAGES>
__global__ __launch_bounds__(512) void gemm_i8_ring_kernel(const I8Params p) {
    constexpr int TM = BM / 32, TN = BN / 64, PIECES = (BM + BN) / 64, STAGE = (BM + BN) * 128, PITCH = BN + 4;
    static_assert(PIECES * 64 == BM + BN && TN >= 1, "a wave loads PIECES pieces of eight rows");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    // consecutive tiles on one XCD (workgroup b runs on XCD b mod 8): they share rows in its L2
    const int ntn = (p.N + BN - 1) / BN, xcd = blockIdx.x & 7;
    const int bid = xcd * (gridDim.x >> 3) + min(xcd, (int)(gridDim.x & 7)) + (blockIdx.x >> 3);
    const int m0 = bid / ntn * BM, n0 = bid % ntn * BN;
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;
    const int8_t* src[PIECES];
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {   // rows past the edge repeat the last one; what they give is not stored
        const int r = (wave * PIECES + j) * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        src[j] = (r < BM ? p.a + (long long)min(m0 + r, p.M - 1) * p.lda : p.w + (long long)min(n0 + r - BM, p.N - 1) * p.ldw) + 16 * c;
    }
    const unsigned dst = lds0 + (unsigned)(wave * PIECES) * 1024u;
    auto issue = [&](int t, int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) glds16_untracked(src[j] + (long long)t * 128, dst + (unsigned)stage * STAGE + 1024u * j);
    };
    i32x4 acc[TM][TN] = {};
    auto multiply = [&](const char* st) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i32x4 fa[TM], fw[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int r = BM + (wn * TN + j) * 16 + (lane & 15);
                fw[j] = *reinterpret_cast<const i32x4*>(st + r * 128 + (((4 * h + (lane >> 4)) ^ ((r >> 1) & 7)) << 4));
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int r = (wm * TM + i) * 16 + (lane & 15);
                fa[i] = *reinterpret_cast<const i32x4*>(st + r * 128 + (((4 * h + (lane >> 4)) ^ ((r >> 1) & 7)) << 4));
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[j], fa[i], acc[i][j], 0, 0, 0);
        }
    };
    const int kt = p.K >> 7;
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t)
        if (t < kt) issue(t, t);
    int stage = 0;
    for (int t = 0; t < kt; ++t) {
        // tiles t + 1 .. t + STAGES - 2 may stay in flight; then every wave's pieces of tile t are there, and stage t - 1 has been read
        wait_tiles_in_flight<PIECES>(min(STAGES - 2, kt - 1 - t));
        asm volatile("s_barrier" ::: "memory");
        if (t + STAGES - 1 < kt) issue(t + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
        multiply(smem + stage * STAGE);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // this wave's reads are done before it meets the next barrier
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    if (p.K & 127) {   // the columns behind the whole tiles, through registers, cleared behind K
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const int r = (wave * PIECES + j) * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
            *reinterpret_cast<i32x4*>(smem + (wave * PIECES + j) * 1024 + lane * 16) = load_chunk(src[j] - 16 * c, kt * 128 + 16 * c, p.K);
        }
        __syncthreads();
        multiply(smem);
    }
    __syncthreads();
    int* const sums = reinterpret_cast<int*>(smem);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
            *reinterpret_cast<i32x4*>(sums + ((wm * TM + i) * 16 + (lane & 15)) * PITCH + (wn * TN + j) * 16 + 4 * (lane >> 4)) = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int e = tid; e < BM * BN / 8; e += 512) {
        const int r = e / (BN / 8), c = e % (BN / 8) * 8;
        if (m0 + r >= p.M || n0 + c >= p.N) continue;
        Finish8<Out> finish;
        finish.load(p, m0 + r, n0 + c);
        finish.store(p, m0 + r, n0 + c, *reinterpret_cast<const i32x4*>(sums + r * PITCH + c), *reinterpret_cast<const i32x4*>(sums + r * PITCH + c + 4));
    }
}

// ---- few rows: the waves of a workgroup share its BM x BN tile and split K ---------------------------------------------------
// A unit is 128 columns (a cache line of a row, two MFMA steps).  Wave w takes units w, w + WAVES, ..; its fragments go from memory to
// registers (no LDS stage, no barrier), DEPTH units in flight.  The partial sums meet in LDS; integer sums do not depend on their
// order.  Bound by the latency of one or two rounds of loads; the tile is kept small so that enough workgroups share the weights' bytes.
// 1 x 2048 x 2048 in 4.1 us (the weights' 4 MB at 1.0 TB/s), 32 x 2048 x 4096 in 6.8 us.
template <typename Out, int BM, int BN, int WAVES, int DEPTH>
__global__ __launch_bounds__(64 * WAVES) void gemm_i8_split_kernel(const I8Params p) {
    constexpr int TM = BM / 16, TN = BN / 16, PITCH = BN + 4;
    __shared__ __attribute__((aligned(16))) int part[WAVES][BM * PITCH];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ntn = (p.N + BN - 1) / BN;
    const int m0 = blockIdx.x / ntn * BM, n0 = blockIdx.x % ntn * BN;
    const int8_t *ra[TM], *rw[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) ra[i] = p.a + (long long)min(m0 + 16 * i + (lane & 15), p.M - 1) * p.lda;
#pragma unroll
    for (int j = 0; j < TN; ++j) rw[j] = p.w + (long long)min(n0 + 16 * j + (lane & 15), p.N - 1) * p.ldw;
    const int kl = (lane >> 4) * 16;
    const int units = (p.K + 127) / 128;
    const bool ragged = (p.K & 15) != 0;
    i32x4 acc[TM][TN] = {};
    i32x4 fa[DEPTH][2][TM], fw[DEPTH][2][TN];
    // Only the weights are cleared behind K; the rows' codes there meet zeros.
    auto load = [&](int d, int u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = u * 128 + h * 64 + kl;
            const bool in = k < p.K;
            const int ka = in ? k : 0;
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                fw[d][h][j] = *reinterpret_cast<const i32x4*>(rw[j] + ka);
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) fa[d][h][i] = *reinterpret_cast<const i32x4*>(ra[i] + ka);
        }
    };
    auto multiply = [&](int d, int u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (u + 1 == units) {   // the last unit: clear what lies behind K
                const int keep = p.K - (u * 128 + h * 64 + kl);
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int b = keep - 4 * i;
                        fw[d][h][j][i] = b >= 4 ? fw[d][h][j][i] : b <= 0 || !ragged ? 0 : fw[d][h][j][i] & (int)((1u << (8 * (b & 3))) - 1u);
                    }
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[d][h][j], fa[d][h][i], acc[i][j], 0, 0, 0);
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (wave + d * WAVES < units) load(d, wave + d * WAVES);
    // the outputs of this thread, eight of a row, and what they need beside the sums: on its way together with the codes
    // (1 x 2048 x 2048: 4.30 -> 4.09 us, 64 x 2048 x 2048: 6.02 -> 5.57 us)
    static_assert(BM * BN / 8 <= 64 * WAVES, "one round of outputs");
    const int er = tid / (BN / 8), ec = tid % (BN / 8) * 8;
    const bool mine = er < BM && m0 + er < p.M && n0 + ec < p.N;
    Finish8<Out> finish;
    if (mine) finish.load(p, m0 + er, n0 + ec);
    for (int u = wave; u < units; u += DEPTH * WAVES) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int v = u + d * WAVES;
            if (v < units) {
                multiply(d, v);
                if (v + DEPTH * WAVES < units) load(d, v + DEPTH * WAVES);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
            *reinterpret_cast<i32x4*>(&part[wave][(16 * i + (lane & 15)) * PITCH + 16 * j + 4 * (lane >> 4)]) = acc[i][j];
    __syncthreads();
    if (mine) {
        i32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            lo += *reinterpret_cast<const i32x4*>(&part[w][er * PITCH + ec]);
            hi += *reinterpret_cast<const i32x4*>(&part[w][er * PITCH + ec + 4]);
        }
        finish.store(p, m0 + er, n0 + ec, lo, hi);
    }
}

// ---- many rows: 256 x 256 tile, 4 waves (2 x 2, 128 x 128 each), one wave per SIMD --------------------------------------------
// The main loop is the hand-allocated assembly of the bf16 product (gen_w4_mainloop.py, which documents registers, LDS image and
// protocol) with the 8-bit MFMA: a K tile is the same 128 bytes of a row, now 128 codes.  It runs over the whole K tiles; columns
// behind them are added by a short tail on fragments loaded straight from memory.  A tile at the lower or right edge is moved back inside
// the matrix (every load in range) and stores only the rows and columns that no other tile stores.
// 65536 x 2048 x 2048 to bfloat16: 266 us (2.07 POP/s, what the library's int8 product reaches), 302 us with a residual, whose 268 MB stand
// against the epilogue's stores.
#include "w4_mainloop_i8.inc"

// SIDE: bit 0 residual, bit 1 SiLU, known at compile time so that loads and stores are counted exactly and no wait covers the stores.
// WHOLE: N is a multiple of 8; else eight outputs at the edge of a tile that moved back may belong to two tiles and are stored one by one.
template <typename Out, int SIDE, bool WHOLE>
__global__ __launch_bounds__(256, 1) void gemm_i8_w4_kernel(const I8Params p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;
    // consecutive tiles (the columns of one tile row first) run on one XCD, whose L2 they share; workgroup b runs on XCD b mod 8
    const int nwg = gridDim.x, ntn = (p.N + 255) >> 8;
    const int xcd = blockIdx.x & 7, share_of = nwg >> 3, more = nwg & 7;
    const int bid = xcd * share_of + min(xcd, more) + (blockIdx.x >> 3);
    const int nidx = bid % ntn;
    const int m_lo = bid / ntn * 256, n_lo = nidx * 256;
    const int m0 = min(m_lo, p.M - 256), n0 = min(n_lo, p.N - 256);
    const int kt = p.K >> 7;

    const bool loads_a = wave < 2;
    const int half = wave & 1;
    const unsigned ld = (unsigned)(loads_a ? p.lda : p.ldw);
    const unsigned long long base = loads_a ? (unsigned long long)p.a + (unsigned long long)(m0 + half * 128) * p.lda
                                            : (unsigned long long)p.w + (unsigned long long)(n0 + half * 128) * p.ldw;
    const int seg_lo = __builtin_amdgcn_readfirstlane((int)(unsigned)base);
    const int seg_hi = __builtin_amdgcn_readfirstlane((int)((unsigned)(base >> 32) & 0xffffu));
    const int seg_ld = __builtin_amdgcn_readfirstlane((int)ld);
    const int seg_kt = __builtin_amdgcn_readfirstlane(kt);
    const int seg_nrec = __builtin_amdgcn_readfirstlane((int)(127u * ld + (unsigned)kt * 128u));
    const int zero = __builtin_amdgcn_readfirstlane(0);
    const int s_dst = __builtin_amdgcn_readfirstlane((int)(lds0 + (loads_a ? 0u : 32768u) + (unsigned)half * 16384u));
    const int frow = lane & 15, fchunk = lane >> 4, fx = (frow >> 1) & 7;
    const int v_aoff0 = (int)lds0 + (wm * 128 + frow) * 128 + ((fchunk ^ fx) << 4);
    const int v_aoff1 = (int)lds0 + (wm * 128 + frow) * 128 + (((4 + fchunk) ^ fx) << 4);
    const int v_boff0 = (int)lds0 + 32768 + (wn * 128 + frow) * 128 + ((fchunk ^ fx) << 4);
    const int v_boff1 = (int)lds0 + 32768 + (wn * 128 + frow) * 128 + (((4 + fchunk) ^ fx) << 4);
    const int v_src0 = (int)((unsigned)(lane >> 3) * ld + (unsigned)(((lane & 7) ^ (lane >> 4)) * 16));
    const int v_src1 = (int)((unsigned)(lane >> 3) * ld + (unsigned)(((lane & 7) ^ (4 + (lane >> 4))) * 16));
    // L2 prefetch: the workgroups of a tile row share its A rows and split the touching of them (a share of at most 64 rows each)
    const int share = ntn >= 4 ? max(1, 256 / ntn) : 64;
    const int prow0 = ntn >= 4 ? min(nidx * share, 256 - share) : half * 128 + (ntn == 2 ? nidx * 64 : 0);
    const bool pf_wave = loads_a && (prow0 >> 7) == half;
    const int pf_row = min((prow0 & 127) + lane % share, 127);
    const int v_pf = pf_wave ? (int)((unsigned)pf_row * ld + (unsigned)(lane / share) * 128u) : 0;

    i32x4 acc[8][8];
    asm volatile(ADCDIFF_W4I8_MAINLOOP_ASM
                 : ADCDIFF_W4_OUTS(acc)
                 : "{s40}"(seg_lo), "{s41}"(seg_hi), "{s42}"(seg_ld), "{s43}"(seg_kt), "{s44}"(seg_nrec), "{s45}"(zero), "{s46}"(zero), "{s47}"(zero),
                   "{s48}"(zero), "{s49}"(zero), "{s50}"(zero), "{s51}"(zero), "{s52}"(zero), "{s53}"(zero), "{s54}"(zero), "{s55}"(seg_kt), "{s56}"(s_dst),
                   "{v130}"(v_aoff0), "{v131}"(v_boff0), "{v132}"(v_aoff1), "{v133}"(v_boff1), "{v136}"(v_src0), "{v137}"(v_src1), "{v138}"(v_src0),
                   "{v139}"(v_src1), "{v140}"(v_src0), "{v141}"(v_src1), "{v144}"(v_pf), "{v145}"(v_pf), "{v146}"(v_pf)
                 : ADCDIFF_W4_CLOBBERS);
    const int mw = m0 + wm * 128, nw = n0 + wn * 128;
    for (int k0 = kt * 128; k0 < p.K; k0 += 64) {   // the columns behind the whole K tiles
        const int k = k0 + fchunk * 16;
        const int8_t* rw = p.w + (long long)(nw + frow) * p.ldw;
        const int8_t* ra = p.a + (long long)(mw + frow) * p.lda;
#pragma unroll
        for (int jh = 0; jh < 8; jh += 4) {
            i32x4 fw[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) fw[j] = load_chunk(rw + (long long)(16 * (jh + j)) * p.ldw, k, p.K);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const i32x4 fa = load_chunk(ra + (long long)(16 * i) * p.lda, k, p.K);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][jh + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[j], fa, acc[i][jh + j], 0, 0, 0);
            }
        }
    }
    // A lane holds outputs 4 g .. 4 g + 3 (g = lane / 16) of row lane % 16 in every 16 x 16 block.  Exchanging odd lane rows of block 2 j with even
    // ones of block 2 j + 1 leaves it eight consecutive outputs: columns 0..7 (g 0, 1) or 8..15 (g 2, 3) of block 2 j (g even) or 2 j + 1.
    const int nl = nw + 16 * (fchunk & 1) + 8 * (fchunk >> 1);
    // Scales, biases and the first rows' residual are loaded before the first store, and each further residual one step ahead of its use:
    // a load behind a store to memory that it might share waits a whole round trip (measured: 13 of 27 us outside the K loop).
    float w[4][8], b[4][8], sa[8];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            w[j][c] = p.w_scale[nl + 32 * j + c];
            b[j][c] = p.bias ? p.bias[nl + 32 * j + c] : 0.0f;
        }
#pragma unroll
    for (int i = 0; i < 8; ++i) sa[i] = p.a_scale[mw + 16 * i + frow];
    typedef Out Side __attribute__((ext_vector_type(8)));
    typedef Side SideAny __attribute__((aligned(sizeof(Out))));   // rows start at any element
    constexpr bool residual = (SIDE & 1) != 0, act = (SIDE & 2) != 0;
    const Out* const res = static_cast<const Out*>(p.residual) + (long long)(mw + frow) * p.ldr + nl;
    Side side[2][4];
    auto fetch = [&](int i) __attribute__((always_inline)) {
        if (residual) {
#pragma unroll
            for (int j = 0; j < 4; ++j) side[i & 1][j] = *reinterpret_cast<const SideAny*>(res + (long long)(16 * i) * p.ldr + 32 * j);
        }
    };
    fetch(0);
    bool far = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) far |= far_scale(sa[i]);
    const bool any_far = __any(far);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long m = mw + 16 * i + frow;
        if (i < 7) fetch(i + 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v[8], sum[8];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const auto s = __builtin_amdgcn_permlane16_swap((unsigned)acc[i][2 * j][c], (unsigned)acc[i][2 * j + 1][c], false, false);
                sum[c] = (float)(int)s[0];
                sum[4 + c] = (float)(int)s[1];
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = fmaf(sum[c] * sa[i], w[j][c], b[j][c]);
            if (__builtin_expect(any_far, 0)) {   // (selecting both factors in every output, or the loop twice, cost up to 3 %)
                if (far_scale(sa[i])) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) v[c] = fmaf(sum[c] * w[j][c], sa[i], b[j][c]);
                }
            }
            if (residual) {
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] += (float)side[i & 1][j][c];
            }
            if (act) {
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = silu_fast(v[c]);
            }
            const int n = nl + 32 * j;
            Out* out = static_cast<Out*>(p.out) + m * p.ldo + n;
            Side o;
#pragma unroll
            for (int c = 0; c < 8; ++c) o[c] = (Out)v[c];
            if (m >= m_lo) {
                if (n >= n_lo) {
                    *reinterpret_cast<SideAny*>(out) = o;
                } else if constexpr (!WHOLE) {
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (n + c >= n_lo) out[c] = o[c];
                }
            }
        }
    }
}

template <typename Out, int SIDE, bool WHOLE>
int launch_w4(const I8Params& p, hipStream_t stream) {
    constexpr int smem = 2 * 65536;
    static std::atomic<bool> done[64];
    const int rc = allow_lds("gemm_i8", reinterpret_cast<const void*>(&gemm_i8_w4_kernel<Out, SIDE, WHOLE>), smem, done);
    if (rc != ADCDIFF_OK) return rc;
    const long long tiles = (((long long)p.M + 255) / 256) * (((long long)p.N + 255) / 256);
    if (tiles > 0xffffff) return fail(ADCDIFF_E_BADARG, "gemm_i8: %d x %d outputs are too many for one call", p.M, p.N);
    hipLaunchKernelGGL((gemm_i8_w4_kernel<Out, SIDE, WHOLE>), dim3((unsigned)tiles), dim3(256), smem, stream, p);
    return check_launch("gemm_i8");
}

template <typename Out, int SIDE>
int launch_w4_shape(const I8Params& p, hipStream_t stream) {
    return p.N % 8 == 0 ? launch_w4<Out, SIDE, true>(p, stream) : launch_w4<Out, SIDE, false>(p, stream);
}

template <typename Out>
int launch_w4_side(const I8Params& p, hipStream_t stream) {
    if (p.act) return p.residual ? launch_w4_shape<Out, 3>(p, stream) : launch_w4_shape<Out, 2>(p, stream);
    return p.residual ? launch_w4_shape<Out, 1>(p, stream) : launch_w4_shape<Out, 0>(p, stream);
}

template <typename Out, int BM, int BN, int WAVES, int DEPTH>
int launch_split(const I8Params& p, hipStream_t stream) {
    const long long tiles = (((long long)p.M + BM - 1) / BM) * (((long long)p.N + BN - 1) / BN);
    if (tiles * WAVES * 64 > 0xffffffffLL) return fail(ADCDIFF_E_BADARG, "gemm_i8: %d x %d outputs are too many for one call", p.M, p.N);
    hipLaunchKernelGGL((gemm_i8_split_kernel<Out, BM, BN, WAVES, DEPTH>), dim3((unsigned)tiles), dim3(64 * WAVES), 0, stream, p);
    return check_launch("gemm_i8");
}

template <typename Out, int BM, int BN, int STAGES>
int launch_ring(const I8Params& p, hipStream_t stream) {
    constexpr int smem = std::max((BM + BN) * 128 * STAGES, BM * (BN + 4) * 4);
    static std::atomic<bool> done[64];
    const int rc = allow_lds("gemm_i8", reinterpret_cast<const void*>(&gemm_i8_ring_kernel<Out, BM, BN, STAGES>), smem, done);
    if (rc != ADCDIFF_OK) return rc;
    const long long tiles = (((long long)p.M + BM - 1) / BM) * (((long long)p.N + BN - 1) / BN);
    if (tiles > 0x7fffff) return fail(ADCDIFF_E_BADARG, "gemm_i8: %d x %d outputs are too many for one call", p.M, p.N);
    hipLaunchKernelGGL((gemm_i8_ring_kernel<Out, BM, BN, STAGES>), dim3((unsigned)tiles), dim3(512), smem, stream, p);
    return check_launch("gemm_i8");
}

// Which kernel: measured on all of them over 1..65536 rows, 512..4096 outputs, 512..8192 columns (us, M x N x K).
//   few rows: the smallest split tile that still gives at most one workgroup per CU
//     32 x 2048 x 4096: 16 x 16 tile 7.1, 32 x 16 8.6, 32 x 32 10.2;  64 x 2048 x 2048: 6.9, 6.0, 6.7;  128 x 2048 x 2048: 11.4, 8.8, 7.2, 64 x 64 ring 7.9
//   more: the least of three estimates fitted to the measured times (kt: K tiles of 128, r: tiles / 256 CUs, at least 1)
//     64 x 64 ring     2.0 + 0.65 r + (0.09 + 0.25 r) kt:   512 x 2048 x 2048 8.6 (128 x 128: 15.0, 256 x 256: 25.6), 1024 x 2048 x 2048 11.2 (15.9, 26.0)
//     128 x 128 ring   3.7 + 2.9 r + (0.23 + 0.42 r) kt:    2048 x 2048 x 2048 16.8 (20.6, 27.3), 4096 x 2048 x 2048 26.0 (37.9, 29.4)
//     256 x 256        a round of 256 workgroups 10.9 + 1.45 kt, one of at most 128 11 + 1.1 kt:  8192 x 2048 x 2048 34.1 (66.9, 46.1), 65536 x 512 x 512 33.4 (52.8, 41.9)
// The result names the tile: 16 (16 x 16), 3216 (32 x 16), 32 (32 x 32), 64, 128, 256.
int choose_kernel(const I8Params& p, bool whole256) {
    auto tiles = [&](int bm, int bn) { return (((long long)p.M + bm - 1) / bm) * (((long long)p.N + bn - 1) / bn); };
    if (p.M <= 16 || tiles(16, 16) <= 256) return 16;
    if (tiles(32, 16) <= 256) return 3216;
    if (tiles(32, 32) <= 256) return 32;
    const double kt = (p.K + 127) / 128;
    const double r64 = std::max(1.0, tiles(64, 64) / 256.0), r128 = std::max(1.0, tiles(128, 128) / 256.0);
    const double t64 = 2.0 + 0.65 * r64 + (0.09 + 0.25 * r64) * kt, t128 = 3.7 + 2.9 * r128 + (0.23 + 0.42 * r128) * kt;
    if (whole256) {
        const long long n = tiles(256, 256), last = n % 256;
        const double t256 = (double)((n + 127) / 256) * (10.9 + 1.45 * kt) + (last > 0 && last <= 128 ? 11.0 + 1.1 * kt : 0.0);
        if (t256 < std::min(t64, t128)) return 256;
    }
    return t64 < t128 ? 64 : 128;
}

template <typename Out>
int launch_gemm(const I8Params& p, hipStream_t stream) {
    // the 256 x 256 kernel needs whole tiles in every direction and 32-bit offsets inside them
    const bool whole256 = p.M >= 256 && p.N >= 256 && p.K >= 256 && p.lda < (1 << 23) && p.ldw < (1 << 23);
    const long long forced = debug_value(DBG_GEMM_I8_KERNEL);
    if (forced == 256 && !whole256) return fail(ADCDIFF_E_BADARG, "gemm_i8: gemm_i8_kernel = 256 asks for M, N and K of 256 and pitches below 2^23, got %d x %d x %d", p.M, p.N, p.K);
    switch (forced ? forced : choose_kernel(p, whole256)) {
        case 16: return launch_split<Out, 16, 16, 8, 4>(p, stream);
        case 3216: return launch_split<Out, 32, 16, 8, 4>(p, stream);
        case 32: return launch_split<Out, 32, 32, 8, 2>(p, stream);
        case 64: return launch_ring<Out, 64, 64, 3>(p, stream);
        case 128: return launch_ring<Out, 128, 128, 2>(p, stream);
        case 256: return launch_w4_side<Out>(p, stream);
    }
    return fail(ADCDIFF_E_BADARG, "gemm_i8: gemm_i8_kernel = %lld names no kernel", forced);
}

constexpr int kMaxK = 131071;   // 128 * 128 * K stays below 2^31
constexpr int kMaxRow = 1 << 30;   // columns of a quantised row: 32-bit counters step 1024 past the last one

}  // namespace
}  // namespace adcdiff

extern "C" int adcdiff_quantize_rows(const void* x, long long ldx, int dtype, int M, int K, int8_t* q, long long ldq, float* scale, adcdiff_stream_t stream_) {
    using namespace adcdiff;
    if (M < 0 || K < 1 || K > kMaxRow) return fail(ADCDIFF_E_BADARG, "quantize_rows: %d rows of %d columns (1..%d)", M, K, kMaxRow);
    if (!type_ok(dtype)) return fail(ADCDIFF_E_BADARG, "quantize_rows: type %d", dtype);
    if (M == 0) return ADCDIFF_OK;
    if (!x || !q || !scale) return fail(ADCDIFF_E_BADARG, "quantize_rows: null pointer");
    if (ldx < K || ldq < K) return fail(ADCDIFF_E_BADARG, "quantize_rows: a row pitch below %d columns", K);
    hipStream_t stream = as_stream(stream_);
    const int Kp = (int)std::min<long long>(ldq, ((long long)K + 15) / 16 * 16);
    TimingScope timing(ADCDIFF_KIND_OTHER, M, K, 0, 0.0, (double)M * K * (type_size(dtype) + 1), stream);
    const bool pairs = Kp % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0 && ldq % 8 == 0;
    const QuantizeArgs a{x, ldx, M, K, Kp, q, ldq, scale};
    if (dtype == ADCDIFF_BF16) {
        if (pairs) quantize_by_shape<bf16_t, true>(a, stream);
        else quantize_by_shape<bf16_t, false>(a, stream);
    } else {
        if (pairs) quantize_by_shape<float, true>(a, stream);
        else quantize_by_shape<float, false>(a, stream);
    }
    return check_launch("quantize_rows");
}

extern "C" int adcdiff_pitch_rows_i8(const adcdiff_i8_copy* copies, int n, adcdiff_stream_t stream_) {
    using namespace adcdiff;
    if (!copies || n < 1 || n > 2) return fail(ADCDIFF_E_BADARG, "pitch_rows_i8: null table or %d copies", n);
    PitchParams p{};
    long long blocks[2] = {0, 0};
    double bytes = 0.0;
    for (int i = 0; i < n; ++i) {
        const adcdiff_i8_copy& c = copies[i];
        if (c.M < 0 || c.K < 1 || c.ld_src < c.K || c.ld_dst < c.K || c.ld_dst % 16 != 0)
            return fail(ADCDIFF_E_BADARG, "pitch_rows_i8: %d rows of %d columns, pitches %lld -> %lld", c.M, c.K, c.ld_src, c.ld_dst);
        if (c.M > 0 && (!c.src || !c.dst || !aligned16(c.dst))) return fail(ADCDIFF_E_BADARG, "pitch_rows_i8: null pointer, or a destination off its 16-byte boundary");
        p.c[i] = c;
        blocks[i] = (c.ld_dst / 16 * c.M + 255) / 256;
        bytes += 2.0 * c.M * c.K;
    }
    if (blocks[0] + blocks[1] > 0xffffff) return fail(ADCDIFF_E_BADARG, "pitch_rows_i8: too many rows");
    if (blocks[0] + blocks[1] == 0) return ADCDIFF_OK;
    p.first = (unsigned)blocks[0];
    hipStream_t stream = as_stream(stream_);
    TimingScope timing(ADCDIFF_KIND_OTHER, copies[0].M, copies[0].K, 0, 0.0, bytes, stream);
    hipLaunchKernelGGL(pitch_rows_kernel, dim3((unsigned)(blocks[0] + blocks[1])), dim3(256), 0, stream, p);
    return check_launch("pitch_rows_i8");
}

namespace adcdiff {
namespace {
int check_gemm(const adcdiff_gemm_i8_args* a) {
    if (!a) return fail(ADCDIFF_E_BADARG, "gemm_i8: null args");
    if (a->M < 0 || a->N < 1 || a->K < 1 || a->K > kMaxK) return fail(ADCDIFF_E_BADARG, "gemm_i8: M %d, N %d, K %d (1..%d)", a->M, a->N, a->K, kMaxK);
    if (!type_ok(a->out_dtype) || (a->act != 0 && a->act != 1)) return fail(ADCDIFF_E_BADARG, "gemm_i8: type %d, act %d", a->out_dtype, a->act);
    if (a->M == 0) return ADCDIFF_OK;
    if (!a->a || !a->w || !a->a_scale || !a->w_scale || !a->out) return fail(ADCDIFF_E_BADARG, "gemm_i8: null pointer");
    if (!aligned16(a->a) || !aligned16(a->w) || a->lda % 16 != 0 || a->ldw % 16 != 0 || a->lda < a->K || a->ldw < a->K)
        return fail(ADCDIFF_E_BADARG, "gemm_i8: the rows of a and w start on 16-byte boundaries and hold %d columns (pitches %lld, %lld)", a->K, a->lda, a->ldw);
    if (a->ldo < a->N || (a->residual && a->ldr < a->N)) return fail(ADCDIFF_E_BADARG, "gemm_i8: a row pitch below %d columns", a->N);
    return ADCDIFF_OK;
}
}  // namespace
}  // namespace adcdiff

extern "C" int adcdiff_gemm_i8(const adcdiff_gemm_i8_args* a, adcdiff_stream_t stream_) {
    using namespace adcdiff;
    const int rc = check_gemm(a);
    if (rc != ADCDIFF_OK || a->M == 0) return rc;
    hipStream_t stream = as_stream(stream_);
    I8Params p{a->a, a->w, a->a_scale, a->w_scale, a->bias, a->residual, a->out, a->lda, a->ldw, a->ldr, a->ldo, a->M, a->N, a->K, a->act};
    const int so = type_size(a->out_dtype);
    TimingScope timing(ADCDIFF_KIND_OTHER, a->M, a->N, a->K, 2.0 * a->M * a->N * a->K,
                       (double)a->M * a->K + (double)a->N * a->K + (double)a->M * a->N * so * (a->residual ? 2 : 1), stream);
    return a->out_dtype == ADCDIFF_BF16 ? launch_gemm<bf16_t>(p, stream) : launch_gemm<float>(p, stream);
}

extern "C" size_t adcdiff_linear_i8_workspace_bytes(int M, int K) {
    if (M < 0 || K < 1) return 0;
    return ((size_t)K + 15) / 16 * 16 * (size_t)M + 4 * (size_t)M + 16;
}

extern "C" int adcdiff_linear_i8(const void* x, long long ldx, int dtype, const adcdiff_gemm_i8_args* a, void* workspace, size_t workspace_bytes,
                                 adcdiff_stream_t stream) {
    using namespace adcdiff;
    if (!a || a->M < 0 || a->K < 1) return fail(ADCDIFF_E_BADARG, "linear_i8: null args, or %d rows of %d columns", a ? a->M : 0, a ? a->K : 0);
    const size_t need = adcdiff_linear_i8_workspace_bytes(a->M, a->K);
    if (!workspace || !aligned16(workspace) || workspace_bytes < need)
        return fail(ADCDIFF_E_WORKSPACE, "linear_i8: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    const long long pitch = ((long long)a->K + 15) / 16 * 16;
    adcdiff_gemm_i8_args g = *a;
    g.a = static_cast<const int8_t*>(workspace);
    g.lda = pitch;
    g.a_scale = reinterpret_cast<const float*>(g.a + pitch * a->M);
    int rc = check_gemm(&g);     // before the first launch: a refused call leaves nothing behind
    if (rc != ADCDIFF_OK) return rc;
    rc = adcdiff_quantize_rows(x, ldx, dtype, a->M, a->K, static_cast<int8_t*>(workspace), pitch, const_cast<float*>(g.a_scale), stream);
    return rc != ADCDIFF_OK ? rc : adcdiff_gemm_i8(&g, stream);
}

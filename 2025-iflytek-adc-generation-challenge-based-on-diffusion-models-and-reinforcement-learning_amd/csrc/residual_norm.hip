// The norms before and after a residual block, fused with the block's gate and the residual scale, and their gradients:
//   x' = residual_scale * x + gate . N_post(h),   y = N_pre(x'),   N(v) = (v - [mean]) / sqrt(mean((v - [mean])^2) + eps) . weight + bias
// The bracketed mean belongs to the layer norm; the rms norm has none.  All arithmetic is float32; h, y share one type, x, x' another,
// the gate has its own, and each output is rounded once.  y is formed from the unrounded x'.
//
// A team of TPR threads owns a row and holds it in registers (8 columns per thread), so every pass over the row after the
// first load is free; both kernels are bound by HBM.  Statistics are two-pass (mean, then centred squares) on those registers.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "row_access.h"

namespace adcdiff {
namespace {

struct ResNormParams {
    const void *h, *x, *gate;
    const float *post_w, *post_b, *pre_w, *pre_b;
    void *xn, *y;
    float* stats;                 // [M, 4]: post mean, 1 / post deviation, pre mean, 1 / pre deviation
    long long ldh, ldx, ldg, ldxn, ldy;
    int M, D, post, pre, gate_bf16, gate_share;   // gate_share: rows per gate row
    int crossing;                 // x is overwritten in place and a row's last thread moves back over a wave's end
    float scale, eps, inv_d;
};

struct ResNormGradParams {
    ResNormParams f;
    const void *d_xn, *d_y;
    void *d_h, *d_x, *d_gate;
    long long ld_dxn, ld_dy, ld_dh, ld_dx, ld_dg;
    float* partial;               // [workgroups][vectors][D] weight and bias gradients of a workgroup's rows
    float* gate_partial;          // [chunks][D] gate gradients, where several chunks share a gate row
    int slot_post_w, slot_post_b, slot_pre_w, slot_pre_b, vectors;   // row of each vector in a workgroup's partials, or -1
    int chunks, chunk_rows, chunks_per_gate;
    int group_rows;               // rows of one gate row (M where the gate's gradient is not summed over rows)
};

// A gate row of either type
template <RowShape SHAPE>
struct RawGate {
    RawRow<float, SHAPE> f;
    __device__ __forceinline__ void clear() { f.clear(); }
    __device__ __forceinline__ void load(const void* gate, int bf16, long long offset, int t, int D) {
        if (bf16) {
            RawRow<bf16_t, SHAPE> b;
            b.load(static_cast<const bf16_t*>(gate) + offset, t, D);
#pragma unroll
            for (int i = 0; i < RawRow<bf16_t, SHAPE>::N; ++i) f.r[i] = b.r[i];
        } else {
            f.load(static_cast<const float*>(gate) + offset, t, D);
        }
    }
    __device__ __forceinline__ void get(int bf16, float (&v)[8]) const {
        if (bf16) {
            RawRow<bf16_t, SHAPE> b;
#pragma unroll
            for (int i = 0; i < RawRow<bf16_t, SHAPE>::N; ++i) b.r[i] = f.r[i];
            b.get(v);
        } else {
            f.get(v);
        }
    }
};

// a weight or bias, or what it is without one
template <RowShape SHAPE>
__device__ __forceinline__ void load_vector(const float* p, float absent, int t, int D, float (&v)[8]) {
    RawRow<float, SHAPE> r;
    r.clear();
    if (p) r.load(p, t, D);
    r.get(v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = p ? v[e] : absent;
}

// mean and 1 / sqrt(variance + eps) of the row in v (mean = 0 for the rms norm); `in`: the elements that count
template <typename Sum>
__device__ __forceinline__ void row_stats(const float (&v)[8], int kind, unsigned in, int tid, float inv_d, float eps, Sum& sum, float& mean, float& inv) {
    float s[1] = {0.0f};
    mean = 0.0f;
    if (kind == 2) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[0] += in >> e & 1 ? v[e] : 0.0f;
        sum(s, tid);
        mean = s[0] * inv_d;
        s[0] = 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float c = in >> e & 1 ? v[e] - mean : 0.0f;
        s[0] = fmaf(c, c, s[0]);
    }
    sum(s, tid);
    inv = 1.0f / sqrtf(fmaf(s[0], inv_d, eps));
}

// A team of TPR threads per row, eight columns per thread; weights, biases and a gate shared by all rows stay in registers over the rows of a
// workgroup, and the next row is on its way while the one in hand is reduced.
// Bound by HBM: 65536 x 2048 bfloat16 with a gate for each row 267 us (1.34 GB at 5.0 TB/s), 4096 x 1024 float32 17 us; 32 x 512: 3.8 us, a latency.
template <typename T, typename R, RowShape SHAPE, int TPR>
__global__ __launch_bounds__(threads_for<TPR>()) void residual_norm_kernel(const ResNormParams p) {
    constexpr int THREADS = threads_for<TPR>(), TEAMS = THREADS / TPR;
    __shared__ float red[2 * (THREADS / 64)];
    const int tid = threadIdx.x, t = TEAMS == 1 ? tid : tid % TPR, team = TEAMS == 1 ? 0 : tid / TPR, D = p.D;
    const unsigned in = own_columns<SHAPE>(t, D);
    const bool one_gate = p.gate && p.gate_share >= p.M, row_gate = p.gate && !one_gate;
    RawRow<R, SHAPE> rx;
    RawRow<T, SHAPE> rh;
    RawGate<SHAPE> rg;
    rx.clear(); rh.clear(); rg.clear();
    auto fetch = [&](long long row) __attribute__((always_inline)) {
        if (row < p.M) {
            rx.load(static_cast<const R*>(p.x) + row * p.ldx, t, D);
            if (p.h) rh.load(static_cast<const T*>(p.h) + row * p.ldh, t, D);
            if (row_gate) rg.load(p.gate, p.gate_bf16, (p.gate_share == 1 ? row : row / p.gate_share) * p.ldg, t, D);
        }
    };
    const long long step = (long long)gridDim.x * TEAMS;
    fetch((long long)blockIdx.x * TEAMS + team);
    float post_w[8], post_b[8], pre_w[8], pre_b[8], gate[8];
    load_vector<SHAPE>(p.post_w, 1.0f, t, D, post_w);
    load_vector<SHAPE>(p.post_b, 0.0f, t, D, post_b);
    load_vector<SHAPE>(p.pre_w, 1.0f, t, D, pre_w);
    load_vector<SHAPE>(p.pre_b, 0.0f, t, D, pre_b);
#pragma unroll
    for (int e = 0; e < 8; ++e) gate[e] = 1.0f;
    if (one_gate) {
        RawGate<SHAPE> g;
        g.load(p.gate, p.gate_bf16, 0, t, D);
        g.get(p.gate_bf16, gate);
    }
    TeamSum<TPR, 1> sum(red);
    // every team of a workgroup makes the same turns: the sums of teams wider than a wave have barriers in them
    for (long long base = (long long)blockIdx.x * TEAMS; base < p.M; base += step) {
        const long long row = base + team;
        const bool live = row < p.M;
        float v[8], u[8];
        rx.get(v);
        rh.get(u);
        if (row_gate) rg.get(p.gate_bf16, gate);
        fetch(row + step);
        float post_mean = 0.0f, post_inv = 1.0f, pre_mean = 0.0f, pre_inv = 1.0f;
        if (p.h) {
            if (p.post) {
                row_stats(u, p.post, in, tid, p.inv_d, p.eps, sum, post_mean, post_inv);
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] = fmaf((u[e] - post_mean) * post_inv, post_w[e], post_b[e]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf(p.scale, v[e], gate[e] * u[e]);
        }
        if constexpr (SHAPE == kMoved) {
            if (p.crossing) {   // every wave has its part of the row (and of the next one)
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
            }
        }
        if (p.xn && live) store_row<R, SHAPE>(static_cast<R*>(p.xn) + row * p.ldxn, t, D, v);
        if (p.pre) {
            row_stats(v, p.pre, in, tid, p.inv_d, p.eps, sum, pre_mean, pre_inv);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf((v[e] - pre_mean) * pre_inv, pre_w[e], pre_b[e]);
            if (live) store_row<T, SHAPE>(static_cast<T*>(p.y) + row * p.ldy, t, D, v);
        }
        if (p.stats && t == 0 && live) *reinterpret_cast<f32x4*>(p.stats + row * 4) = f32x4{post_mean, post_inv, pre_mean, pre_inv};
    }
}

// Eight column sums of a thread.  In registers, or (a team of 1024 threads has 128 registers per thread) in LDS, where each thread owns its words.
template <bool IN_LDS>
struct ColumnSums {
    float a[8];
    __device__ __forceinline__ void init(float*, int) {
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = 0.0f;
    }
    __device__ __forceinline__ void add_product(const float (&x)[8], const float (&y)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = fmaf(x[e], y[e], a[e]);
    }
    __device__ __forceinline__ void add(const float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] += x[e];
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = a[e];
    }
};
template <>
struct ColumnSums<true> {
    f32x4* p;   // two vectors of four, 1024 threads apart
    __device__ __forceinline__ void init(float* lds, int tid) {
        p = reinterpret_cast<f32x4*>(lds) + tid;
        p[0] = p[1024] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ void add_product(const float (&x)[8], const float (&y)[8]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 v = p[1024 * h];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = fmaf(x[4 * h + e], y[4 * h + e], v[e]);
            p[1024 * h] = v;
        }
    }
    __device__ __forceinline__ void add(const float (&x)[8]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 v = p[1024 * h];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += x[4 * h + e];
            p[1024 * h] = v;
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = p[1024 * (e >> 2)][e & 3];
    }
};
constexpr int kWideSums = 4 * 8 * 1024 * 4;   // bytes of LDS for the four vectors of a team of 1024

// Gradients.  With u = N_post(h), xhat / uhat the normalised rows, g the gradient of a norm's output times its weight:
//   d = d_x' + (g - [mean g] - xhat mean(g xhat)) / deviation      (g = d_y . pre_weight)
//   d_x = residual_scale d,   d_gate = d . u,   d_h = N_post's gradient of d . gate,   d_weight = sum over rows of d_y . xhat, ...
// x' and u are formed again from h and x in float32 (the rounded x' would cost the same traffic as x and lose bits); the statistics
// come from the forward pass.  The rows are cut into chunks of consecutive rows that share a gate row; a team runs over chunks with
// its column sums in registers, so weights cost one partial row per workgroup and the gate one row per chunk.  The partial rows are
// added in a fixed order by column_sum_kernel: no atomics, results do not change from run to run.
// Bound by HBM up to 4096 columns: 32768 x 2048 bfloat16 blocks on a float32 stream 250 us (1.21 GB at 4.8 TB/s), 4096 x 1024 float32 24 us; by the
// rows' latency where a row takes a whole CU (8192 x 8192: 223 us, 3.6 TB/s).
template <typename T, typename R, RowShape SHAPE, int TPR>
__global__ __launch_bounds__(threads_for<TPR>()) void residual_norm_grad_kernel(const ResNormGradParams q) {
    constexpr int THREADS = threads_for<TPR>(), TEAMS = THREADS / TPR;
    constexpr bool WIDE = TPR == 1024;
    constexpr int TPW = TPR < 64 ? TPR : 64;   // columns of a wave in `joined`: a wave's own teams are added by shuffles first
    __shared__ float red[4 * (THREADS / 64)];
    __shared__ float joined[TEAMS > 1 ? THREADS / 64 * TPW * 8 : 1];
    extern __shared__ __attribute__((aligned(16))) float wide[];     // kWideSums bytes where WIDE
    const ResNormParams& p = q.f;
    const int tid = threadIdx.x, t = TEAMS == 1 ? tid : tid % TPR, team = TEAMS == 1 ? 0 : tid / TPR, D = p.D;
    const unsigned in = own_columns<SHAPE>(t, D);
    TeamSum<TPR, 2> sum(red);
    ColumnSums<WIDE> a_pre_w, a_pre_b, a_post_w, a_post_b;
    a_pre_w.init(wide, tid);
    a_pre_b.init(wide + 8192, tid);
    a_post_w.init(wide + 2 * 8192, tid);
    a_post_b.init(wide + 3 * 8192, tid);
    // Teams of 768 and 1024 threads have 168 and 128 registers per thread.  They load weights where they are used and no row ahead, and a row's raw
    // values end with its turn (kept over turns they spilled: 8192 x 8192 bfloat16 461 us against 223 us).
    constexpr bool LEAN = TPR > 512;
    float post_w[8], post_b[8], pre_w[8];
    if constexpr (!LEAN) {
        load_vector<SHAPE>(p.post_w, 1.0f, t, D, post_w);
        load_vector<SHAPE>(p.post_b, 0.0f, t, D, post_b);
        load_vector<SHAPE>(p.pre_w, 1.0f, t, D, pre_w);
    }
    const bool row_gate = p.gate && p.gate_share == 1;
    const int teams = gridDim.x * TEAMS;
    // Every team of a workgroup makes the same number of turns (barriers inside the sums); turns without a row do nothing.
    for (int c0 = blockIdx.x * TEAMS; c0 < q.chunks; c0 += teams) {
        const int c = c0 + team;
        const int group = c / q.chunks_per_gate;
        const long long first = (long long)group * q.group_rows + (long long)(c % q.chunks_per_gate) * q.chunk_rows;
        const long long last = c < q.chunks ? min(first + q.chunk_rows, (long long)(group + 1) * q.group_rows) : first;
        RawRow<R, SHAPE> rx, rd;
        RawRow<T, SHAPE> rh, ry;
        RawGate<SHAPE> rg;
        f32x4 rs = {0.0f, 1.0f, 0.0f, 1.0f};
        rx.clear(); rd.clear(); rh.clear(); ry.clear(); rg.clear();
        long long gate_row = -1;
        auto fetch = [&](long long row) __attribute__((always_inline)) {
            if (row < last) {
                if (p.post || p.pre) rs = *reinterpret_cast<const f32x4*>(p.stats + row * 4);
                if (q.d_xn) rd.load(static_cast<const R*>(q.d_xn) + row * q.ld_dxn, t, D);
                if (p.pre) rx.load(static_cast<const R*>(p.x) + row * p.ldx, t, D);
                if (p.h) rh.load(static_cast<const T*>(p.h) + row * p.ldh, t, D);
                if (q.d_y) ry.load(static_cast<const T*>(q.d_y) + row * q.ld_dy, t, D);
                if (p.gate) {
                    const long long g = row_gate ? row : row / p.gate_share;
                    if (LEAN || g != gate_row) rg.load(p.gate, p.gate_bf16, g * p.ldg, t, D);
                    gate_row = g;
                }
            }
        };
        if constexpr (!LEAN) fetch(first);
        float a_gate[8] = {}, gate[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) gate[e] = 1.0f;
        for (int r = 0; r < q.chunk_rows; ++r) {
            const long long row = first + r;
            const bool live = row < last;
            float d[8], v[8], u[8], uhat[8], g[8], s[2];
            if constexpr (LEAN) {
                rx.clear(); rd.clear(); rh.clear(); ry.clear(); rg.clear();
                fetch(row);
            }
            const f32x4 st = rs;
            rd.get(d);
            rx.get(v);
            rh.get(u);
            ry.get(g);
            if (p.gate) rg.get(p.gate_bf16, gate);
            if constexpr (!LEAN) fetch(row + 1);   // under this row's arithmetic
            if (p.h) {
                if constexpr (LEAN) {
                    load_vector<SHAPE>(p.post_w, 1.0f, t, D, post_w);
                    load_vector<SHAPE>(p.post_b, 0.0f, t, D, post_b);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    uhat[e] = u[e];
                    if (p.post) {
                        uhat[e] = (u[e] - st[0]) * st[1];
                        u[e] = fmaf(uhat[e], post_w[e], post_b[e]);
                    }
                    v[e] = fmaf(p.scale, v[e], gate[e] * u[e]);
                }
            }
            if (p.pre) {
                if constexpr (LEAN) load_vector<SHAPE>(p.pre_w, 1.0f, t, D, pre_w);
                s[0] = s[1] = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = (v[e] - st[2]) * st[3];
                }
                if (live) {
                    a_pre_w.add_product(g, v);
                    a_pre_b.add(g);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    g[e] *= pre_w[e];
                    if (in >> e & 1) { s[0] += g[e]; s[1] = fmaf(g[e], v[e], s[1]); }
                }
                sum(s, tid);
                const float m0 = p.pre == 2 ? s[0] * p.inv_d : 0.0f, m1 = s[1] * p.inv_d;
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = fmaf(g[e] - m0 - v[e] * m1, st[3], d[e]);
            }
            if (q.d_x && live) {
                float o[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = p.scale * d[e];
                store_row<R, SHAPE>(static_cast<R*>(q.d_x) + row * q.ld_dx, t, D, o);
            }
            if (p.h) {
                if (q.d_gate && live) {
                    if (row_gate) {
                        float o[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] = d[e] * u[e];
                        if (p.gate_bf16) store_row<bf16_t, SHAPE>(static_cast<bf16_t*>(q.d_gate) + row * q.ld_dg, t, D, o);
                        else store_row<float, SHAPE>(static_cast<float*>(q.d_gate) + row * q.ld_dg, t, D, o);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) a_gate[e] = fmaf(d[e], u[e], a_gate[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] *= gate[e];
                if (p.post) {
                    if constexpr (LEAN) load_vector<SHAPE>(p.post_w, 1.0f, t, D, post_w);
                    if (live) {
                        a_post_w.add_product(d, uhat);
                        a_post_b.add(d);
                    }
                    s[0] = s[1] = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        d[e] *= post_w[e];
                        if (in >> e & 1) { s[0] += d[e]; s[1] = fmaf(d[e], uhat[e], s[1]); }
                    }
                    sum(s, tid);
                    const float m0 = p.post == 2 ? s[0] * p.inv_d : 0.0f, m1 = s[1] * p.inv_d;
#pragma unroll
                    for (int e = 0; e < 8; ++e) d[e] = (d[e] - m0 - uhat[e] * m1) * st[1];
                }
                if (q.d_h && live) store_row<T, SHAPE>(static_cast<T*>(q.d_h) + row * q.ld_dh, t, D, d);
            }
        }
        if (q.d_gate && !row_gate && c < q.chunks) {
            if (q.chunks_per_gate > 1) store_row<float, SHAPE>(q.gate_partial + (long long)c * D, t, D, a_gate);
            else if (p.gate_bf16) store_row<bf16_t, SHAPE>(static_cast<bf16_t*>(q.d_gate) + group * q.ld_dg, t, D, a_gate);
            else store_row<float, SHAPE>(static_cast<float*>(q.d_gate) + group * q.ld_dg, t, D, a_gate);
        }
    }
    float* out = q.partial + (long long)blockIdx.x * q.vectors * D;
    auto flush = [&](const ColumnSums<WIDE>& sums, int slot) {
        if (slot < 0) return;
        float a[8];
        sums.get(a);
        if constexpr (TEAMS > 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int m = TPR; m < 64; m <<= 1) a[e] += __shfl_xor(a[e], m);
            __syncthreads();
            const int row = tid / 64, col = tid % TPW;
            if (TPR >= 64 || (tid & 63) < TPR) {
#pragma unroll
                for (int e = 0; e < 8; ++e) joined[(row * 8 + e) * TPW + col] = a[e];
            }
            __syncthreads();
            if (team == 0) {   // waves of the same columns: every WAVES-th one
                constexpr int WAVES = TPR > 64 ? TPR / 64 : 1;
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int k = WAVES; k < THREADS / 64; k += WAVES) a[e] += joined[((row + k) * 8 + e) * TPW + col];
            }
        }
        if (team == 0) store_row<float, SHAPE>(out + (long long)slot * D, t, D, a);
    };
    flush(a_pre_w, q.slot_pre_w);
    flush(a_pre_b, q.slot_pre_b);
    flush(a_post_w, q.slot_post_w);
    flush(a_post_b, q.slot_post_b);
}

// The partial rows added up in a fixed order.  Segments 0 .. vectors - 1 are the weight and bias gradients (a partial row from each
// workgroup), the others the gate rows (one from each chunk).  Tall sums: a workgroup takes 32 columns of a segment with 32 threads down the rows and
// a tree over them.  Gate rows of few chunks (flat): a thread takes one element; the tall form would start 1024 threads for every
// 32 columns of every gate row (64 gate rows of 8 chunks, D = 2048: 13.4 us for 12 MB).
struct ColumnSumParams {
    const float *partial, *gate_partial;
    float* out[4];
    void* d_gate;
    long long ld_dg, flat;      // flat: elements summed by single threads (gate rows x D, or 0)
    int D, vectors, tall, workgroups, chunks_per_gate, gate_bf16;   // tall: segments summed by whole workgroups
};

__device__ __forceinline__ void store_gate(const ColumnSumParams& p, long long row, int col, float v) {
    if (p.gate_bf16) static_cast<bf16_t*>(p.d_gate)[row * p.ld_dg + col] = (bf16_t)v;
    else static_cast<float*>(p.d_gate)[row * p.ld_dg + col] = v;
}

__global__ __launch_bounds__(1024) void column_sum_kernel(const ColumnSumParams p) {
    __shared__ float part[32][33];
    const int blocks = (p.D + 31) / 32;
    const long long tall_blocks = (long long)blocks * p.tall;
    if (blockIdx.x < tall_blocks) {
        const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
        const int seg = blockIdx.x / blocks, col = blockIdx.x % blocks * 32 + cx;
        const bool weight = seg < p.vectors;
        const float* src = weight ? p.partial + (long long)seg * p.D : p.gate_partial + (long long)(seg - p.vectors) * p.chunks_per_gate * p.D;
        const long long step = weight ? (long long)p.vectors * p.D : p.D;
        const int count = weight ? p.workgroups : p.chunks_per_gate;
        float s = 0.0f;
        if (col < p.D) {
#pragma unroll 4
            for (int i = ry; i < count; i += 32) s += src[i * step + col];
        }
        part[ry][cx] = s;
        __syncthreads();
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) {
            if (ry < m) part[ry][cx] += part[ry + m][cx];
            __syncthreads();
        }
        if (ry == 0 && col < p.D) {
            if (weight) p.out[seg][col] = part[0][cx];
            else store_gate(p, seg - p.vectors, col, part[0][cx]);
        }
        return;
    }
    const long long stride = (gridDim.x - tall_blocks) * 1024;
    for (long long e = (blockIdx.x - tall_blocks) * 1024 + threadIdx.x; e < p.flat; e += stride) {
        const long long row = e / p.D;
        const int col = (int)(e - row * p.D);
        const float* src = p.gate_partial + row * p.chunks_per_gate * p.D + col;
        float s = 0.0f;
#pragma unroll 8
        for (int i = 0; i < p.chunks_per_gate; ++i) s += src[(long long)i * p.D];
        store_gate(p, row, col, s);
    }
}

bool norm_kind(int k) { return k >= 0 && k <= 2; }

constexpr int kMaxD = 8192;

int check_args(const char* who, const adcdiff_residual_norm_args* a) {
    if (!a) return fail(ADCDIFF_E_BADARG, "%s: null args", who);
    if (a->M < 0 || a->D < 1 || a->D > kMaxD) return fail(ADCDIFF_E_BADARG, "%s: %d rows of %d columns (1..%d)", who, a->M, a->D, kMaxD);
    if (!type_ok(a->dtype) || !type_ok(a->stream_dtype) || (a->gate && !type_ok(a->gate_dtype)))
        return fail(ADCDIFF_E_BADARG, "%s: types %d, %d, %d are not ADCDIFF_F32 / ADCDIFF_BF16", who, a->dtype, a->stream_dtype, a->gate_dtype);
    if (!norm_kind(a->post_norm) || !norm_kind(a->pre_norm)) return fail(ADCDIFF_E_BADARG, "%s: norms %d, %d", who, a->post_norm, a->pre_norm);
    if (!(a->eps >= 0.0f)) return fail(ADCDIFF_E_BADARG, "%s: eps %g", who, (double)a->eps);
    if (a->M > 0 && !a->x) return fail(ADCDIFF_E_BADARG, "%s: null x", who);
    if (a->M > 0 && !a->h && (a->gate || a->post_norm || a->residual_scale != 1.0f))
        return fail(ADCDIFF_E_BADARG, "%s: a gate, a post norm or a residual scale without h", who);
    if ((!a->post_norm && (a->post_weight || a->post_bias)) || (!a->pre_norm && (a->pre_weight || a->pre_bias)))
        return fail(ADCDIFF_E_BADARG, "%s: a weight or bias without its norm", who);
    if (a->gate && (a->gate_rows < (a->M > 0) || (a->M > 0 && a->M % a->gate_rows != 0)))
        return fail(ADCDIFF_E_BADARG, "%s: %d gate rows do not divide %d rows", who, a->gate_rows, a->M);
    if ((a->h && a->ldh < a->D) || (a->x && a->ldx < a->D) || (a->gate && a->gate_rows > 1 && a->ldg != 0 && a->ldg < a->D))
        return fail(ADCDIFF_E_BADARG, "%s: a row pitch below %d columns", who, a->D);
    return ADCDIFF_OK;
}

ResNormParams forward_params(const adcdiff_residual_norm_args& a) {
    ResNormParams p{};
    p.h = a.h; p.x = a.x; p.gate = a.gate;
    p.post_w = a.post_weight; p.post_b = a.post_bias; p.pre_w = a.pre_weight; p.pre_b = a.pre_bias;
    p.xn = a.x_new; p.y = a.y; p.stats = a.stats;
    p.ldh = a.ldh; p.ldx = a.ldx; p.ldg = a.ldg; p.ldxn = a.ldx_new; p.ldy = a.ldy;
    p.M = a.M; p.D = a.D; p.post = a.h ? a.post_norm : 0; p.pre = a.pre_norm;
    p.gate_bf16 = a.gate_dtype == ADCDIFF_BF16;
    p.gate_share = a.gate && a.M > 0 ? a.M / a.gate_rows : 1;
    p.crossing = a.x_new == a.x && wave_crossing(a.D);
    p.scale = a.residual_scale; p.eps = a.eps; p.inv_d = 1.0f / (float)a.D;
    return p;
}

// Threads for a row of D columns, eight each: a power of two, and more sizes where both sides were measured (67 M elements, bfloat16; f / b: forward,
// backward).  768 instead of 1024 at D = 6000, f 148 -> 131 us, b 970 -> 230 us; 32 instead of 64 at D = 136, f 36.8 -> 21.6, b 75 -> 52; and in the
// backward pass 192, 320 and 384, where fewer idle threads hold registers (D = 2056: b 298 -> 266 us, D = 1032: 288 -> 283, in float32 335 -> 319), while
// the forward pass loses with them (D = 2056: 166 -> 176 us, D = 3000: 124 -> 139 us).
int team_width(int D, bool backward) {
    const int waves = (D + 511) / 512;
    if (D <= 128) return 16;
    if (D <= 256) return 32;
    if (backward && waves <= 6) return 64 * waves;
    return waves <= 1 ? 64 : waves <= 2 ? 128 : waves <= 4 ? 256 : waves <= 8 ? 512 : waves <= 12 ? 768 : 1024;
}

// Calls f(std::integral_constant<int, threads>) for the team of a row
template <RowShape SHAPE, bool BACKWARD, typename F>
void for_width(int tpr, F f) {
    if constexpr (SHAPE == kTiny) return f(std::integral_constant<int, 16>());
    if constexpr (BACKWARD) {
        switch (tpr) {
            case 192: return f(std::integral_constant<int, 192>());
            case 320: return f(std::integral_constant<int, 320>());
            case 384: return f(std::integral_constant<int, 384>());
        }
    }
    switch (tpr) {
        case 16: return f(std::integral_constant<int, 16>());
        case 32: return f(std::integral_constant<int, 32>());
        case 64: return f(std::integral_constant<int, 64>());
        case 128: return f(std::integral_constant<int, 128>());
        case 256: return f(std::integral_constant<int, 256>());
        case 512: return f(std::integral_constant<int, 512>());
        case 768: return f(std::integral_constant<int, 768>());
        default: return f(std::integral_constant<int, 1024>());
    }
}

template <typename T, typename R, RowShape SHAPE, int TPR>
void launch_forward(const ResNormParams& p, hipStream_t stream) {
    constexpr int threads = threads_for<TPR>(), teams = threads / TPR;
    const long long groups = ((long long)p.M + teams - 1) / teams;
    hipLaunchKernelGGL((residual_norm_kernel<T, R, SHAPE, TPR>), dim3((unsigned)std::min<long long>(groups, 2048)), dim3(threads), 0, stream, p);
}

template <typename T, typename R, RowShape SHAPE>
void forward_by_width(const ResNormParams& p, hipStream_t stream) {
    for_width<SHAPE, false>(team_width(p.D, false), [&](auto tpr) { launch_forward<T, R, SHAPE, decltype(tpr)::value>(p, stream); });
}

template <typename T, typename R>
void forward_by_shape(const ResNormParams& p, hipStream_t stream) {
    switch (row_shape(p.D)) {
        case kWhole: return forward_by_width<T, R, kWhole>(p, stream);
        case kMoved: return forward_by_width<T, R, kMoved>(p, stream);
        case kTiny: return forward_by_width<T, R, kTiny>(p, stream);
    }
}

void forward_by_type(const ResNormParams& p, int dtype, int stream_dtype, hipStream_t stream) {
    if (dtype == ADCDIFF_BF16) {
        if (stream_dtype == ADCDIFF_BF16) forward_by_shape<bf16_t, bf16_t>(p, stream);
        else forward_by_shape<bf16_t, float>(p, stream);
    } else {
        if (stream_dtype == ADCDIFF_BF16) forward_by_shape<float, bf16_t>(p, stream);
        else forward_by_shape<float, float>(p, stream);
    }
}

// How a backward pass cuts its rows.  A chunk lies inside one gate row's rows; a workgroup runs over several chunks.
struct Cut {
    int tpr, teams, workgroups, chunk_rows, chunks_per_gate, chunks, group_rows, vectors;
    bool gate_sum;      // the gate's gradient is a sum over rows
};

constexpr int kMaxGroups = 512;

Cut cut_rows(int M, int D, int gate_rows, bool gate_grad, int vectors) {
    Cut c{};
    c.tpr = team_width(D, true);
    c.teams = c.tpr >= kThreads ? 1 : kThreads / c.tpr;
    c.vectors = vectors;
    c.gate_sum = gate_grad && gate_rows > 0 && M / std::max(gate_rows, 1) != 1;
    const int groups = c.gate_sum ? gate_rows : 1;
    c.group_rows = M / groups;
    if (M == 0) { c.chunks_per_gate = 1; c.chunk_rows = 1; return c; }
    // Two workgroups of 256 threads fit a CU (230 registers per thread): 512 workgroups' worth of teams, and chunks of at least two rows.  More
    // workgroups write and add more partial rows (1024: column sums of 32768 x 2048 17 us), longer chunks leave few rows waiting on each
    // other (8 rows: 1003 x 777 24 us).
    const int workers = kMaxGroups * c.teams;
    const int want = std::max(1, (workers + groups - 1) / groups);
    c.chunk_rows = std::max(std::min(c.group_rows, 2), (c.group_rows + want - 1) / want);
    c.chunks_per_gate = (c.group_rows + c.chunk_rows - 1) / c.chunk_rows;
    c.chunks = groups * c.chunks_per_gate;
    c.workgroups = std::min(kMaxGroups, (c.chunks + c.teams - 1) / c.teams);
    return c;
}

size_t workspace_floats(const Cut& c, int D) {
    size_t n = (size_t)c.workgroups * c.vectors * D;
    if (c.gate_sum && c.chunks_per_gate > 1) n += (size_t)c.chunks * D;
    return n;
}

template <typename T, typename R, RowShape SHAPE>
int backward_by_width(const ResNormGradParams& q, const Cut& c, hipStream_t stream) {
    int rc = ADCDIFF_OK;
    for_width<SHAPE, true>(c.tpr, [&](auto tpr) {
        constexpr int TPR = decltype(tpr)::value;
        const auto kernel = &residual_norm_grad_kernel<T, R, SHAPE, TPR>;
        constexpr int lds = TPR == 1024 ? kWideSums : 0;
        if constexpr (lds > 0) {
            static std::atomic<bool> done[64];
            rc = allow_lds("residual_norm_backward", reinterpret_cast<const void*>(kernel), lds, done);
            if (rc != ADCDIFF_OK) return;
        }
        hipLaunchKernelGGL(kernel, dim3(c.workgroups), dim3(threads_for<TPR>()), lds, stream, q);
    });
    return rc;
}

template <typename T, typename R>
int backward_by_shape(const ResNormGradParams& q, const Cut& c, hipStream_t stream) {
    switch (row_shape(q.f.D)) {
        case kWhole: return backward_by_width<T, R, kWhole>(q, c, stream);
        case kMoved: return backward_by_width<T, R, kMoved>(q, c, stream);
        default: return backward_by_width<T, R, kTiny>(q, c, stream);
    }
}

int backward_by_type(const ResNormGradParams& q, const Cut& c, int dtype, int stream_dtype, hipStream_t stream) {
    if (dtype == ADCDIFF_BF16) {
        if (stream_dtype == ADCDIFF_BF16) return backward_by_shape<bf16_t, bf16_t>(q, c, stream);
        return backward_by_shape<bf16_t, float>(q, c, stream);
    } else {
        if (stream_dtype == ADCDIFF_BF16) return backward_by_shape<float, bf16_t>(q, c, stream);
        return backward_by_shape<float, float>(q, c, stream);
    }
}

int vector_count(const adcdiff_residual_norm_grads& g) { return !!g.post_weight + !!g.post_bias + !!g.pre_weight + !!g.pre_bias; }

}  // namespace
}  // namespace adcdiff

extern "C" int adcdiff_residual_norm(const adcdiff_residual_norm_args* a, adcdiff_stream_t stream_) {
    using namespace adcdiff;
    int rc = check_args("residual_norm", a);
    if (rc != ADCDIFF_OK) return rc;
    if (a->M == 0) return ADCDIFF_OK;
    if ((a->pre_norm != 0) != (a->y != nullptr)) return fail(ADCDIFF_E_BADARG, "residual_norm: y goes with a pre norm and only with one");
    if (!a->y && !a->x_new) return fail(ADCDIFF_E_BADARG, "residual_norm: no output");
    if ((a->x_new && a->ldx_new < a->D) || (a->y && a->ldy < a->D)) return fail(ADCDIFF_E_BADARG, "residual_norm: a row pitch below %d columns", a->D);
    if (a->stats && !aligned16(a->stats)) return fail(ADCDIFF_E_BADARG, "residual_norm: stats are not on a 16-byte boundary");
    hipStream_t stream = as_stream(stream_);
    const ResNormParams p = forward_params(*a);
    const int st = type_size(a->dtype), sr = type_size(a->stream_dtype);
    TimingScope timing(ADCDIFF_KIND_OTHER, a->M, a->D, 0, 0.0, (double)a->M * a->D * ((a->h ? st : 0) + (a->y ? st : 0) + sr + (a->x_new ? sr : 0)), stream);
    forward_by_type(p, a->dtype, a->stream_dtype, stream);
    return check_launch("residual_norm");
}

extern "C" size_t adcdiff_residual_norm_backward_workspace_bytes(const adcdiff_residual_norm_args* a, const adcdiff_residual_norm_grads* g) {
    using namespace adcdiff;
    if (check_args("residual_norm_backward", a) != ADCDIFF_OK || !g) return 0;
    return std::max<size_t>(16, workspace_floats(cut_rows(a->M, a->D, a->gate ? a->gate_rows : 0, g->gate != nullptr, vector_count(*g)), a->D) * 4);
}

extern "C" int adcdiff_residual_norm_backward(const adcdiff_residual_norm_args* a, const adcdiff_residual_norm_grads* g, void* workspace,
                                              size_t workspace_bytes, adcdiff_stream_t stream_) {
    using namespace adcdiff;
    int rc = check_args("residual_norm_backward", a);
    if (rc != ADCDIFF_OK) return rc;
    if (!g) return fail(ADCDIFF_E_BADARG, "residual_norm_backward: null gradients");
    if (a->M > 0 && !g->d_x_new && !g->d_y) return fail(ADCDIFF_E_BADARG, "residual_norm_backward: no incoming gradient");
    if (g->d_y && !a->pre_norm) return fail(ADCDIFF_E_BADARG, "residual_norm_backward: d_y without a pre norm");
    if (a->M > 0 && (a->post_norm || a->pre_norm) && (!a->stats || !aligned16(a->stats)))
        return fail(ADCDIFF_E_BADARG, "residual_norm_backward: the statistics of the forward pass are missing or not on a 16-byte boundary");
    const bool has_h = a->h || a->M == 0;   // the address of no rows may be null
    if ((g->h && !has_h) || (g->gate && !a->gate) || ((g->post_weight || g->post_bias) && !(has_h && a->post_norm)) || ((g->pre_weight || g->pre_bias) && !a->pre_norm))
        return fail(ADCDIFF_E_BADARG, "residual_norm_backward: a gradient of what the forward pass did not have");
    if ((g->d_x_new && g->ld_d_x_new < a->D) || (g->d_y && g->ld_d_y < a->D) || (g->h && g->ld_h < a->D) || (g->x && g->ld_x < a->D) ||
        (g->gate && a->gate_rows > 1 && g->ld_gate < a->D))
        return fail(ADCDIFF_E_BADARG, "residual_norm_backward: a row pitch below %d columns", a->D);
    const Cut c = cut_rows(a->M, a->D, a->gate ? a->gate_rows : 0, g->gate != nullptr, vector_count(*g));
    const size_t need = std::max<size_t>(16, workspace_floats(c, a->D) * 4);
    if (!workspace || !aligned16(workspace) || workspace_bytes < need)
        return fail(ADCDIFF_E_WORKSPACE, "residual_norm_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    hipStream_t stream = as_stream(stream_);
    const int st = type_size(a->dtype), sr = type_size(a->stream_dtype);
    ResNormGradParams q{};
    q.f = forward_params(*a);
    q.d_xn = g->d_x_new; q.d_y = g->d_y; q.d_h = g->h; q.d_x = g->x; q.d_gate = g->gate;
    q.ld_dxn = g->ld_d_x_new; q.ld_dy = g->ld_d_y; q.ld_dh = g->ld_h; q.ld_dx = g->ld_x; q.ld_dg = g->ld_gate;
    q.chunks = c.chunks; q.chunk_rows = c.chunk_rows; q.chunks_per_gate = c.chunks_per_gate; q.group_rows = c.group_rows;
    q.vectors = c.vectors;
    q.partial = static_cast<float*>(workspace);
    q.gate_partial = q.partial + (size_t)c.workgroups * c.vectors * a->D;
    ColumnSumParams s{};
    int slot = 0;
    auto place = [&](float* out) { if (!out) return -1; s.out[slot] = out; return slot++; };
    q.slot_pre_w = place(g->pre_weight); q.slot_pre_b = place(g->pre_bias); q.slot_post_w = place(g->post_weight); q.slot_post_b = place(g->post_bias);
    if (a->M > 0) {
        TimingScope timing(ADCDIFF_KIND_OTHER, a->M, a->D, 0, 0.0, (double)a->M * a->D * ((a->h ? 2.0 : 0.0) * st + (g->d_y ? st : 0) + 2.0 * sr + (g->d_x_new ? sr : 0)), stream);
        rc = backward_by_type(q, c, a->dtype, a->stream_dtype, stream);
        if (rc != ADCDIFF_OK) return rc;
        rc = check_launch("residual_norm_backward");
        if (rc != ADCDIFF_OK) return rc;
    }
    const int gate_segments = g->gate && (a->M == 0 || (c.gate_sum && c.chunks_per_gate > 1)) ? a->gate_rows : 0;
    const int segments = c.vectors + gate_segments;
    s.partial = q.partial; s.gate_partial = q.gate_partial; s.d_gate = g->gate; s.ld_dg = g->ld_gate;
    s.D = a->D; s.vectors = c.vectors; s.workgroups = a->M > 0 ? c.workgroups : 0;
    s.chunks_per_gate = a->M > 0 ? c.chunks_per_gate : 0; s.gate_bf16 = a->gate_dtype == ADCDIFF_BF16;
    if (segments == 0) return ADCDIFF_OK;
    TimingScope timing(ADCDIFF_KIND_OTHER, segments, a->D, 0, 0.0, 4.0 * workspace_floats(c, a->D), stream);
    const bool flat = s.chunks_per_gate <= 32;
    s.tall = c.vectors + (flat ? 0 : gate_segments);
    s.flat = flat ? (long long)gate_segments * a->D : 0;
    const long long blocks = (long long)((a->D + 31) / 32) * s.tall + std::min<long long>((s.flat + 1023) / 1024, 4096);
    hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)blocks), dim3(1024), 0, stream, s);
    return check_launch("residual_norm_backward: column sums");
}

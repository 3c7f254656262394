// The global norm over many gradient tensors, and clipping by it.  Both are bound by memory: the norm reads every element once, the
// clipping reads it once more and writes it.  The tensors' addresses and lengths travel as kernel arguments (kTable per launch), so a
// call keeps nothing between calls, copies nothing to the device and can be captured into a graph.
#include <algorithm>
#include <cmath>
#include <exception>
#include <vector>

#include "row_access.h"

namespace adcdiff {
namespace {

constexpr int kTable = 120;          // tensors per launch: 120 * 32 bytes of kernel arguments
constexpr long long kChunk = 8192;   // elements of one workgroup: 44 M gradients 42 us (4096: 48, 16384: 44, 65536: 46; 4.2 TB/s, read only)
constexpr long long kPiece = 2048;   // elements of one wave where a single workgroup does the whole call
constexpr int kFewPieces = 64;       // up to here: four rounds of loads for its 16 waves, against three launches

struct GradEntry {
    const void* grad;
    void* out;
    long long numel;
    int first_chunk;                 // among the launch's chunks (or pieces)
    int types;                       // bit 0: grad is bf16, bit 1: out is bf16
};

struct GradTable {
    GradEntry t[kTable];
    int n;
};

// the tensor that a chunk of the launch belongs to
__device__ __forceinline__ int find_entry(const GradTable& g, int chunk) {
    int lo = 0, hi = g.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (g.t[mid].first_chunk <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Gradients are aligned to their element only (views into an arena); the memory system takes 16-byte accesses at any address.

// float64: any float32 gradient squares exactly, without overflow or underflow; the sum takes one rounding of 2^-53 for each addition on an element's
// path (32 in a thread, 6 + 4 in the workgroup, and as many again over the chunks), far below the 2^-24 of the result's own
struct SumSquares {
    typedef double Acc;
    static __device__ __forceinline__ double zero() { return 0.0; }
    static __device__ __forceinline__ void add(double& s, float v) { s = fma((double)v, (double)v, s); }
    static __device__ __forceinline__ double join(double a, double b) { return a + b; }
};
struct MaxAbs {       // compared as bit patterns: those of NaN lie above infinity's, so a NaN stays
    typedef uint32_t Acc;
    static __device__ __forceinline__ uint32_t zero() { return 0u; }
    static __device__ __forceinline__ void add(uint32_t& s, float v) { s = max(s, __builtin_bit_cast(uint32_t, v) & 0x7fffffffu); }
    static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) { return max(a, b); }
};

template <typename Op, int THREADS>
__device__ __forceinline__ typename Op::Acc block_join(typename Op::Acc s, typename Op::Acc* red) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) s = Op::join(s, __shfl_xor(s, m));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = red[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) s = Op::join(s, red[w]);
    return s;
}

// A thread's share of a chunk: eight 16-byte loads in flight, then what is left
template <typename Op, int THREADS, typename In>
__device__ __forceinline__ typename Op::Acc reduce_chunk(const In* __restrict__ p, int cnt, int tid) {
    constexpr int W = 16 / sizeof(In), U = 8;
    typename Op::Acc s = Op::zero();
    auto add = [&](const u32x4 w) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t bits = w[k];      // (a bit cast of a vector's element itself reads element 0)
            if constexpr (sizeof(In) == 2) {
                Op::add(s, bf_lo(bits));
                Op::add(s, bf_hi(bits));
            } else {
                Op::add(s, __builtin_bit_cast(float, bits));
            }
        }
    };
    int i = tid * W;
    for (; i + (U - 1) * THREADS * W + W <= cnt; i += U * THREADS * W) {
        u32x4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = *reinterpret_cast<const u32x4_any*>(p + i + u * THREADS * W);
#pragma unroll
        for (int u = 0; u < U; ++u) add(w[u]);
    }
    for (; i + W <= cnt; i += THREADS * W) add(*reinterpret_cast<const u32x4_any*>(p + i));
    for (i = cnt / W * W + tid; i < cnt; i += THREADS) {
        if constexpr (sizeof(In) == 2) Op::add(s, bf_lo(p[i]));
        else Op::add(s, p[i]);
    }
    return s;
}

template <typename Op, int THREADS>
__device__ __forceinline__ typename Op::Acc reduce_part(const GradEntry& d, long long base, int cnt, int tid) {
    if (d.types & 1) return reduce_chunk<Op, THREADS>(static_cast<const uint16_t*>(d.grad) + base, cnt, tid);
    return reduce_chunk<Op, THREADS>(static_cast<const float*>(d.grad) + base, cnt, tid);
}

template <typename Op>
__global__ __launch_bounds__(256) void grad_partial_kernel(const GradTable g, typename Op::Acc* __restrict__ partial) {
    __shared__ typename Op::Acc red[4];
    const int tid = threadIdx.x;
    const GradEntry& d = g.t[find_entry(g, blockIdx.x)];
    const long long base = (long long)((int)blockIdx.x - d.first_chunk) * kChunk;
    const int cnt = (int)min(kChunk, d.numel - base);
    typename Op::Acc s = reduce_part<Op, 256>(d, base, cnt, tid);
    s = block_join<Op, 256>(s, red);
    if (tid == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ float as_norm(double s) { return (float)sqrt(s); }
__device__ __forceinline__ float as_norm(uint32_t s) { return __builtin_bit_cast(float, s); }

// min(1, max_norm / (norm + 1e-6)); NaN for a NaN norm
__device__ __forceinline__ float clip_factor(float max_norm, float norm) {
    const float f = max_norm / (norm + 1e-6f);
    return f >= 1.0f ? 1.0f : f;
}

template <typename Op>
__global__ __launch_bounds__(1024) void grad_total_kernel(const typename Op::Acc* __restrict__ partial, int n, float max_norm, float* __restrict__ norm,
                                                          float* __restrict__ factor) {
    __shared__ typename Op::Acc red[16];
    typename Op::Acc s = Op::zero();
    for (int i = threadIdx.x; i < n; i += 1024) s = Op::join(s, partial[i]);
    s = block_join<Op, 1024>(s, red);
    if (threadIdx.x == 0) {
        const float v = as_norm(s);
        *norm = v;
        if (factor) *factor = clip_factor(max_norm, v);
    }
}

// In place p and o are the same memory, so four vectors are loaded before the first is stored: a thread's loads are then in flight
// together without the compiler having to prove that a store leaves the next load alone.
template <int THREADS, typename In, typename Out>
__device__ __forceinline__ void scale_chunk(const In* p, Out* o, int cnt, float f, int tid) {
    constexpr int W = sizeof(In) == 2 ? 8 : 4, U = 4;
    const int whole = cnt / W * W;
    for (int i0 = tid * W; i0 < whole; i0 += THREADS * W * U) {
        float v[U][W];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * THREADS * W;
            if (i < whole) {
                if constexpr (sizeof(In) == 2) {
                    const u32x4 w = *reinterpret_cast<const u32x4_any*>(p + i);
#pragma unroll
                    for (int k = 0; k < 4; ++k) { v[u][2 * k] = bf_lo(w[k]); v[u][2 * k + 1] = bf_hi(w[k]); }
                } else {
                    const f32x4 w = *reinterpret_cast<const f32x4_any*>(p + i);
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[u][k] = w[k];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * THREADS * W;
            if (i < whole) {
                if constexpr (sizeof(Out) == 4) {
#pragma unroll
                    for (int h = 0; h < W / 4; ++h)
                        *reinterpret_cast<f32x4_any*>(o + i + 4 * h) = f32x4{v[u][4 * h] * f, v[u][4 * h + 1] * f, v[u][4 * h + 2] * f, v[u][4 * h + 3] * f};
                } else {
                    typedef __bf16 bf16xw __attribute__((ext_vector_type(W)));
                    typedef bf16xw bf16xw_any __attribute__((aligned(2)));
                    bf16xw q;
#pragma unroll
                    for (int k = 0; k < W; ++k) q[k] = (bf16_t)(v[u][k] * f);
                    *reinterpret_cast<bf16xw_any*>(o + i) = q;
                }
            }
        }
    }
    for (int i = whole + tid; i < cnt; i += THREADS) o[i] = (Out)((float)p[i] * f);
}

template <int THREADS>
__device__ __forceinline__ void scale_part(const GradEntry& d, long long base, int cnt, float f, int tid) {
    const bf16_t* pb = static_cast<const bf16_t*>(d.grad) + base;
    const float* pf = static_cast<const float*>(d.grad) + base;
    bf16_t* ob = static_cast<bf16_t*>(d.out) + base;
    float* of = static_cast<float*>(d.out) + base;
    switch (d.types) {
        case 0: scale_chunk<THREADS>(pf, of, cnt, f, tid); break;
        case 1: scale_chunk<THREADS>(pb, of, cnt, f, tid); break;
        case 2: scale_chunk<THREADS>(pf, ob, cnt, f, tid); break;
        default: scale_chunk<THREADS>(pb, ob, cnt, f, tid); break;
    }
}

__global__ __launch_bounds__(256) void grad_scale_kernel(const GradTable g, const float* __restrict__ factor) {
    const GradEntry& d = g.t[find_entry(g, blockIdx.x)];
    const float f = *factor;
    if (f == 1.0f && d.out == d.grad) return;   // in place: g * 1 is what is there
    const long long base = (long long)((int)blockIdx.x - d.first_chunk) * kChunk;
    const int cnt = (int)min(kChunk, d.numel - base);
    scale_part<256>(d, base, cnt, f, threadIdx.x);
}

// 44 M float32 gradients into another buffer: 57 us (355 MB at 6.2 TB/s, part of the gradients still in the last-level cache after the norm).
// The whole call in one workgroup, where the gradients are few (five tensors of 12 k elements in all 2.9 us): a wave takes pieces of kPiece elements, for the norm and again for the scaling.
template <typename Op>
__global__ __launch_bounds__(1024) void grad_small_kernel(const GradTable g, int pieces, float max_norm, float* __restrict__ norm, int clip) {
    __shared__ typename Op::Acc red[16];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    typename Op::Acc s = Op::zero();
    for (int i = wave; i < pieces; i += 16) {
        const GradEntry& d = g.t[find_entry(g, i)];
        const long long base = (long long)(i - d.first_chunk) * kPiece;
        s = Op::join(s, reduce_part<Op, 64>(d, base, (int)min(kPiece, d.numel - base), lane));
    }
    const float v = as_norm(block_join<Op, 1024>(s, red));
    if (threadIdx.x == 0) *norm = v;
    const float f = clip_factor(max_norm, v);
    if (!clip) return;
    for (int i = wave; i < pieces; i += 16) {
        const GradEntry& d = g.t[find_entry(g, i)];
        if (f == 1.0f && d.out == d.grad) continue;
        const long long base = (long long)(i - d.first_chunk) * kPiece;
        scale_part<64>(d, base, (int)min(kPiece, d.numel - base), f, lane);
    }
}

long long parts_of(long long numel, long long part) { return (numel + part - 1) / part; }
long long chunks_of(long long numel) { return parts_of(numel, kChunk); }

int check_tensors(const char* who, const adcdiff_grad_tensor* ts, int n, bool clip, long long* chunks) {
    if (n < 0 || (n > 0 && !ts)) return fail(ADCDIFF_E_BADARG, "%s: null table or %d tensors", who, n);
    *chunks = 0;
    for (int i = 0; i < n; ++i) {
        const adcdiff_grad_tensor& t = ts[i];
        if (t.numel < 0 || !type_ok(t.dtype) || (clip && !type_ok(t.out_dtype)) || (t.numel > 0 && (!t.grad || (clip && !t.out))))
            return fail(ADCDIFF_E_BADARG, "%s: tensor %d: %lld elements, types %d -> %d, null pointer or not", who, i, t.numel, t.dtype, t.out_dtype);
        if ((reinterpret_cast<uintptr_t>(t.grad) % type_size(t.dtype)) || (clip && reinterpret_cast<uintptr_t>(t.out) % type_size(t.out_dtype)))
            return fail(ADCDIFF_E_BADARG, "%s: tensor %d is not aligned to its elements", who, i);
        *chunks += chunks_of(t.numel);
    }
    if (*chunks > 0xffffffLL) return fail(ADCDIFF_E_BADARG, "%s: too many elements", who);
    return ADCDIFF_OK;
}

// What is written must not be read or written by another tensor's workgroups: they run in any order.
int check_overlap(const adcdiff_grad_tensor* ts, int n) {
    struct Span { uintptr_t lo, hi; int i; bool write; };
    std::vector<Span> spans;
    spans.reserve(2 * (size_t)n);
    for (int i = 0; i < n; ++i) {
        const adcdiff_grad_tensor& t = ts[i];
        if (t.numel == 0) continue;
        const uintptr_t g = reinterpret_cast<uintptr_t>(t.grad), o = reinterpret_cast<uintptr_t>(t.out);
        spans.push_back(Span{o, o + (uintptr_t)t.numel * type_size(t.out_dtype), i, true});
        if (g != o || t.dtype != t.out_dtype) spans.push_back(Span{g, g + (uintptr_t)t.numel * type_size(t.dtype), i, false});
    }
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
    uintptr_t any_hi = 0, write_hi = 0;
    int any_i = -1, write_i = -1;
    for (const Span& s : spans) {
        if (s.write && s.lo < any_hi) return fail(ADCDIFF_E_BADARG, "clip_grad_norm: the output of tensor %d overlaps tensor %d", s.i, any_i);
        if (s.lo < write_hi) return fail(ADCDIFF_E_BADARG, "clip_grad_norm: tensor %d overlaps the output of tensor %d", s.i, write_i);
        if (s.hi > any_hi) { any_hi = s.hi; any_i = s.i; }
        if (s.write && s.hi > write_hi) { write_hi = s.hi; write_i = s.i; }
    }
    return ADCDIFF_OK;
}

// Calls launch(table, chunks of the table, chunks before it) for the tensors in groups of kTable
template <typename F>
void for_tables(const adcdiff_grad_tensor* ts, int n, long long part, F launch) {
    GradTable table;
    table.n = 0;
    int chunks = 0, before = 0;
    for (int i = 0; i < n; ++i) {
        if (ts[i].numel > 0) {
            GradEntry& e = table.t[table.n++];
            e.grad = ts[i].grad; e.out = ts[i].out; e.numel = ts[i].numel; e.first_chunk = chunks;
            e.types = (ts[i].dtype == ADCDIFF_BF16 ? 1 : 0) | (ts[i].out && ts[i].out_dtype == ADCDIFF_BF16 ? 2 : 0);
            chunks += (int)parts_of(ts[i].numel, part);
        }
        if (table.n == kTable || (i == n - 1 && table.n > 0)) {
            launch(table, chunks, before);
            before += chunks;
            chunks = 0;
            table.n = 0;
        }
    }
}

constexpr size_t kHead = 64;   // bytes in front of the partial results: the clipping factor

template <typename Op>
int norm_launches(const char* who, const adcdiff_grad_tensor* ts, int n, long long chunks, float max_norm, float* norm, float* factor, void* partial_, hipStream_t stream) {
    typename Op::Acc* partial = static_cast<typename Op::Acc*>(partial_);
    for_tables(ts, n, kChunk, [&](const GradTable& t, int count, int before) {
        TimingScope timing(ADCDIFF_KIND_OTHER, count, (int)kChunk, 0, 0.0, 4.0 * count * kChunk, stream);
        hipLaunchKernelGGL(grad_partial_kernel<Op>, dim3(count), dim3(256), 0, stream, t, partial + before);
    });
    TimingScope timing(ADCDIFF_KIND_OTHER, 1, (int)chunks, 0, 0.0, 8.0 * chunks, stream);
    hipLaunchKernelGGL(grad_total_kernel<Op>, dim3(1), dim3(1024), 0, stream, partial, (int)chunks, max_norm, norm, factor);
    return check_launch(who);
}

int run(const char* who, const adcdiff_grad_tensor* ts, int n, int norm_type, bool clip, double max_norm, float* norm, void* workspace, size_t workspace_bytes,
        adcdiff_stream_t stream_) {
    long long chunks;
    int rc = check_tensors(who, ts, n, clip, &chunks);
    if (rc != ADCDIFF_OK) return rc;
    if (norm_type != 0 && norm_type != 2) return fail(ADCDIFF_E_BADARG, "%s: norm type %d is not 2 or 0 (maximum)", who, norm_type);
    if (!norm) return fail(ADCDIFF_E_BADARG, "%s: null norm", who);
    if (clip && !(max_norm >= 0.0)) return fail(ADCDIFF_E_BADARG, "%s: max_norm %g", who, max_norm);
    if (clip) {
        try {   // the list of address ranges is host memory
            rc = check_overlap(ts, n);
        } catch (const std::exception&) {
            rc = fail(ADCDIFF_E_WORKSPACE, "%s: out of host memory", who);
        }
        if (rc != ADCDIFF_OK) return rc;
    }
    const size_t need = adcdiff_grad_norm_workspace_bytes(ts, n);
    if (!workspace || !aligned16(workspace) || workspace_bytes < need)
        return fail(ADCDIFF_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
    hipStream_t stream = as_stream(stream_);
    float* factor = clip ? static_cast<float*>(workspace) : nullptr;
    void* partial = static_cast<char*>(workspace) + kHead;
    long long pieces = 0;
    for (int i = 0; i < n && pieces <= kFewPieces; ++i) pieces += parts_of(ts[i].numel, kPiece);
    if (n <= kTable && pieces > 0 && pieces <= kFewPieces) {
        for_tables(ts, n, kPiece, [&](const GradTable& t, int count, int) {   // one table
            TimingScope timing(ADCDIFF_KIND_OTHER, count, (int)kPiece, 0, 0.0, (clip ? 12.0 : 4.0) * count * kPiece, stream);
            if (norm_type == 2) hipLaunchKernelGGL(grad_small_kernel<SumSquares>, dim3(1), dim3(1024), 0, stream, t, count, (float)max_norm, norm, (int)clip);
            else hipLaunchKernelGGL(grad_small_kernel<MaxAbs>, dim3(1), dim3(1024), 0, stream, t, count, (float)max_norm, norm, (int)clip);
        });
        return check_launch(who);
    }
    rc = norm_type == 2 ? norm_launches<SumSquares>(who, ts, n, chunks, (float)max_norm, norm, factor, partial, stream)
                        : norm_launches<MaxAbs>(who, ts, n, chunks, (float)max_norm, norm, factor, partial, stream);
    if (rc != ADCDIFF_OK || !clip) return rc;
    for_tables(ts, n, kChunk, [&](const GradTable& t, int count, int) {
        TimingScope timing(ADCDIFF_KIND_OTHER, count, (int)kChunk, 0, 0.0, 8.0 * count * kChunk, stream);
        hipLaunchKernelGGL(grad_scale_kernel, dim3(count), dim3(256), 0, stream, t, factor);
    });
    return check_launch(who);
}

}  // namespace
}  // namespace adcdiff

extern "C" size_t adcdiff_grad_norm_workspace_bytes(const adcdiff_grad_tensor* tensors, int n_tensors) {
    using namespace adcdiff;
    long long chunks;
    if (check_tensors("grad_norm", tensors, n_tensors, false, &chunks) != ADCDIFF_OK) return 0;
    return kHead + (size_t)chunks * sizeof(double);
}

extern "C" int adcdiff_grad_norm(const adcdiff_grad_tensor* tensors, int n_tensors, int norm_type, float* norm, void* workspace,
                                 size_t workspace_bytes, adcdiff_stream_t stream) {
    return adcdiff::run("grad_norm", tensors, n_tensors, norm_type, false, 0.0, norm, workspace, workspace_bytes, stream);
}

extern "C" int adcdiff_clip_grad_norm(const adcdiff_grad_tensor* tensors, int n_tensors, int norm_type, double max_norm, float* norm, void* workspace,
                                      size_t workspace_bytes, adcdiff_stream_t stream) {
    return adcdiff::run("clip_grad_norm", tensors, n_tensors, norm_type, true, max_norm, norm, workspace, workspace_bytes, stream);
}

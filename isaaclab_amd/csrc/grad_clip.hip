// The norm of many gradients taken as one vector, and clipping to it.
//
//   norm = (sum |g|^q)^(1/q) over every element of every tensor (q = 1, 2; or the maximum);  out = g min(1, max_norm / (norm + 1e-6))
//
// Sums are held in 64 bits (the square of a float is exact there, so neither large nor small gradients leave the range) and
// taken in an order that depends on the sizes and element types alone, not on where a tensor starts.
//
// Bound by memory: 160 M elements, half float32 and half bfloat16, into float32: 133 us for the 480 MB that the norm reads and 197 us
// for the 1120 MB that the scaling reads and writes (part of them still cached), 329 us where three passes at the copy rate,
// 4.7 TB/s, are 341; 50 M bfloat16 elements at an odd offset into float32 175.  An actor-critic of 0.57 M elements: 4.4 + 3.9 us, what
// two small launches take.  2048 partial sums instead of 1024 gain 2 % there and cost every block of the second launch a second
// kilobyte-long read; stores past the caches lose 7 %.
#include "mdp_device.hpp"
#include "mdp_host.hpp"
#include "elements_device.hpp"
#include <algorithm>
#include <memory>
#include <new>

using namespace mdp;

namespace {

constexpr int kTable = 96;             // tensors of a launch: the table travels in the kernel arguments (4 KB at most)
constexpr int kChunk = 4096;           // elements that a block takes at a time
constexpr int kBlocks = 1024;          // partial sums of a launch
constexpr int64_t kMost = (int64_t)1 << 40;   // elements of a call: its chunks are counted in 32 bits

struct Table {
    int n;
    int chunks;                        // of all tensors
    int start[kTable + 1];             // first chunk of each tensor
    const void* grad[kTable];
    void* out[kTable];
    int64_t count[kTable];
    uint8_t dtype[kTable], out_dtype[kTable];
};
static_assert(sizeof(Table) <= 3600, "the table has to fit the kernel arguments");

template <int KIND>
MDP_DEV double joined(double a, double b) {
    if (KIND) return a + b;
    return b > a || b != b ? b : a;    // a NaN stays
}

template <int KIND>
MDP_DEV double block_join(double v, double* red) {
    for (int o = 32; o > 0; o >>= 1) v = joined<KIND>(v, __shfl_xor(v, o));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (unsigned w = 1; w < blockDim.x / 64; ++w) v = joined<KIND>(v, red[w]);
    return v;
}

// calls f(tensor, first element, elements) for each of this block's chunks: block b of B takes chunks [b C / B, (b + 1) C / B),
// backwards from the last block on if BACK
template <bool BACK = false, class F>
MDP_DEV void for_chunks(const Table& t, F&& f) {
    const int64_t b = BACK ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    const int first = (int)(b * t.chunks / gridDim.x), end = (int)((b + 1) * t.chunks / gridDim.x);
    if (first == end) return;
    int i = 0;                                         // the tensor of the first chunk: the last that starts at or before it
    const int c0 = BACK ? end - 1 : first;
    for (int step = 64; step; step >>= 1)
        if (i + step < t.n && t.start[i + step] <= c0) i += step;
    for (int k = 0; k < end - first; ++k) {
        const int c = BACK ? end - 1 - k : first + k;
        while (BACK ? t.start[i] > c : t.start[i + 1] <= c) i += BACK ? -1 : 1;
        const int64_t at = (int64_t)(c - t.start[i]) * kChunk, left = t.count[i] - at;
        f(i, at, (int)(left < kChunk ? left : kChunk));
    }
}

// f(value) for each of this thread's elements of a chunk.  A full one by 16-byte loads, all of them in flight, wherever the tensor
// starts (elements are aligned to themselves): which thread sums up which elements does not depend on the address.
template <typename T, class F>
MDP_DEV void each(const T* g, int n, F&& f) {
    constexpr int N = Chunk<T>::N, B = kChunk / (256 * N);
    struct __attribute__((packed, aligned(sizeof(T)))) Anywhere { uint32_t w[4]; };
    if (n == kChunk) {
        Chunk<T> c[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const Anywhere q = ((const Anywhere*)g)[b * 256 + threadIdx.x];
            c[b].raw = uint4{q.w[0], q.w[1], q.w[2], q.w[3]};
        }
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int e = 0; e < N; ++e) f(c[b].at(e));
    } else {
        for (int i = threadIdx.x; i < n; i += 256) f(to_f32(g[i]));
    }
}

template <int KIND, typename T>
MDP_DEV double chunk_norm(const void* grad, int64_t at, int n, double acc) {
    each((const T*)grad + at, n, [&](float x) {
        const double v = (double)x;
        acc = KIND == 2 ? fma(v, v, acc) : joined<KIND>(acc, fabs(v));
    });
    return acc;
}

template <int KIND>
__global__ __launch_bounds__(256) void k_grad_partial(Table t, double* __restrict__ partial) {
    __shared__ double red[4];
    double acc = 0.0;
    for_chunks(t, [&](int i, int64_t at, int n) {
        if (t.dtype[i] == MDP_DTYPE_F32) acc = chunk_norm<KIND, float>(t.grad[i], at, n, acc);
        else if (t.dtype[i] == MDP_DTYPE_BF16) acc = chunk_norm<KIND, bf16>(t.grad[i], at, n, acc);
        else acc = chunk_norm<KIND, f16>(t.grad[i], at, n, acc);
    });
    acc = block_join<KIND>(acc, red);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// every thread of a block gets what the partial sums join to
template <int KIND>
MDP_DEV double joined_partials(const double* __restrict__ partial, int n, double* red) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) acc = joined<KIND>(acc, partial[i]);
    return block_join<KIND>(acc, red);
}

// the norm of the partial sums, and what they join to in their place: for a call that only wants the norm, or has so many
// tensors that the partial sums are more than every block should read
template <int KIND>
__global__ __launch_bounds__(256) void k_grad_finish(const double* __restrict__ partial, int n, double* __restrict__ all,
                                                     float* __restrict__ norm) {
    __shared__ double red[4];
    const double acc = joined_partials<KIND>(partial, n, red);
    if (threadIdx.x) return;
    *all = acc;
    *norm = (float)(KIND == 2 ? sqrt(acc) : acc);
}

template <typename T, typename U>
MDP_DEV void chunk_scale(const void* grad, void* to, int64_t at, int n, float f) {
    constexpr int N = Chunk<T>::N, B = kChunk / (256 * N), M = Chunk<U>::N;
    const T* g = (const T*)grad + at;
    U* out = (U*)to + at;
    if (n == kChunk && (((uintptr_t)g | (uintptr_t)out) & 15) == 0) {
        Chunk<T> c[B];
#pragma unroll
        for (int b = 0; b < B; ++b) c[b].raw = ((const uint4*)g)[b * 256 + threadIdx.x];
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int h = 0; h < N / M; ++h) {
                float v[M];
#pragma unroll
                for (int e = 0; e < M; ++e) v[e] = c[b].at(h * M + e) * f;
                ((uint4*)out)[(b * 256 + threadIdx.x) * (N / M) + h] = Chunk<U>::of(v).raw;
            }
    } else {
        for (int i = threadIdx.x; i < n; i += 256) from_f32(to_f32(g[i]) * f, out[i]);
    }
}

// Every block joins the partial sums by itself (at most 1024 of them, from the caches): no launch between the two.  Chunks are
// taken from the last one back, so that what the norm read last, and is still in the caches, comes first.
template <int KIND>
__global__ __launch_bounds__(256) void k_grad_scale(Table t, const double* __restrict__ partial, int partials, double max_norm,
                                                    float* __restrict__ norm) {
    __shared__ double red[4];
    double total = joined_partials<KIND>(partial, partials, red);
    total = KIND == 2 ? sqrt(total) : total;
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
    const double ratio = max_norm / (total + 1e-6);
    const float f = ratio != ratio || ratio < 1.0 ? (float)ratio : 1.0f;
    for_chunks<true>(t, [&](int i, int64_t at, int n) {
        if (t.out[i] == t.grad[i] && f == 1.0f) return;
        const int from = t.dtype[i], to = t.out_dtype[i];
        if (from == MDP_DTYPE_F32) chunk_scale<float, float>(t.grad[i], t.out[i], at, n, f);
        else if (from == MDP_DTYPE_BF16 && to == from) chunk_scale<bf16, bf16>(t.grad[i], t.out[i], at, n, f);
        else if (from == MDP_DTYPE_BF16) chunk_scale<bf16, float>(t.grad[i], t.out[i], at, n, f);
        else if (to == from) chunk_scale<f16, f16>(t.grad[i], t.out[i], at, n, f);
        else chunk_scale<f16, float>(t.grad[i], t.out[i], at, n, f);
    });
}

int64_t bytes_of(int dtype) { return dtype == MDP_DTYPE_F32 ? 4 : 2; }

// Outputs may not overlap each other, nor a gradient other than their own (exactly the same memory, for a call in place).
int check_overlap(const mdp_grad_t* g, int64_t n) {
    struct Range { uintptr_t lo, hi; int64_t of; bool out; };
    std::unique_ptr<Range[]> r(new (std::nothrow) Range[2 * n]);
    if (!r) return fail(MDP_ERR_RUNTIME, "grad_clip: out of host memory");
    int64_t k = 0;
    for (int64_t i = 0; i < n; ++i) {
        if (!g[i].count) continue;
        const uintptr_t in = (uintptr_t)g[i].grad, out = (uintptr_t)g[i].out;
        r[k++] = Range{out, out + (uintptr_t)(g[i].count * bytes_of(g[i].out_dtype)), i, true};
        if (in != out) r[k++] = Range{in, in + (uintptr_t)(g[i].count * bytes_of(g[i].dtype)), i, false};
        else MDP_REQUIRE(g[i].dtype == g[i].out_dtype, "grad_clip: tensor %lld is clipped in place into another type", (long long)i);
    }
    std::sort(r.get(), r.get() + k, [](const Range& a, const Range& b) { return a.lo < b.lo; });
    uintptr_t hi_out = 0, hi_any = 0;                  // furthest end of the ranges before
    for (int64_t i = 0; i < k; ++i) {
        MDP_REQUIRE(r[i].lo >= hi_out && !(r[i].out && r[i].lo < hi_any),
                    "grad_clip: the output of a tensor overlaps another tensor (tensor %lld)", (long long)r[i].of);
        if (r[i].out) hi_out = std::max(hi_out, r[i].hi);
        hi_any = std::max(hi_any, r[i].hi);
    }
    return MDP_OK;
}

int check_grads(const mdp_grad_t* g, int64_t n, int kind, const double* workspace, const float* norm, bool clip) {
    MDP_REQUIRE(n >= 0 && n <= (1 << 24), "grad norm: %lld tensors", (long long)n);
    MDP_REQUIRE(kind >= 0 && kind <= 2, "grad norm: kind %d is not 0 (inf), 1 or 2", kind);
    MDP_REQUIRE(n == 0 || g, "grad norm: null table");
    MDP_REQUIRE(workspace && norm, "grad norm: null workspace or norm");
    int64_t total = 0;
    for (int64_t i = 0; i < n; ++i) {
        MDP_REQUIRE(g[i].count >= 0, "grad norm: tensor %lld holds %lld elements", (long long)i, (long long)g[i].count);
        MDP_REQUIRE(g[i].count <= kMost && (total += g[i].count) <= kMost, "grad norm: more than 2^40 elements");
        MDP_REQUIRE(g[i].dtype >= 0 && g[i].dtype < MDP_DTYPE_NUM, "grad norm: tensor %lld has element type %d", (long long)i, g[i].dtype);
        MDP_REQUIRE(!g[i].count || g[i].grad, "grad norm: tensor %lld is null", (long long)i);
        MDP_REQUIRE((uintptr_t)g[i].grad % bytes_of(g[i].dtype) == 0, "grad norm: tensor %lld starts between two elements", (long long)i);
        if (!clip) continue;
        MDP_REQUIRE(!g[i].count || g[i].out, "grad_clip: output %lld is null", (long long)i);
        MDP_REQUIRE(g[i].out_dtype == g[i].dtype || g[i].out_dtype == MDP_DTYPE_F32,
                    "grad_clip: output %lld is neither of its gradient's type nor float32", (long long)i);
        MDP_REQUIRE((uintptr_t)g[i].out % bytes_of(g[i].out_dtype) == 0, "grad_clip: output %lld starts between two elements", (long long)i);
    }
    return MDP_OK;
}

// Cuts the list into tables and calls f(table, blocks) for each.
template <class F>
void for_tables(const mdp_grad_t* g, int64_t n, F&& f) {
    Table t;
    std::memset(&t, 0, sizeof(t));
    int64_t chunks = 0;
    const auto flush = [&] {
        if (!t.n) return;
        t.start[t.n] = t.chunks = (int)chunks;
        f(t, (unsigned)std::min<int64_t>(chunks, kBlocks));
        t.n = 0;
        chunks = 0;
    };
    for (int64_t i = 0; i < n; ++i) {
        if (!g[i].count) continue;
        const int64_t c = (g[i].count + kChunk - 1) / kChunk;
        if (t.n == kTable) flush();
        t.grad[t.n] = g[i].grad;
        t.out[t.n] = g[i].out;
        t.count[t.n] = g[i].count;
        t.dtype[t.n] = (uint8_t)g[i].dtype;
        t.out_dtype[t.n] = (uint8_t)g[i].out_dtype;
        t.start[t.n++] = (int)chunks;
        chunks += c;
    }
    flush();
}

#define BY_KIND(kind, launch)                                   \
    do {                                                        \
        if ((kind) == 2) { constexpr int K = 2; launch; }       \
        else if ((kind) == 1) { constexpr int K = 1; launch; }  \
        else { constexpr int K = 0; launch; }                   \
    } while (0)

int64_t launch_partials(const mdp_grad_t* g, int64_t n, int kind, double* partial, hipStream_t s) {
    int64_t partials = 0;
    for_tables(g, n, [&](const Table& t, unsigned blocks) {
        BY_KIND(kind, hipLaunchKernelGGL(k_grad_partial<K>, dim3(blocks), dim3(256), 0, s, t, partial + partials));
        partials += blocks;
    });
    return partials;
}

}  // namespace

// the partial sums of each table, and what they join to
extern "C" int64_t mdp_grad_workspace(int64_t num_grads) {
    const int64_t n = num_grads > 0 ? num_grads : 0;
    return 1 + kBlocks * ((n + kTable - 1) / kTable);
}

extern "C" int mdp_grad_norm(const mdp_grad_t* grads, int64_t num_grads, int norm_kind, double* workspace, float* norm,
                             void* stream) {
    if (int rc = check_grads(grads, num_grads, norm_kind, workspace, norm, false)) return rc;
    hipStream_t s = as_stream(stream);
    const int partials = (int)launch_partials(grads, num_grads, norm_kind, workspace, s);
    BY_KIND(norm_kind, hipLaunchKernelGGL(k_grad_finish<K>, dim3(1), dim3(256), 0, s, workspace, partials, workspace + partials, norm));
    MDP_LAUNCH_CHECK();
    return MDP_OK;
}

extern "C" int mdp_grad_clip(const mdp_grad_t* grads, int64_t num_grads, int norm_kind, double max_norm, double* workspace,
                             float* norm, void* stream) {
    if (int rc = check_grads(grads, num_grads, norm_kind, workspace, norm, true)) return rc;
    MDP_REQUIRE(max_norm >= 0.0, "grad_clip: max_norm %g is negative or NaN", max_norm);
    if (int rc = check_overlap(grads, num_grads)) return rc;
    hipStream_t s = as_stream(stream);
    const int partials = (int)launch_partials(grads, num_grads, norm_kind, workspace, s);
    const bool joined = partials == 0 || partials > kBlocks;
    if (joined)
        BY_KIND(norm_kind, hipLaunchKernelGGL(k_grad_finish<K>, dim3(1), dim3(256), 0, s, workspace, partials, workspace + partials, norm));
    for_tables(grads, num_grads, [&](const Table& t, unsigned blocks) {
        BY_KIND(norm_kind, hipLaunchKernelGGL(k_grad_scale<K>, dim3(blocks), dim3(256), 0, s, t, workspace + (joined ? partials : 0),
                                              joined ? 1 : partials, max_norm, joined ? nullptr : norm));
    });
    MDP_LAUNCH_CHECK();
    return MDP_OK;
}

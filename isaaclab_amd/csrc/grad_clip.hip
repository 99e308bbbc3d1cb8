// The norm of many gradients taken as one vector, and clipping to it.
//
//   norm = (sum |g|^q)^(1/q) over every element of every tensor (q = 1, 2; or the maximum);  out = g min(1, max_norm / (norm + 1e-6))
//
// Sums are held in 64 bits (the square of a float is exact there, so neither large nor small gradients leave the range) and
// taken in an order that depends on the sizes alone.
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

// calls f(tensor, first element, elements) for each of this block's chunks: block b of B takes chunks [b C / B, (b + 1) C / B)
template <class F>
MDP_DEV void for_chunks(const Table& t, F&& f) {
    int64_t c = (int64_t)blockIdx.x * t.chunks / gridDim.x;
    const int64_t end = (int64_t)(blockIdx.x + 1) * t.chunks / gridDim.x;
    int i = 0;
    while (i + 1 < t.n && t.start[i + 1] <= c) ++i;
    for (; c < end; ++c) {
        while (t.start[i + 1] <= c) ++i;
        const int64_t at = (c - t.start[i]) * kChunk, left = t.count[i] - at;
        f(i, at, (int)(left < kChunk ? left : kChunk));
    }
}

template <int KIND, typename T>
MDP_DEV double chunk_norm(const T* g, int n, double acc) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const double v = (double)to_f32(g[i]);
        acc = joined<KIND>(acc, KIND == 2 ? v * v : fabs(v));
    }
    return acc;
}

template <int KIND>
__global__ __launch_bounds__(256) void k_grad_partial(Table t, double* __restrict__ partial) {
    __shared__ double red[4];
    double acc = 0.0;
    for_chunks(t, [&](int i, int64_t at, int n) {
        if (t.dtype[i] == MDP_DTYPE_F32) acc = chunk_norm<KIND>((const float*)t.grad[i] + at, n, acc);
        else if (t.dtype[i] == MDP_DTYPE_BF16) acc = chunk_norm<KIND>((const bf16*)t.grad[i] + at, n, acc);
        else acc = chunk_norm<KIND>((const f16*)t.grad[i] + at, n, acc);
    });
    acc = block_join<KIND>(acc, red);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

template <int KIND>
__global__ __launch_bounds__(256) void k_grad_finish(const double* __restrict__ partial, int64_t n, double max_norm,
                                                     float* __restrict__ norm, float* __restrict__ factor) {
    __shared__ double red[4];
    double acc = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 256) acc = joined<KIND>(acc, partial[i]);
    acc = block_join<KIND>(acc, red);
    if (threadIdx.x) return;
    if (KIND == 2) acc = sqrt(acc);
    *norm = (float)acc;
    const double f = max_norm / (acc + 1e-6);
    if (factor) *factor = f != f || f < 1.0 ? (float)f : 1.0f;
}

template <typename T, typename U>
MDP_DEV void chunk_scale(const T* g, U* out, int n, float f) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) from_f32(to_f32(g[i]) * f, out[i]);
}

__global__ __launch_bounds__(256) void k_grad_scale(Table t, const float* __restrict__ factor) {
    const float f = *factor;
    for_chunks(t, [&](int i, int64_t at, int n) {
        if (t.out[i] == t.grad[i] && f == 1.0f) return;
        const int from = t.dtype[i], to = t.out_dtype[i];
        if (from == MDP_DTYPE_F32) chunk_scale((const float*)t.grad[i] + at, (float*)t.out[i] + at, n, f);
        else if (from == MDP_DTYPE_BF16 && to == from) chunk_scale((const bf16*)t.grad[i] + at, (bf16*)t.out[i] + at, n, f);
        else if (from == MDP_DTYPE_BF16) chunk_scale((const bf16*)t.grad[i] + at, (float*)t.out[i] + at, n, f);
        else if (to == from) chunk_scale((const f16*)t.grad[i] + at, (f16*)t.out[i] + at, n, f);
        else chunk_scale((const f16*)t.grad[i] + at, (float*)t.out[i] + at, n, f);
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
        if (!clip) continue;
        MDP_REQUIRE(!g[i].count || g[i].out, "grad_clip: output %lld is null", (long long)i);
        MDP_REQUIRE(g[i].out_dtype == g[i].dtype || g[i].out_dtype == MDP_DTYPE_F32,
                    "grad_clip: output %lld is neither of its gradient's type nor float32", (long long)i);
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

void launch_norm(const mdp_grad_t* g, int64_t n, int kind, double max_norm, double* workspace, float* norm, float* factor,
                 hipStream_t s) {
    int64_t partials = 0;
    for_tables(g, n, [&](const Table& t, unsigned blocks) {
        BY_KIND(kind, hipLaunchKernelGGL(k_grad_partial<K>, dim3(blocks), dim3(256), 0, s, t, workspace + 1 + partials));
        partials += blocks;
    });
    BY_KIND(kind, hipLaunchKernelGGL(k_grad_finish<K>, dim3(1), dim3(256), 0, s, workspace + 1, partials, max_norm, norm, factor));
}

}  // namespace

// one word for the factor, then the partial sums of each table
extern "C" int64_t mdp_grad_workspace(int64_t num_grads) {
    const int64_t n = num_grads > 0 ? num_grads : 0;
    return 1 + kBlocks * ((n + kTable - 1) / kTable);
}

extern "C" int mdp_grad_norm(const mdp_grad_t* grads, int64_t num_grads, int norm_kind, double* workspace, float* norm,
                             void* stream) {
    if (int rc = check_grads(grads, num_grads, norm_kind, workspace, norm, false)) return rc;
    launch_norm(grads, num_grads, norm_kind, 0.0, workspace, norm, nullptr, as_stream(stream));
    MDP_LAUNCH_CHECK();
    return MDP_OK;
}

extern "C" int mdp_grad_clip(const mdp_grad_t* grads, int64_t num_grads, int norm_kind, double max_norm, double* workspace,
                             float* norm, void* stream) {
    if (int rc = check_grads(grads, num_grads, norm_kind, workspace, norm, true)) return rc;
    MDP_REQUIRE(max_norm >= 0.0, "grad_clip: max_norm %g is negative or NaN", max_norm);
    if (int rc = check_overlap(grads, num_grads)) return rc;
    hipStream_t s = as_stream(stream);
    float* factor = (float*)workspace;
    launch_norm(grads, num_grads, norm_kind, max_norm, workspace, norm, factor, s);
    for_tables(grads, num_grads, [&](const Table& t, unsigned blocks) {
        hipLaunchKernelGGL(k_grad_scale, dim3(blocks), dim3(256), 0, s, t, factor);
    });
    MDP_LAUNCH_CHECK();
    return MDP_OK;
}

// Entry points of the categorical distributions, and the evaluation of stored entries with its gradient.
#include "categorical_device.hpp"

using namespace mdp;

namespace {

__global__ void k_state_advance(unsigned long long* state) { state[1] += 1ull; }

// -- evaluation -------------------------------------------------------------------------------------------------------
// One pass: about the largest entry m so far, s = sum w and t = sum w log2 w with w = 2^((x - m) log2(e) / T).  Entries that
// are not allowed read as -inf and add nothing; a NaN or +inf makes s a NaN.
//
// Bound by memory: a bfloat16 entry costs about ten issue slots (four of them v_exp_f32), two thirds of what a CU issues in the time
// its share of the memory rate brings one.  8192 x 32768 bfloat16: 125 - 137 us for 537 MB while up to 256 MB that ran before are
// still written back (a plain read: 6.1 TB/s), the gradient 170 us for 1074 MB; both in a row 294 us, where three passes at the
// card's copy rate, 4.7 TB/s, are 342.  294912 x 64 float32: 21 and 27 us (75 and 151 MB).  One multiply-add an entry instead of
// subtract and multiply gains nothing and loses the exact 0 of a lone entry; stores past the caches gain nothing either.
constexpr float kLog2E = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct EvalArgs {
    const void* logits; int64_t ld;
    const uint8_t* mask; int64_t ld_mask;
    int vocab; int64_t rows;
    const int64_t* actions;
    const float* temperature; float temperature_s;
    float* log_prob; float* entropy;
    float* stats;                                      // (rows, 3): max, ln s, H
};

struct GradArgs {
    const void* logits; int64_t ld;
    const uint8_t* mask; int64_t ld_mask;
    int vocab; int64_t rows;
    const int64_t* actions;
    const float* temperature; float temperature_s;
    const float* stats;
    const float* grad_log_prob; const float* grad_entropy;
    void* grad; int64_t ld_grad;
    int pieces;                                        // blocks a row
};

MDP_DEV float inverse_temperature(const float* per_row, float scalar, int64_t row) {
    const float t = per_row ? per_row[row] : scalar;
    return t >= 1.17549435e-38f && t < kInf ? 1.0f / t : __builtin_nanf("");     // of a denormal it may be infinite
}

// Half of x - m, from hm = m / 2: stays in range whatever the signs, and is exact to the same bits; its factors are doubled.
MDP_DEV float half_apart(float x, float hm) { return fmaf(x, 0.5f, -hm); }

struct Running {
    float m;
    double s, t;                                       // of chunks that were summed up in 32 bits
    MDP_DEV static Running none() { return Running{-__FLT_MAX__, 0.0, 0.0}; }
    MDP_DEV void move(float to, float c) {             // about another maximum >= m
        float d = half_apart(m, 0.5f * to) * c;
        d = d < -300.0f ? -300.0f : d;                 // 2^-300 is 0: 0 * inf must not arise
        const double f = (double)__builtin_amdgcn_exp2f(d);
        t = f * (t + (double)d * s);
        s *= f;
        m = to;
    }
    // n entries, none above m; summed on their own first: short chains of additions
    template <int N>
    MDP_DEV void add(const float (&v)[N], float c) {
        const float hm = 0.5f * m;
        float cs = 0.0f, ct = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float d = half_apart(v[e], hm) * c, w = __builtin_amdgcn_exp2f(d);
            cs += w;
            ct = fmaf(w, larger(d, -300.0f), ct);      // w is 0 there, and a NaN shows in s
        }
        s += cs;
        t += ct;
    }
};

template <typename T>
MDP_DEV void finish_row(const EvalArgs& g, const Row<T>& r, int64_t row, float m, double s, double t, float inv_t) {
    const float log_s = logf((float)s);
    const float h = s == 0.0 ? 0.0f : log_s - kLn2 * (float)(t / s);
    const int64_t a = g.actions[row];
    float lp;
    if (a == -1) lp = 0.0f;
    else if (a < 0 || a >= r.V) lp = __builtin_nanf("");
    else {
        const float x = r.entry((int)a);               // -inf: masked, or not allowed by itself, also where nothing is (ln s = -inf)
        lp = x > -kInf || s != s ? half_apart(x, 0.5f * m) * (2.0f * inv_t) - log_s : -kInf;
    }
    g.log_prob[row] = lp;
    g.entropy[row] = h;
    if (g.stats) {
        g.stats[3 * row] = m;
        g.stats[3 * row + 1] = log_s;
        g.stats[3 * row + 2] = h;
    }
}

// Rows of up to G K chunks: G lanes of a wave hold a row in registers, so its maximum is known before the first exponential.
template <typename T, bool MASK, int G, int K>
__global__ __launch_bounds__(256) void k_evaluate_short(EvalArgs g) {
    constexpr int N = Chunk<T>::N;
    const int64_t row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const int lane = threadIdx.x % G;
    if (row >= g.rows) return;
    const Row<T> r(g.logits, g.ld, g.mask, g.ld_mask, g.vocab, row);
    const float inv_t = inverse_temperature(g.temperature, g.temperature_s, row), c = 2.0f * inv_t * kLog2E;
    float v[K][N];
#pragma unroll
    for (int k = 0; k < K; ++k) r.template load<MASK>(k * G + lane, v[k]);
    Running q = Running::none();
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e) q.m = larger(v[k][e], q.m);
    q.m = group_max<G>(q.m);
#pragma unroll
    for (int k = 0; k < K; ++k) q.add(v[k], c);
    q.s = group_sum<G>(q.s);
    q.t = group_sum<G>(q.t);
    if (lane == 0) finish_row(g, r, row, q.m, q.s, q.t, inv_t);
}

// Longer rows: a block a row, four chunks a thread in flight, their maximum looked at once.
template <typename T, bool MASK>
__global__ __launch_bounds__(256) void k_evaluate_long(EvalArgs g) {
    constexpr int N = Chunk<T>::N, B = 4;
    __shared__ float wave_m[4];
    __shared__ double wave_s[4], wave_t[4];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const Row<T> r(g.logits, g.ld, g.mask, g.ld_mask, g.vocab, row);
    const float inv_t = inverse_temperature(g.temperature, g.temperature_s, row), c = 2.0f * inv_t * kLog2E;
    const int first = r.full_first(), end = r.full_end();
    Running q = Running::none();
    for (int j0 = first + tid; j0 < end; j0 += 256 * B) {
        Chunk<T> raw[B];
        uint32_t ok[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int j = j0 + 256 * b;
            raw[b] = Chunk<T>::lowest();
            ok[b] = 0;
            if (j < end) {
                raw[b] = r.chunk(j);
                if (MASK) ok[b] = r.allowed_chunk(j);
            }
        }
        float v[B][N], top = q.m;
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                v[b][e] = !MASK || (ok[b] >> e & 1u) ? raw[b].at(e) : -kInf;
                top = larger(v[b][e], top);
            }
        if (top > q.m) q.move(top, c);
#pragma unroll
        for (int b = 0; b < B; ++b) q.add(v[b], c);
    }
    // the entries of the two edge chunks, one a lane
    const int head = first ? min(r.V, N - r.shift) : 0, tail = max(head, end * N - r.shift);
    const int i = tid < head ? tid : tail + tid - head;
    if (i < r.V) {
        const float v[1] = {r.entry(i)};
        if (v[0] > q.m) q.move(v[0], c);
        q.add(v, c);
    }
    const float wm = group_max<64>(q.m);
    if ((tid & 63) == 0) wave_m[tid >> 6] = wm;
    __syncthreads();
    q.move(larger(larger(wave_m[0], wave_m[1]), larger(wave_m[2], wave_m[3])), c);
    q.s = group_sum<64>(q.s);
    q.t = group_sum<64>(q.t);
    if ((tid & 63) == 0) { wave_s[tid >> 6] = q.s; wave_t[tid >> 6] = q.t; }
    __syncthreads();
    if (tid == 0)
        finish_row(g, r, row, q.m, wave_s[0] + wave_s[1] + wave_s[2] + wave_s[3], wave_t[0] + wave_t[1] + wave_t[2] + wave_t[3], inv_t);
}

// Gradient of an entry: -p (gl + ge (ln p + H)) / T, and + gl / T at the action, with log2 p = (x - m) log2(e) / T - log2 s.
// Held at or above -300, where p is 0 in 32 bits, an entry that is not allowed gives a zero by itself; only rows that hold a NaN, or
// whose terms by themselves leave the 32-bit range as 1 / T does near its end (`whole` false), are told apart entry by entry and
// divided by T last.
template <typename T>
struct RowGrad {
    float hm, c, log2_s, a0, a1, hot, last;             // the last: 1 / T in a row whose other terms are not divided by T
    int action;                                        // -1: none in the row
    bool whole;
    MDP_DEV RowGrad(const GradArgs& g, int64_t row) {
        const float inv_t = inverse_temperature(g.temperature, g.temperature_s, row);
        hm = 0.5f * g.stats[3 * row];
        c = 2.0f * inv_t * kLog2E;
        const float log_s = g.stats[3 * row + 1], h = g.stats[3 * row + 2];
        log2_s = log_s == -kInf ? 0.0f : log_s * kLog2E;               // a row without allowed entries: p = 0 everywhere
        const int64_t a = g.actions[row];
        action = a >= 0 && a < g.vocab ? (int)a : -1;
        float gl = g.grad_log_prob ? g.grad_log_prob[row] : 0.0f;
        const float ge = g.grad_entropy ? g.grad_entropy[row] : 0.0f;
        if (a == -1) gl = 0.0f;
        else if (action < 0) gl = __builtin_nanf("");
        hot = gl * inv_t;
        a0 = -(gl + ge * h) * inv_t;
        a1 = -ge * kLn2 * inv_t;
        const float most = fmaf(fabsf(a1), 300.0f, fabsf(a0)) + fabsf(hot);
        whole = most - most == 0.0f && log2_s == log2_s;
        last = 1.0f;
        if (!whole) {
            hot = gl;
            a0 = -(gl + ge * h);
            a1 = -ge * kLn2;
            last = inv_t;
        }
    }
    MDP_DEV float operator()(float x) const {
        const float lp = larger(fmaf(half_apart(x, hm), c, -log2_s), -300.0f);
        return __builtin_amdgcn_exp2f(lp) * fmaf(a1, lp, a0);
    }
    MDP_DEV float by_itself(float x, float own) const {
        if (x == -kInf) return 0.0f;
        float lp = fmaf(half_apart(x, hm), c, -log2_s);
        lp = lp < -300.0f ? -300.0f : lp;              // a NaN stays
        return (__builtin_amdgcn_exp2f(lp) * fmaf(a1, lp, a0) + own) * last;
    }
    // gradients of N entries from entry i0 on, in place
    template <int N>
    MDP_DEV void apply(float (&v)[N], int i0) const {
        const int at = action - i0;
        const bool here = (unsigned)at < (unsigned)N;  // the action is one of them
        if (!whole) {
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = by_itself(v[e], here && e == at ? hot : 0.0f);
            return;
        }
        uint32_t possible = 0;
        if (here)
#pragma unroll
            for (int e = 0; e < N; ++e) possible |= e == at && v[e] != -kInf ? 1u << e : 0u;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = (*this)(v[e]);
        if (here)
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] += possible >> e & 1u ? hot : 0.0f;
    }
};

template <typename T, bool MASK, int G, int K>
__global__ __launch_bounds__(256) void k_grad_short(GradArgs g) {
    constexpr int N = Chunk<T>::N;
    const int64_t row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const int lane = threadIdx.x % G;
    if (row >= g.rows) return;
    const Row<T> r(g.logits, g.ld, g.mask, g.ld_mask, g.vocab, row);
    T* out = (T*)g.grad + row * g.ld_grad;
    const bool same = ((uintptr_t)out & 15) == ((uintptr_t)r.x & 15);
    const RowGrad<T> f(g, row);
    float v[K][N];
#pragma unroll
    for (int k = 0; k < K; ++k) r.template load<MASK>(k * G + lane, v[k]);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int j = k * G + lane, i0 = j * N - r.shift;
        f.apply(v[k], i0);
        if (same && r.full(j)) *(uint4*)(out + i0) = Chunk<T>::of(v[k]).raw;
        else
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (i0 + e >= 0 && i0 + e < r.V) from_f32(v[k][e], out[i0 + e]);
    }
}

// Longer rows: `pieces` blocks a row.  Rows are taken from the last one on: those the evaluation read last, so that part of
// them is still in the caches.
template <typename T, bool MASK>
__global__ __launch_bounds__(256) void k_grad_long(GradArgs g) {
    constexpr int N = Chunk<T>::N, B = 4;
    const int64_t row = g.rows - 1 - blockIdx.x / g.pieces;
    const int piece = blockIdx.x % g.pieces, tid = threadIdx.x;
    const Row<T> r(g.logits, g.ld, g.mask, g.ld_mask, g.vocab, row);
    T* out = (T*)g.grad + row * g.ld_grad;
    const bool same = ((uintptr_t)out & 15) == ((uintptr_t)r.x & 15);
    const int first = r.full_first(), end = r.full_end();
    for (int j0 = first + piece * (256 * B) + tid; j0 < end; j0 += g.pieces * (256 * B)) {
        Chunk<T> raw[B];
        uint32_t ok[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int j = j0 + 256 * b;
            raw[b] = Chunk<T>::lowest();
            ok[b] = 0;
            if (j < end) {
                raw[b] = r.chunk(j);
                if (MASK) ok[b] = r.allowed_chunk(j);
            }
        }
        const RowGrad<T> f(g, row);                    // after the loads of the entries are on their way
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int j = j0 + 256 * b, i0 = j * N - r.shift;
            if (j >= end) break;
            float v[N];
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = !MASK || (ok[b] >> e & 1u) ? raw[b].at(e) : -kInf;
            f.apply(v, i0);
            if (same) *(uint4*)(out + i0) = Chunk<T>::of(v).raw;
            else
#pragma unroll
                for (int e = 0; e < N; ++e) from_f32(v[e], out[i0 + e]);
        }
    }
    if (piece) return;
    const int head = first ? min(r.V, N - r.shift) : 0, tail = max(head, end * N - r.shift);
    const int i = tid < head ? tid : tail + tid - head;
    if (i < r.V) {
        const RowGrad<T> f(g, row);
        float v[1] = {r.entry(i)};
        f.apply(v, i);
        from_f32(v[0], out[i]);
    }
}

int check_rows(const char* what, const void* logits, int64_t rows, int64_t vocab, int64_t ld, int dtype, const uint8_t* mask,
               int64_t ld_mask) {
    MDP_REQUIRE(rows >= 0 && vocab >= 0, "%s: negative shape (%lld, %lld)", what, (long long)rows, (long long)vocab);
    MDP_REQUIRE(dtype >= 0 && dtype < MDP_DTYPE_NUM, "%s: unknown element type %d", what, dtype);
    MDP_REQUIRE(rows <= ((int64_t)1 << 40), "%s: %lld rows are too many", what, (long long)rows);
    MDP_REQUIRE(vocab < (1 << 30), "%s: rows of %lld entries are too long", what, (long long)vocab);
    if (rows == 0) return MDP_OK;
    MDP_REQUIRE(vocab > 0, "%s: rows without entries", what);
    MDP_REQUIRE(logits, "%s: null logits", what);
    MDP_REQUIRE(ld >= 0 && ld_mask >= 0, "%s: negative row stride", what);
    MDP_REQUIRE((uintptr_t)logits % (dtype == MDP_DTYPE_F32 ? 4 : 2) == 0, "%s: logits between two elements", what);
    return MDP_OK;
}

// That number decides how many lanes hold a row; beyond 512 chunks (2048 floats, 4096 16-bit entries) a row is a block's.  float32,
// 2^26 entries, both passes: rows of 1028 159 us by a wave, 222 by a block; of 2048 154 and 151; of 4096 141 by a block.
template <typename T, bool MASK>
void launch_evaluate(const EvalArgs& g, hipStream_t s) {
    const int chunks = most_chunks<T>(g.logits, g.ld, g.rows, g.vocab);
#define SHORT(G, K)                                                                                                            \
    if (chunks <= G * K) {                                                                                                     \
        hipLaunchKernelGGL((k_evaluate_short<T, MASK, G, K>), dim3((unsigned)((g.rows + 256 / G - 1) / (256 / G))), dim3(256), 0, s, g); \
        return;                                                                                                                \
    }
    SHORT(4, 1) SHORT(4, 2) SHORT(4, 4) SHORT(8, 4) SHORT(16, 4) SHORT(32, 4) SHORT(64, 4) SHORT(64, 8)
#undef SHORT
    hipLaunchKernelGGL((k_evaluate_long<T, MASK>), dim3((unsigned)g.rows), dim3(256), 0, s, g);
}

template <typename T, bool MASK>
void launch_grad(GradArgs g, hipStream_t s) {
    const int chunks = most_chunks<T>(g.logits, g.ld, g.rows, g.vocab);
#define SHORT(G, K)                                                                                                        \
    if (chunks <= G * K) {                                                                                                 \
        hipLaunchKernelGGL((k_grad_short<T, MASK, G, K>), dim3((unsigned)((g.rows + 256 / G - 1) / (256 / G))), dim3(256), 0, s, g); \
        return;                                                                                                            \
    }
    SHORT(4, 1) SHORT(4, 2) SHORT(4, 4) SHORT(8, 4) SHORT(16, 4) SHORT(32, 4) SHORT(64, 4) SHORT(64, 8)
#undef SHORT
    const int64_t most = ((1 << 24) - 1) / g.rows;     // a launch's blocks of 256 threads
    g.pieces = (int)std::max<int64_t>(1, std::min<int64_t>(most, (chunks + 1023) / 1024));
    hipLaunchKernelGGL((k_grad_long<T, MASK>), dim3((unsigned)(g.rows * g.pieces)), dim3(256), 0, s, g);
}

// A launch holds fewer than 2^32 threads: calls of more rows than blocks of 1024 fill that with are cut, f(first row, rows).
constexpr int64_t kRows = 1 << 21;
template <class F>
void by_rows(int64_t rows, F&& f) {
    for (int64_t at = 0; at < rows; at += kRows) f(at, std::min(kRows, rows - at));
}
template <typename P>
P* offset(P* p, int64_t by) { return p ? p + by : p; }

template <class F>
void by_type(int dtype, bool mask, F&& f) {
    if (dtype == MDP_DTYPE_F32) mask ? f(float{}, std::true_type{}) : f(float{}, std::false_type{});
    else if (dtype == MDP_DTYPE_BF16) mask ? f(bf16{}, std::true_type{}) : f(bf16{}, std::false_type{});
    else mask ? f(f16{}, std::true_type{}) : f(f16{}, std::false_type{});
}

}  // namespace

extern "C" int mdp_categorical_sample(const mdp_categorical_sample_t* a, void* stream) {
    MDP_REQUIRE(a, "null arguments");
    if (int rc = check_rows("categorical_sample", a->logits, a->rows, a->vocab, a->ld, a->dtype, a->mask, a->ld_mask)) return rc;
    if (a->rows == 0) return MDP_OK;
    MDP_REQUIRE(a->actions && a->log_prob, "categorical_sample: null output");
    MDP_REQUIRE(a->u || a->state, "categorical_sample needs uniforms or a generator state {seed, epoch}");
    hipStream_t s = as_stream(stream);
    by_type(a->dtype, a->mask, [&](auto t, auto m) {
        using T = decltype(t);
        by_rows(a->rows, [&](int64_t at, int64_t rows) {
            const SampleArgs g{(const T*)a->logits + at * a->ld, a->ld, offset(a->mask, at * a->ld_mask), a->ld_mask, (int)a->vocab,
                               rows, at, offset(a->temperature, at), offset(a->top_k, at), offset(a->top_p, at), offset(a->min_p, at),
                               rate_of(a->temperature_scalar), a->top_k_scalar, a->top_p_scalar, a->min_p_scalar, offset(a->u, at),
                               (const unsigned long long*)a->state, a->actions + at, a->log_prob + at};
            launch_sample<T, decltype(m)::value>(g, s);
        });
    });
    if (!a->u) hipLaunchKernelGGL(k_state_advance, dim3(1), dim3(1), 0, s, (unsigned long long*)a->state);
    MDP_LAUNCH_CHECK();
    return MDP_OK;
}

extern "C" int mdp_categorical_evaluate(const mdp_categorical_eval_t* a, void* stream) {
    MDP_REQUIRE(a, "null arguments");
    if (int rc = check_rows("categorical_evaluate", a->logits, a->rows, a->vocab, a->ld, a->dtype, a->mask, a->ld_mask)) return rc;
    if (a->rows == 0) return MDP_OK;
    MDP_REQUIRE(a->actions && a->log_prob && a->entropy, "categorical_evaluate: null pointer");
    hipStream_t s = as_stream(stream);
    by_type(a->dtype, a->mask, [&](auto t, auto m) {
        using T = decltype(t);
        by_rows(a->rows, [&](int64_t at, int64_t rows) {
            const EvalArgs g{(const T*)a->logits + at * a->ld, a->ld, offset(a->mask, at * a->ld_mask), a->ld_mask, (int)a->vocab, rows,
                             a->actions + at, offset(a->temperature, at), a->temperature_scalar, a->log_prob + at, a->entropy + at,
                             offset(a->stats, 3 * at)};
            launch_evaluate<T, decltype(m)::value>(g, s);
        });
    });
    MDP_LAUNCH_CHECK();
    return MDP_OK;
}

extern "C" int mdp_categorical_evaluate_grad(const mdp_categorical_eval_t* a, const float* grad_log_prob,
                                             const float* grad_entropy, void* grad_logits, int64_t ld_grad, void* stream) {
    MDP_REQUIRE(a, "null arguments");
    if (int rc = check_rows("categorical_evaluate_grad", a->logits, a->rows, a->vocab, a->ld, a->dtype, a->mask, a->ld_mask)) return rc;
    if (a->rows == 0) return MDP_OK;
    MDP_REQUIRE(a->actions && a->stats && grad_logits, "categorical_evaluate_grad: null pointer");
    MDP_REQUIRE(ld_grad >= a->vocab, "categorical_evaluate_grad: gradient rows overlap");
    MDP_REQUIRE((uintptr_t)grad_logits % (a->dtype == MDP_DTYPE_F32 ? 4 : 2) == 0, "categorical_evaluate_grad: gradient between two elements");
    hipStream_t s = as_stream(stream);
    by_type(a->dtype, a->mask, [&](auto t, auto m) {
        using T = decltype(t);
        by_rows(a->rows, [&](int64_t at, int64_t rows) {
            const GradArgs g{(const T*)a->logits + at * a->ld, a->ld, offset(a->mask, at * a->ld_mask), a->ld_mask, (int)a->vocab, rows,
                             a->actions + at, offset(a->temperature, at), a->temperature_scalar, a->stats + 3 * at,
                             offset(grad_log_prob, at), offset(grad_entropy, at), (T*)grad_logits + at * ld_grad, ld_grad, 1};
            launch_grad<T, decltype(m)::value>(g, s);
        });
    });
    MDP_LAUNCH_CHECK();
    return MDP_OK;
}

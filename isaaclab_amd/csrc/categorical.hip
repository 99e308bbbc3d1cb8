// Categorical distributions over the last axis of a tensor of logits: drawing an entry from given uniforms, and the
// log-probability and entropy of stored entries with their gradient by the logits.
//
// With the allowed entries A = {i : mask_i and x_i > -inf}, m = max_A x and w_i = exp((x_i - m) / T):
//   draw      order A by (x falling, i rising); keep the first k, of these the shortest prefix that holds a share p of
//             their mass, of these the entries with w_i >= min_p.  What is kept is a prefix of the order, so it is the set
//             {x > tau} plus the first r entries equal to tau.  With W = its mass, the answer is the first i (by index)
//             whose running mass exceeds u W; its log-probability is ln(w_i / W).
//   evaluate  s = sum_A w, t = sum_A w ln w: log p_a = ln w_a - ln s, H = ln s - t / s.
//   gradient  d/dx_i = (gl (d_ia - p_i) - ge p_i (ln p_i + H)) / T.
#include "mdp_device.hpp"
#include "mdp_host.hpp"
#include "elements_device.hpp"
#include <algorithm>
#include <type_traits>

using namespace mdp;

namespace {

constexpr float kInf = __builtin_inff();

// order-preserving key of a float; -0 and +0 are one value
MDP_DEV uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u >> 31) ? ~u : u | 0x80000000u;
}
MDP_DEV float of_key(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }

// 2^t for t <= 0 in 64 bits: t = n + f with |f| <= 1/2, 2^f by its Taylor series (ln 2)^k / k! f^k; the first term left
// out, (ln 2 / 2)^13 / 13!, is 1.7e-16.  64-bit multiply-adds issue at the rate of 32-bit ones on this chip.
MDP_DEV double exp2_neg(double t) {
    t = t < -1100.0 ? -1100.0 : t;               // below the smallest denormal: 0
    const double n = __builtin_rint(t), f = t - n;
    double p = 2.5678435993488196e-11;
    p = fma(p, f, 4.44553827187081e-10);
    p = fma(p, f, 7.054911620801121e-09);
    p = fma(p, f, 1.0178086009239696e-07);
    p = fma(p, f, 1.3215486790144305e-06);
    p = fma(p, f, 1.5252733804059838e-05);
    p = fma(p, f, 0.00015403530393381606);
    p = fma(p, f, 0.0013333558146428441);
    p = fma(p, f, 0.009618129107628477);
    p = fma(p, f, 0.055504108664821576);
    p = fma(p, f, 0.2402265069591007);
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)n);
}

// -- reductions: every lane gets the result; sums in a fixed order -----------------------------------------------------
MDP_DEV double wave_sum(double v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
MDP_DEV int64_t wave_sum(int64_t v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((long long)v, o);
    return v;
}
MDP_DEV float wave_max(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
MDP_DEV double wave_scan(double v) {                 // inclusive
    const int lane = threadIdx.x & 63;
    for (int o = 1; o < 64; o <<= 1) {
        const double up = __shfl_up(v, o);
        if (lane >= o) v += up;
    }
    return v;
}

struct SampleArgs {
    const void* logits; int64_t ld;
    const uint8_t* mask; int64_t ld_mask;
    int vocab;
    const float* temperature; const int* top_k; const float* top_p; const float* min_p;
    float temperature_s; int top_k_s; float top_p_s; float min_p_s;
    const float* u; const unsigned long long* state;
    int64_t* actions; float* log_prob;
};

constexpr uint32_t kStream = 0x43415447u;

template <int THREADS>
struct Block {
    static constexpr int W = THREADS / 64;
    struct Shared { double d[W]; int64_t n[W]; float f[W]; int bad[W]; };
    Shared* s;
    MDP_DEV double sum(double v) {
        v = wave_sum(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s->d[threadIdx.x >> 6] = v;
        __syncthreads();
        double r = 0.0;
        for (int w = 0; w < W; ++w) r += s->d[w];
        return r;
    }
    MDP_DEV int64_t sum(int64_t v) {
        v = wave_sum(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s->n[threadIdx.x >> 6] = v;
        __syncthreads();
        int64_t r = 0;
        for (int w = 0; w < W; ++w) r += s->n[w];
        return r;
    }
    MDP_DEV float max(float v) {
        v = wave_max(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s->f[threadIdx.x >> 6] = v;
        __syncthreads();
        float r = s->f[0];
        for (int w = 1; w < W; ++w) r = fmaxf(r, s->f[w]);
        return r;
    }
};

// One block draws one row.  Each question about the row (its maximum, how many entries and how much mass lie at or above a
// key, where the running mass passes u W) is one pass over it.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void k_sample_row(SampleArgs g) {
    using B = Block<THREADS>;
    __shared__ typename B::Shared sh;
    __shared__ double wave_mass[B::W];
    __shared__ int64_t wave_level[B::W];
    B b{&sh};
    const int64_t row = blockIdx.x;
    const int V = g.vocab, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T* x = (const T*)g.logits + row * g.ld;
    const uint8_t* mask = g.mask ? g.mask + row * g.ld_mask : nullptr;
    const auto load = [&](int i) { return mask && !mask[i] ? -kInf : to_f32(x[i]); };

    const float temp = g.temperature ? g.temperature[row] : g.temperature_s;
    float m = -kInf;
    int64_t bad = 0;
    for (int i = tid; i < V; i += THREADS) {
        const float v = load(i);
        bad |= v != v || v == kInf;
        m = fmaxf(m, v);
    }
    m = b.max(m);
    bad = b.sum(bad);
    if (bad || !(temp >= 0.0f)) {                      // no distribution
        if (tid == 0) { g.actions[row] = -1; g.log_prob[row] = __builtin_nanf(""); }
        return;
    }
    if (m == -kInf) {                                  // nothing to choose from
        if (tid == 0) { g.actions[row] = -1; g.log_prob[row] = 0.0f; }
        return;
    }
    const bool greedy = temp == 0.0f;
    const double c = greedy ? 0.0 : 1.4426950408889634 / (double)temp;
    const auto weight = [&](float v) { return v == -kInf ? 0.0 : exp2_neg(((double)v - (double)m) * c); };
    const auto count_from = [&](uint32_t k) {
        int64_t n = 0;
        for (int i = tid; i < V; i += THREADS) n += key_of(load(i)) >= k;
        return b.sum(n);
    };
    const auto mass_from = [&](uint32_t k) {
        double n = 0.0;
        for (int i = tid; i < V; i += THREADS) { const float v = load(i); n += key_of(v) >= k ? weight(v) : 0.0; }
        return b.sum(n);
    };

    // the prefix {key > tau} and the first `room` entries of key tau
    const uint32_t top = key_of(m), lowest = key_of(-kInf) + 1u;
    uint32_t tau = greedy ? top : lowest;
    int64_t room = greedy ? 1 : V;
    float p = g.top_p ? g.top_p[row] : g.top_p_s, mp = g.min_p ? g.min_p[row] : g.min_p_s;
    const int64_t k = g.top_k ? g.top_k[row] : g.top_k_s;
    if (!greedy) {
        if (k > 0 && k < V && count_from(lowest) > k) {
            uint32_t lo = lowest, hi = top;
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo + 1u) / 2u;
                if (count_from(mid) >= k) lo = mid; else hi = mid - 1u;
            }
            tau = lo;
            room = k - count_from(tau + 1u);
        }
        if (p < 1.0f) {
            p = p > 0.0f ? p : 0.0f;
            const double above = mass_from(tau + 1u);
            int64_t level = count_from(tau) - count_from(tau + 1u);
            if (level > room) level = room;
            const double aim = (double)p * (above + (double)level * weight(of_key(tau)));
            uint32_t lo = tau, hi = top;
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo + 1u) / 2u;
                if (mass_from(mid) >= aim) lo = mid; else hi = mid - 1u;
            }
            // entries of the level: each that has less than `aim` before it
            const double need = (aim - mass_from(lo + 1u)) / weight(of_key(lo));
            int64_t r = need < 1.0 ? 1 : need > (double)V ? V : (int64_t)__builtin_ceil(need);
            room = lo == tau && room < r ? room : r;
            tau = lo;
        }
    }
    mp = mp > 0.0f ? (mp < 1.0f ? mp : 1.0f) : 0.0f;

    // each wave owns a contiguous piece of the row, so running counts and masses follow the index
    const int piece = ((V + THREADS - 1) / THREADS) * 64, first = wave * piece, last = min(V, first + piece);
    int64_t level = 0;
    for (int i = first + lane; i < last; i += 64) level += key_of(load(i)) == tau;
    level = wave_sum(level);
    if (lane == 0) wave_level[wave] = level;
    __syncthreads();
    int64_t rank0 = 0;
    for (int w = 0; w < wave; ++w) rank0 += wave_level[w];
    const auto walk = [&](auto&& visit) {              // visit(i, weight of entry i if it is kept): uniform over the wave
        int64_t rank = rank0;
        for (int i0 = first; i0 < last; i0 += 64) {
            const int i = i0 + lane;
            const float v = i < last ? load(i) : -kInf;
            const uint32_t key = key_of(v);
            const uint64_t eq = __ballot(key == tau);
            const int64_t mine = rank + __popcll(eq & ((1ull << lane) - 1ull));
            rank += __popcll(eq);
            double w = key > tau || (key == tau && mine < room) ? weight(v) : 0.0;
            w = w >= (double)mp ? w : 0.0;
            if (visit(i, w)) return;
        }
    };
    double mass = 0.0;
    walk([&](int, double w) { mass += w; return false; });
    mass = wave_sum(mass);
    if (lane == 0) wave_mass[wave] = mass;
    __syncthreads();
    double total = 0.0;
    for (int w = 0; w < B::W; ++w) total += wave_mass[w];
    float u = 0.0f;
    if (g.u) u = g.u[row];
    else u = u01(rng4(g.state[0], g.state[1], kStream, (uint64_t)row).x);
    u = u > 0.0f ? (u < 0.99999994f ? u : 0.99999994f) : 0.0f;
    const double aim = (double)u * total;
    int target = -1;
    double before = 0.0, run = 0.0;
    for (int w = 0; w < B::W; ++w) {
        if (wave_mass[w] > 0.0 && run <= aim) { target = w; before = run; }   // the last one that begins at or below the aim
        run += wave_mass[w];
    }
    if (wave != target) return;
    int found = -1;
    double found_w = 0.0;
    walk([&](int i, double w) {
        const double upto = before + wave_scan(w);
        const uint64_t over = __ballot(upto > aim && w > 0.0), some = __ballot(w > 0.0);
        // rounding may leave the aim at the very end of the piece: the last entry with mass is the answer then
        if (some) {
            const int l = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)some);
            found = __shfl(i, l);
            found_w = __shfl(w, l);
        }
        before = __shfl(upto, 63);
        return over != 0ull;
    });
    if (lane == 0) {
        g.actions[row] = found;
        g.log_prob[row] = greedy ? 0.0f : (float)log(found_w / total);
    }
}

__global__ void k_state_advance(unsigned long long* state) { state[1] += 1ull; }

// -- rows ---------------------------------------------------------------------------------------------------------------
// A row as the 16-byte chunks of memory that it touches: chunk j holds entries j N - shift .. j N - shift + N - 1, of which
// the first and the last chunk may hold some that are not the row's.  Those are never read: an edge chunk is read entry by
// entry.  A masked entry reads as -inf.
template <typename T>
struct Row {
    static constexpr int N = Chunk<T>::N;
    const T* x;
    const uint8_t* mask;
    int V, shift;
    bool mask_chunks;                                  // the mask's chunks start on N-byte boundaries where the logits' do

    MDP_DEV Row(const void* logits, int64_t ld, const uint8_t* m, int64_t ld_mask, int vocab, int64_t row)
        : x((const T*)logits + row * ld), mask(m ? m + row * ld_mask : nullptr), V(vocab),
          shift((int)(((uintptr_t)x & 15) / sizeof(T))), mask_chunks((((uintptr_t)mask - (uintptr_t)shift) & (N - 1)) == 0) {}
    MDP_DEV int chunks() const { return (V + shift + N - 1) / N; }
    MDP_DEV int full_first() const { return shift ? 1 : 0; }
    MDP_DEV int full_end() const { return (V + shift) / N; }     // one past the last full chunk
    MDP_DEV bool full(int j) const { return j >= full_first() && j < full_end(); }
    MDP_DEV Chunk<T> chunk(int j) const { return Chunk<T>{*(const uint4*)(x + (j * N - shift))}; }
    MDP_DEV bool allowed(int i) const { return !mask || mask[i]; }
    MDP_DEV float entry(int i) const { return allowed(i) ? to_f32(x[i]) : -kInf; }
    // the mask of a full chunk, one bit an entry
    MDP_DEV uint32_t allowed_chunk(int j) const {
        const uint8_t* m = mask + (j * N - shift);
        uint32_t bits = 0;
        if (mask_chunks) {
            uint32_t w[2];
            if constexpr (N == 4) { w[0] = *(const uint32_t*)m; w[1] = 0; }
            else { const uint2 q = *(const uint2*)m; w[0] = q.x; w[1] = q.y; }
#pragma unroll
            for (int e = 0; e < N; ++e) bits |= ((w[e / 4] >> (8 * (e % 4))) & 0xffu ? 1u : 0u) << e;
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) bits |= (m[e] ? 1u : 0u) << e;
        }
        return bits;
    }
    // entries of chunk j; what is not the row's, or masked, is -inf
    template <bool MASK>
    MDP_DEV void load(int j, float (&v)[N]) const {
        if (full(j)) {
            const Chunk<T> c = chunk(j);
            const uint32_t ok = MASK ? allowed_chunk(j) : ~0u;
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = !MASK || (ok >> e & 1u) ? c.at(e) : -kInf;
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int i = j * N - shift + e;
                v[e] = i >= 0 && i < V && (!MASK || mask[i]) ? to_f32(x[i]) : -kInf;
            }
        }
    }
};

// the larger of two numbers, b where a is a NaN (one instruction, without fmaxf's canonicalisation of its operands)
MDP_DEV float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, kInf); }

// lane i gets lane i ^ m's value (m < 4), or, for m = 4 and 8, that of the lane mirrored inside 8 or 16: what a reduction
// needs whose groups of m already agree
template <int M>
MDP_DEV float across(float v) {
    const int x = __float_as_int(v);
    if constexpr (M == 1) return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0xB1, 0xf, 0xf, true));        // quad_perm 1 0 3 2
    else if constexpr (M == 2) return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x4E, 0xf, 0xf, true));   // quad_perm 2 3 0 1
    else if constexpr (M == 4) return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, true));  // row_half_mirror
    else if constexpr (M == 8) return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, true));  // row_mirror
    else return __shfl_xor(v, M);
}
template <int G, class F>
MDP_DEV float over_group(float v, F&& f) {             // every lane of a group of G gets the result
    if constexpr (G > 1) v = f(v, across<1>(v));
    if constexpr (G > 2) v = f(v, across<2>(v));
    if constexpr (G > 4) v = f(v, across<4>(v));
    if constexpr (G > 8) v = f(v, across<8>(v));
    if constexpr (G > 16) v = f(v, across<16>(v));
    if constexpr (G > 32) v = f(v, across<32>(v));
    return v;
}
template <int G>
MDP_DEV float group_max(float v) { return over_group<G>(v, [](float a, float b) { return larger(a, b); }); }
template <int G>
MDP_DEV float group_sum(float v) { return over_group<G>(v, [](float a, float b) { return a + b; }); }

// -- evaluation -------------------------------------------------------------------------------------------------------
// One pass: about the largest entry m so far, s = sum w and t = sum w log2 w with w = 2^((x - m) log2(e) / T).  Entries that
// are not allowed read as -inf and add nothing; a NaN or +inf makes s a NaN.
//
// Bound by memory: a bfloat16 entry costs about ten issue slots (four of them v_exp_f32), two thirds of what a CU issues in
// the time its share of the memory rate brings one.
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
    return t > 0.0f && t < kInf ? 1.0f / t : __builtin_nanf("");
}

struct Running {
    float m, s, t;
    MDP_DEV static Running none() { return Running{-__FLT_MAX__, 0.0f, 0.0f}; }
    MDP_DEV void move(float to, float c) {             // about another maximum >= m
        float d = (m - to) * c;
        d = d < -300.0f ? -300.0f : d;                 // 2^-300 is 0: 0 * inf must not arise
        const float f = __builtin_amdgcn_exp2f(d);
        t = f * (t + d * s);
        s *= f;
        m = to;
    }
    // n entries, none above m; summed on their own first: short chains of additions
    template <int N>
    MDP_DEV void add(const float (&v)[N], float c) {
        float cs = 0.0f, ct = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float d = (v[e] - m) * c, w = __builtin_amdgcn_exp2f(d);
            cs += w;
            ct = fmaf(w, larger(d, -300.0f), ct);      // w is 0 there, and a NaN shows in s
        }
        s += cs;
        t += ct;
    }
};

template <typename T>
MDP_DEV void finish_row(const EvalArgs& g, const Row<T>& r, int64_t row, float m, float s, float t, float inv_t) {
    const float log_s = logf(s);
    const float h = s == 0.0f ? 0.0f : log_s - kLn2 * (t / s);
    const int64_t a = g.actions[row];
    float lp;
    if (a == -1) lp = 0.0f;
    else if (a < 0 || a >= r.V) lp = __builtin_nanf("");
    else if (!r.allowed((int)a)) lp = s == s ? -kInf : s;
    else lp = (to_f32(r.x[a]) - m) * inv_t - log_s;
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
    const float inv_t = inverse_temperature(g.temperature, g.temperature_s, row), c = inv_t * kLog2E;
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
    __shared__ float wave_m[4], wave_s[4], wave_t[4];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const Row<T> r(g.logits, g.ld, g.mask, g.ld_mask, g.vocab, row);
    const float inv_t = inverse_temperature(g.temperature, g.temperature_s, row), c = inv_t * kLog2E;
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
// Held at or above -300, where p is 0 in 32 bits, an entry that is not allowed gives a zero by itself; only rows that hold a NaN
// (`whole` false) are told apart entry by entry.
template <typename T>
struct RowGrad {
    float m, c, log2_s, a0, a1, hot;
    int action;                                        // -1: none in the row
    bool whole;
    MDP_DEV RowGrad(const GradArgs& g, int64_t row) {
        const float inv_t = inverse_temperature(g.temperature, g.temperature_s, row);
        m = g.stats[3 * row];
        c = inv_t * kLog2E;
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
        whole = a0 - a0 == 0.0f && a1 - a1 == 0.0f && log2_s == log2_s;
    }
    MDP_DEV float operator()(float x) const {
        const float lp = larger(fmaf(x - m, c, -log2_s), -300.0f);
        return __builtin_amdgcn_exp2f(lp) * fmaf(a1, lp, a0);
    }
    MDP_DEV float of_broken(float x) const {
        if (x == -kInf) return 0.0f;
        const float lp = fmaf(x - m, c, -log2_s);
        return __builtin_amdgcn_exp2f(lp) * fmaf(a1, lp, a0);
    }
    // gradients of N entries from entry i0 on, in place
    template <int N>
    MDP_DEV void apply(float (&v)[N], int i0) const {
        const int at = action - i0;
        const bool here = (unsigned)at < (unsigned)N;  // the action is one of them
        uint32_t possible = 0;
        if (here)
#pragma unroll
            for (int e = 0; e < N; ++e) possible |= e == at && v[e] != -kInf ? 1u << e : 0u;
        if (whole)
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = (*this)(v[e]);
        else
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = of_broken(v[e]);
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
    MDP_REQUIRE(rows <= 0x7fffffff, "%s: %lld rows are beyond one launch", what, (long long)rows);
    MDP_REQUIRE(vocab < (1 << 30), "%s: rows of %lld entries are too long", what, (long long)vocab);
    if (rows == 0) return MDP_OK;
    MDP_REQUIRE(vocab > 0, "%s: rows without entries", what);
    MDP_REQUIRE(logits, "%s: null logits", what);
    MDP_REQUIRE(ld >= 0 && ld_mask >= 0, "%s: negative row stride", what);
    return MDP_OK;
}

}  // namespace

extern "C" int mdp_categorical_sample(const mdp_categorical_sample_t* a, void* stream) {
    MDP_REQUIRE(a, "null arguments");
    if (int rc = check_rows("categorical_sample", a->logits, a->rows, a->vocab, a->ld, a->dtype, a->mask, a->ld_mask)) return rc;
    if (a->rows == 0) return MDP_OK;
    MDP_REQUIRE(a->actions && a->log_prob, "categorical_sample: null output");
    MDP_REQUIRE(a->u || a->state, "categorical_sample needs uniforms or a generator state {seed, epoch}");
    SampleArgs g{a->logits, a->ld, a->mask, a->ld_mask, (int)a->vocab, a->temperature, a->top_k, a->top_p, a->min_p,
                 a->temperature_scalar, a->top_k_scalar, a->top_p_scalar, a->min_p_scalar, a->u,
                 (const unsigned long long*)a->state, a->actions, a->log_prob};
    hipStream_t s = as_stream(stream);
    const dim3 grid((unsigned)a->rows);
    switch (a->dtype) {
        case MDP_DTYPE_F32: hipLaunchKernelGGL((k_sample_row<float, 256>), grid, dim3(256), 0, s, g); break;
        case MDP_DTYPE_BF16: hipLaunchKernelGGL((k_sample_row<bf16, 256>), grid, dim3(256), 0, s, g); break;
        default: hipLaunchKernelGGL((k_sample_row<f16, 256>), grid, dim3(256), 0, s, g); break;
    }
    if (!a->u) hipLaunchKernelGGL(k_state_advance, dim3(1), dim3(1), 0, s, (unsigned long long*)a->state);
    MDP_LAUNCH_CHECK();
    return MDP_OK;
}

namespace {

// The most chunks that a row can touch: one more than it fills where rows do not all start on a chunk's boundary.
template <typename T>
int most_chunks(const void* logits, int64_t ld, int64_t rows, int vocab) {
    constexpr int N = Chunk<T>::N;
    const bool aligned = ((uintptr_t)logits & 15) == 0 && (rows == 1 || ld % N == 0);
    return (vocab + (aligned ? 0 : N - 1) + N - 1) / N;
}

// That number decides how many lanes hold a row; beyond 256 chunks (1024 floats, 2048 16-bit entries) a row is a block's.
template <typename T, bool MASK>
void launch_evaluate(const EvalArgs& g, hipStream_t s) {
    const int chunks = most_chunks<T>(g.logits, g.ld, g.rows, g.vocab);
#define SHORT(G, K)                                                                                                            \
    if (chunks <= G * K) {                                                                                                     \
        hipLaunchKernelGGL((k_evaluate_short<T, MASK, G, K>), dim3((unsigned)((g.rows + 256 / G - 1) / (256 / G))), dim3(256), 0, s, g); \
        return;                                                                                                                \
    }
    SHORT(4, 1) SHORT(4, 2) SHORT(4, 4) SHORT(8, 4) SHORT(16, 4) SHORT(32, 4) SHORT(64, 4)
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
    SHORT(4, 1) SHORT(4, 2) SHORT(4, 4) SHORT(8, 4) SHORT(16, 4) SHORT(32, 4) SHORT(64, 4)
#undef SHORT
    const int64_t most = 0x7fffffff / g.rows;          // a launch's blocks
    g.pieces = (int)std::max<int64_t>(1, std::min<int64_t>(most, (chunks + 1023) / 1024));
    hipLaunchKernelGGL((k_grad_long<T, MASK>), dim3((unsigned)(g.rows * g.pieces)), dim3(256), 0, s, g);
}

template <class F>
void by_type(int dtype, bool mask, F&& f) {
    if (dtype == MDP_DTYPE_F32) mask ? f(float{}, std::true_type{}) : f(float{}, std::false_type{});
    else if (dtype == MDP_DTYPE_BF16) mask ? f(bf16{}, std::true_type{}) : f(bf16{}, std::false_type{});
    else mask ? f(f16{}, std::true_type{}) : f(f16{}, std::false_type{});
}

}  // namespace

extern "C" int mdp_categorical_evaluate(const mdp_categorical_eval_t* a, void* stream) {
    MDP_REQUIRE(a, "null arguments");
    if (int rc = check_rows("categorical_evaluate", a->logits, a->rows, a->vocab, a->ld, a->dtype, a->mask, a->ld_mask)) return rc;
    if (a->rows == 0) return MDP_OK;
    MDP_REQUIRE(a->actions && a->log_prob && a->entropy, "categorical_evaluate: null pointer");
    EvalArgs g{a->logits, a->ld, a->mask, a->ld_mask, (int)a->vocab, a->rows, a->actions, a->temperature, a->temperature_scalar,
               a->log_prob, a->entropy, a->stats};
    hipStream_t s = as_stream(stream);
    by_type(a->dtype, a->mask, [&](auto t, auto m) { launch_evaluate<decltype(t), decltype(m)::value>(g, s); });
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
    GradArgs g{a->logits, a->ld, a->mask, a->ld_mask, (int)a->vocab, a->rows, a->actions, a->temperature, a->temperature_scalar,
               a->stats, grad_log_prob, grad_entropy, grad_logits, ld_grad, 1};
    hipStream_t s = as_stream(stream);
    by_type(a->dtype, a->mask, [&](auto t, auto m) { launch_grad<decltype(t), decltype(m)::value>(g, s); });
    MDP_LAUNCH_CHECK();
    return MDP_OK;
}

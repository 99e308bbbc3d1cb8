// Categorical distributions over the last axis of a tensor of logits: drawing an entry from given uniforms, and the
// log-probability and entropy of stored entries with their gradient by the logits.
//
// With the allowed entries A = {i : mask_i and x_i > -inf}, m = max_A x and w_i = exp((x_i - m) / T):
//   draw      order A by (x falling, i rising); keep the first k, of these the shortest prefix that holds a share p of
//             their mass, of these the entries with w_i >= min_p.  What is kept is a prefix of the order: everything up to
//             and with one entry.  With W = its mass, the answer is the first i (by index) whose running mass exceeds u W;
//             its log-probability is ln(w_i / W).
//   evaluate  s = sum_A w, t = sum_A w ln w: log p_a = ln w_a - ln s, H = ln s - t / s.
//   gradient  d/dx_i = (gl (d_ia - p_i) - ge p_i (ln p_i + H)) / T.
#pragma once
#include "mdp_device.hpp"
#include "mdp_host.hpp"
#include "elements_device.hpp"
#include <algorithm>
#include <type_traits>

namespace mdp {

constexpr float kInf = __builtin_inff();

// order-preserving key of a float; -0 and +0 are one value
MDP_DEV uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u >> 31) ? ~u : u | 0x80000000u;
}
MDP_DEV float of_key(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }

// 2^t for t <= 0 in 64 bits: t = n + f with |f| <= 1/2, and (2^f - 1) / f by the polynomial through its values at nine Chebyshev
// points of [-1/2, 1/2]; at most 3.7e-14 of the result off, and 1 at 0.  64-bit multiply-adds issue at the rate of 32-bit ones on
// this chip.  0 for -inf; a NaN is the caller's to look for.
MDP_DEV double exp2_neg(double t) {
    t = __builtin_fmax(t, -1100.0);                    // below the smallest denormal: 0
    const double n = __builtin_rint(t), f = t - n;
    double p = 1.0203121113055101e-07;
    p = fma(p, f, 1.3255224878933224e-06);
    p = fma(p, f, 1.5252686846120593e-05);
    p = fma(p, f, 0.00015403455852451632);
    p = fma(p, f, 0.0013333558179043103);
    p = fma(p, f, 0.009618129159402562);
    p = fma(p, f, 0.055504108664760424);
    p = fma(p, f, 0.2402265069581299);
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)n);
}

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
MDP_DEV float smaller(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, -kInf); }

// lane i gets lane i ^ M's value (M < 4), for M = 4 and 8 that of the lane mirrored inside 8 or 16, for M = 16 and 32 that of a
// lane in the other half of 32 or 64: what a reduction needs whose groups of M already agree
template <int M>
MDP_DEV uint32_t across_word(uint32_t x) {
    if constexpr (M == 1) return __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xf, 0xf, true);        // quad_perm 1 0 3 2
    else if constexpr (M == 2) return __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xf, 0xf, true);   // quad_perm 2 3 0 1
    else if constexpr (M == 4) return __builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, true);  // row_half_mirror
    else return __builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, true);                        // row_mirror
}
// both halves' values, the same for all lanes of a pair of rows of M lanes
template <int M>
MDP_DEV void halves(uint32_t x, uint32_t& a, uint32_t& b) {
    if constexpr (M == 16) { const auto q = __builtin_amdgcn_permlane16_swap(x, x, false, false); a = q[0]; b = q[1]; }
    else { const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false); a = q[0]; b = q[1]; }
}
template <int M, typename V, class F>
MDP_DEV V over_step(V v, F&& f) {
    constexpr int L = sizeof(V) / 4;
    struct Words { uint32_t w[L]; } x = __builtin_bit_cast(Words, v), y;
    if constexpr (M < 16) {
#pragma unroll
        for (int i = 0; i < L; ++i) y.w[i] = across_word<M>(x.w[i]);
        return f(v, __builtin_bit_cast(V, y));
    } else {
#pragma unroll
        for (int i = 0; i < L; ++i) halves<M>(x.w[i], x.w[i], y.w[i]);
        return f(__builtin_bit_cast(V, x), __builtin_bit_cast(V, y));
    }
}
template <int G, typename V, class F>
MDP_DEV V over_group(V v, F&& f) {                     // every lane of a group of G gets the result
    if constexpr (G > 1) v = over_step<1>(v, f);
    if constexpr (G > 2) v = over_step<2>(v, f);
    if constexpr (G > 4) v = over_step<4>(v, f);
    if constexpr (G > 8) v = over_step<8>(v, f);
    if constexpr (G > 16) v = over_step<16>(v, f);
    if constexpr (G > 32) v = over_step<32>(v, f);
    return v;
}
template <int G>
MDP_DEV float group_max(float v) { return over_group<G>(v, [](float a, float b) { return larger(a, b); }); }
template <int G, typename V>
MDP_DEV V group_sum(V v) { return over_group<G>(v, [](V a, V b) { return a + b; }); }

// the value O lanes below in a row of 16, 0 where there is none
template <int O, typename V>
MDP_DEV V from_below(V v) {
    constexpr int L = sizeof(V) / 4;
    struct Words { uint32_t w[L]; } x = __builtin_bit_cast(Words, v);
#pragma unroll
    for (int i = 0; i < L; ++i) x.w[i] = __builtin_amdgcn_update_dpp(0, x.w[i], 0x110 + O, 0xf, 0xf, false);     // row_shr
    return __builtin_bit_cast(V, x);
}
template <typename V>
MDP_DEV V of_lane(V v, int lane) {                     // uniform lane
    constexpr int L = sizeof(V) / 4;
    struct Words { uint32_t w[L]; } x = __builtin_bit_cast(Words, v);
#pragma unroll
    for (int i = 0; i < L; ++i) x.w[i] = __builtin_amdgcn_readlane(x.w[i], lane);
    return __builtin_bit_cast(V, x);
}
// sum over the lanes of the group up to and with this one
template <int G, typename V>
MDP_DEV V group_scan(V v) {
    const int at = threadIdx.x & 63, lane = at % G;
    V up = from_below<1>(v);
    v += lane >= 1 ? up : V(0);
    up = from_below<2>(v);
    if constexpr (G > 2) v += lane >= 2 ? up : V(0);
    up = from_below<4>(v);
    if constexpr (G > 4) v += lane >= 4 ? up : V(0);
    up = from_below<8>(v);
    if constexpr (G > 8) v += lane >= 8 ? up : V(0);
    if constexpr (G == 32) v += lane >= 16 ? (at >= 32 ? of_lane(v, 47) : of_lane(v, 15)) : V(0);
    if constexpr (G == 64) {
        const V a = of_lane(v, 15), b = of_lane(v, 31), c = of_lane(v, 47);
        v += at < 16 ? V(0) : at < 32 ? a : at < 48 ? a + b : a + b + c;
    }
    return v;
}

// The most chunks that a row can touch: one more than it fills where rows do not all start on a chunk's boundary.
template <typename T>
int most_chunks(const void* logits, int64_t ld, int64_t rows, int vocab) {
    constexpr int N = Chunk<T>::N;
    const bool aligned = ((uintptr_t)logits & 15) == 0 && (rows == 1 || ld % N == 0);
    return (vocab + (aligned ? 0 : N - 1) + N - 1) / N;
}

// log2(e) / T in 64 bits: a NaN for a temperature that is negative or NaN, kGreedy for one below the smallest normal number, never
// 0, so that -inf times it stays -inf.  A 64-bit division takes some forty instructions: for one temperature the host makes it.
constexpr double kGreedy = 1e300;
__host__ __device__ inline double rate_of(float t) {
    if (!(t >= 0.0f)) return __builtin_nan("");
    if (t < 1.17549435e-38f) return kGreedy;
    const double c = 1.4426950408889634 / (double)t;
    return c > 1e-300 ? c : 1e-300;
}

struct SampleArgs {
    const void* logits; int64_t ld;
    const uint8_t* mask; int64_t ld_mask;
    int vocab; int64_t rows;
    int64_t row0;                                      // of the call's rows the launch's first
    const float* temperature; const int* top_k; const float* top_p; const float* min_p;
    double rate;                                       // rate_of() the temperature that all rows share
    int top_k_s; float top_p_s; float min_p_s;
    const float* u; const unsigned long long* state;
    int64_t* actions; float* log_prob;
};

// defined for each element type in a file of its own (categorical_sample_*.hip), compiled side by side
template <typename T, bool MASK>
void launch_sample(const SampleArgs& g, hipStream_t s);

}  // namespace mdp

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

// -- evaluation -------------------------------------------------------------------------------------------------------
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
};

// ln w, held at or above -200 (where w is 0 in 32 bits) so that 0 * ln 0 is 0; a NaN stays one
MDP_DEV float log_weight(float x, float m, float inv_t) {
    const float d = (x - m) * inv_t;
    return d < -200.0f ? -200.0f : d;
}

// running (m, s, t) of a softmax: s = sum w, t = sum w ln w about the largest entry so far
struct Running {
    float m, s, t;
    MDP_DEV static Running none() { return Running{-__FLT_MAX__, 0.0f, 0.0f}; }
    MDP_DEV void move(float to, float inv_t) {        // about another maximum >= m
        const float d = log_weight(m, to, inv_t), f = expf(d);
        t = f * (t + d * s);
        s *= f;
        m = to;
    }
    MDP_DEV void add(float x, float inv_t) {
        if (x > m) move(x, inv_t);
        const float d = log_weight(x, m, inv_t), e = expf(d);
        s += e;
        t += e * d;
    }
    MDP_DEV void join(Running o, float inv_t) {
        const float to = fmaxf(m, o.m);
        move(to, inv_t);
        o.move(to, inv_t);
        s += o.s;
        t += o.t;
    }
};

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void k_evaluate_row(EvalArgs g) {
    __shared__ Running part[THREADS / 64];
    const int64_t row = blockIdx.x;
    const int V = g.vocab, tid = threadIdx.x;
    const T* x = (const T*)g.logits + row * g.ld;
    const uint8_t* mask = g.mask ? g.mask + row * g.ld_mask : nullptr;
    const float temp = g.temperature ? g.temperature[row] : g.temperature_s;
    const float inv_t = temp > 0.0f ? 1.0f / temp : __builtin_nanf("");
    Running r = Running::none();
    for (int i = tid; i < V; i += THREADS)
        if (!mask || mask[i]) r.add(to_f32(x[i]), inv_t);
    for (int o = 32; o > 0; o >>= 1) {
        Running q;
        q.m = __shfl_xor(r.m, o); q.s = __shfl_xor(r.s, o); q.t = __shfl_xor(r.t, o);
        r.join(q, inv_t);
    }
    if ((tid & 63) == 0) part[tid >> 6] = r;
    __syncthreads();
    if (tid) return;
    for (int w = 1; w < THREADS / 64; ++w) r.join(part[w], inv_t);
    const float log_s = logf(r.s);
    const float h = r.s == 0.0f ? 0.0f : log_s - r.t / r.s;
    const int64_t a = g.actions[row];
    float lp;
    if (a == -1) lp = 0.0f;
    else if (a < 0 || a >= V) lp = __builtin_nanf("");
    else if (mask && !mask[a]) lp = r.s == r.s ? -kInf : r.s;
    else lp = (to_f32(x[a]) - r.m) * inv_t - log_s;
    g.log_prob[row] = lp;
    g.entropy[row] = h;
    if (g.stats) {
        g.stats[3 * row] = r.m;
        g.stats[3 * row + 1] = log_s;
        g.stats[3 * row + 2] = h;
    }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void k_evaluate_grad(GradArgs g) {
    const int64_t row = blockIdx.x;
    const int V = g.vocab;
    const T* x = (const T*)g.logits + row * g.ld;
    T* out = (T*)g.grad + row * g.ld_grad;
    const uint8_t* mask = g.mask ? g.mask + row * g.ld_mask : nullptr;
    const float temp = g.temperature ? g.temperature[row] : g.temperature_s;
    const float inv_t = temp > 0.0f ? 1.0f / temp : __builtin_nanf("");
    const float m = g.stats[3 * row], log_s = g.stats[3 * row + 1], h = g.stats[3 * row + 2];
    const int64_t a = g.actions[row];
    float gl = g.grad_log_prob ? g.grad_log_prob[row] : 0.0f;
    const float ge = g.grad_entropy ? g.grad_entropy[row] : 0.0f;
    if (a == -1) gl = 0.0f;
    else if (a < 0 || a >= V) gl = __builtin_nanf("");
    const bool empty = log_s == -kInf;
    for (int i = threadIdx.x; i < V; i += THREADS) {
        float y = 0.0f;
        const float v = to_f32(x[i]);
        if (!(mask && !mask[i]) && v != -kInf && !empty) {
            const float lw = log_weight(v, m, inv_t), lp = lw - log_s, p = expf(lp);
            y = -p * (gl + ge * (lp + h));
            if (i == a) y += gl;
            y *= inv_t;
        }
        from_f32(y, out[i]);
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

extern "C" int mdp_categorical_evaluate(const mdp_categorical_eval_t* a, void* stream) {
    MDP_REQUIRE(a, "null arguments");
    if (int rc = check_rows("categorical_evaluate", a->logits, a->rows, a->vocab, a->ld, a->dtype, a->mask, a->ld_mask)) return rc;
    if (a->rows == 0) return MDP_OK;
    MDP_REQUIRE(a->actions && a->log_prob && a->entropy, "categorical_evaluate: null pointer");
    EvalArgs g{a->logits, a->ld, a->mask, a->ld_mask, (int)a->vocab, a->rows, a->actions, a->temperature, a->temperature_scalar,
               a->log_prob, a->entropy, a->stats};
    hipStream_t s = as_stream(stream);
    const dim3 grid((unsigned)a->rows);
    switch (a->dtype) {
        case MDP_DTYPE_F32: hipLaunchKernelGGL((k_evaluate_row<float, 256>), grid, dim3(256), 0, s, g); break;
        case MDP_DTYPE_BF16: hipLaunchKernelGGL((k_evaluate_row<bf16, 256>), grid, dim3(256), 0, s, g); break;
        default: hipLaunchKernelGGL((k_evaluate_row<f16, 256>), grid, dim3(256), 0, s, g); break;
    }
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
               a->stats, grad_log_prob, grad_entropy, grad_logits, ld_grad};
    hipStream_t s = as_stream(stream);
    const dim3 grid((unsigned)a->rows);
    switch (a->dtype) {
        case MDP_DTYPE_F32: hipLaunchKernelGGL((k_evaluate_grad<float, 256>), grid, dim3(256), 0, s, g); break;
        case MDP_DTYPE_BF16: hipLaunchKernelGGL((k_evaluate_grad<bf16, 256>), grid, dim3(256), 0, s, g); break;
        default: hipLaunchKernelGGL((k_evaluate_grad<f16, 256>), grid, dim3(256), 0, s, g); break;
    }
    MDP_LAUNCH_CHECK();
    return MDP_OK;
}

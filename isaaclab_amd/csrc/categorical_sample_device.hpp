// Drawing an entry of every row of logits: see the top of categorical_device.hpp for what is drawn.
#pragma once
#include "categorical_device.hpp"

namespace mdp {

// -- drawing ------------------------------------------------------------------------------------------------------------
// Everything that decides is in 64 bits, which cost what 32 bits cost on this chip's vector units: weights, their sums and the
// comparisons with u W and p S.  Sums in 32 bits only ever bound what has to be looked at.
constexpr uint32_t kStream = 0x43415447u;

// A row's settings.  Temperature 0 (and what is below the smallest normal number) is one entry of the largest logit, with weights
// that are 1 there and 0 elsewhere.
struct Settings {
    double c;                                          // log2(e) / T; a NaN for a temperature that is negative or NaN
    int k;                                             // 0: no limit
    float p, mp;                                       // p = 1, mp = 0: no limit
    double u;
    MDP_DEV Settings(const SampleArgs& g, int64_t row) {
        k = g.top_k ? g.top_k[row] : g.top_k_s;
        float pf = g.top_p ? g.top_p[row] : g.top_p_s, mf = g.min_p ? g.min_p[row] : g.min_p_s;
        if (k < 0) k = 0;
        p = pf < 1.0f ? (pf > 0.0f ? pf : 0.0f) : 1.0f;
        mp = mf > 0.0f ? (mf < 1.0f ? mf : 1.0f) : 0.0f;
        c = g.temperature ? rate_of(g.temperature[row]) : g.rate;
        if (c == kGreedy) { k = 1; p = 1.0f; mp = 0.0f; }
        float uf = g.u ? g.u[row] : u01(rng4(g.state[0], g.state[1], kStream, (uint64_t)(g.row0 + row)).x);
        u = uf > 0.0f ? (uf < 0.99999994f ? (double)uf : 0.99999994039535522) : 0.0;
    }
    MDP_DEV float c32() const { return (float)fmax(fmin(c, 3e38), 1e-38); }     // -inf * c and 0 * c stay what they are
    MDP_DEV bool all() const { return k == 0 && p == 1.0 && mp == 0.0; }
    MDP_DEV double weight(float x, float m) const { return exp2_neg(((double)x - (double)m) * c); }
};

// ln(w / mass), w the weight of x: from x itself where w is a denormal or near one and holds fewer bits than the result
constexpr double kLight = 1e-290;
MDP_DEV float log_share_of_light(float x, float m, double c, double mass) {
    return (float)(((double)x - (double)m) * c * 0.6931471805599453 - log(mass));
}

// an entry as a word that rises in the order (value falling, place rising)
MDP_DEV uint64_t word_of(float x, int place) { return (uint64_t)(~key_of(x)) << 32 | (uint32_t)place; }
MDP_DEV float value_of(uint64_t word) { return of_key(~(uint32_t)(word >> 32)); }

// Nothing that is computed from x before is kept for after this: sixteen entries' worth of it would not fit the registers
template <typename V>
MDP_DEV void anew(V& x) { asm volatile("" : "+v"(x)); }

}  // namespace mdp

#include "categorical_border_device.hpp"

namespace mdp {

// Shared memory that lanes of one wave pass to each other: no barrier, only the order of its accesses
MDP_DEV void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Rows of up to G K chunks, 16 entries a lane: G lanes of a wave, or a block of G = 128 or 256, hold a row and its weights in
// registers.  Groups of a wave go through their loops together until the last is done.
//
// Bound by instructions: 49152 x 256 float32 with top_p takes 43 us, 1665 vector instructions for a wave's four rows (300 of them the
// weights), where the 50 MB are 11 us at the copy rate; uncut it takes 22.  Searching the border by halving the value range, sixteen
// compares and 64-bit adds a step, took 71 where this took 44.  Entries and weights leave four waves a SIMD, and their 128 registers
// do not always hold all: up to 34 are spilled, most by rows of up to 64 entries, none by rows of one wave each.  With five waves (96
// registers) what spills costs more: 53.
template <typename T, int G, int K>
struct ShortRow {
    static constexpr int N = Chunk<T>::N, size = G, capacity = G;
    static constexpr int per_lane = G < 8 ? 16 : G <= 32 ? 8 : G <= 64 ? 4 : 256 / G;      // at most 256 buckets: their numbers are bytes
    static constexpr int W = G / 64;                   // waves of a block that holds one row
    static constexpr float window = 14.0f;
    static constexpr bool total_known = true;
    struct Listed { uint64_t word; double value; };      // the word rises in the order
    struct Shared { Listed list[G]; double d[W ? W : 1]; uint32_t u[W ? W : 1]; uint32_t hist[per_lane * G]; int n; float top; };
    float x[K][N];
    double w[K][N];
    int rank, shift;                                   // this lane's number; the row's shift
    uint32_t* hist;
    Shared* sh;
    bool good;
    float m, bottom;
    const Settings* s;

    MDP_DEV int place(int k, int e) const { return (k * G + rank) * N - shift + e; }
    template <class F>
    MDP_DEV void each(F&& f) const {
        int base = rank * N - shift;
        anew(base);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < N; ++e) f(x[k][e], base + k * G * N + e, [&] { return w[k][e]; });
    }
    MDP_DEV double weight(float v) const { return s->weight(v, m); }
    // the waves' values, for a block
    template <typename V, class F>
    MDP_DEV void exchange(V v, bool mine, F&& f) const {
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if (mine) {
            if constexpr (sizeof(V) == 8) sh->d[wave] = v;
            else sh->u[wave] = __builtin_bit_cast(uint32_t, v);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if constexpr (sizeof(V) == 8) f(i, sh->d[i]);
            else f(i, __builtin_bit_cast(V, sh->u[i]));
        }
    }
    // what is the same for all lanes of a wave, in scalar registers
    template <typename V>
    MDP_DEV static V shared_by_all(V v) {
        if constexpr (G < 64) return v;
        else return of_lane(v, 0);
    }
    template <typename V>
    MDP_DEV V sum(V v) const {
        if constexpr (G <= 64) return shared_by_all(group_sum<G>(v));
        V all = V(0);
        exchange(group_sum<64>(v), (threadIdx.x & 63) == 0, [&](int, V o) { all += o; });
        return shared_by_all(all);
    }
    MDP_DEV float highest(float v) const {
        if constexpr (G <= 64) return shared_by_all(group_max<G>(v));
        float all = -kInf;
        exchange(group_max<64>(v), (threadIdx.x & 63) == 0, [&](int, float o) { all = larger(o, all); });
        return shared_by_all(all);
    }
    MDP_DEV float lowest(float v) const { return -highest(-v); }
    template <typename V>
    MDP_DEV V scan(V v) const {
        if constexpr (G <= 64) return group_scan<G>(v);
        v = group_scan<64>(v);
        V before = V(0);
        exchange(v, (threadIdx.x & 63) == 63, [&](int i, V o) { before += i < (int)(threadIdx.x >> 6) ? o : V(0); });
        return before + v;
    }
    // the votes of a group that is not a block, from its first lane on
    MDP_DEV uint64_t votes(bool v) const {
        const uint64_t all = __ballot(v) >> ((threadIdx.x & 63) - rank);
        return G == 64 ? all : all & ((1ull << (G & 63)) - 1ull);
    }
    // the group's first (last) lane of which v holds, -1 if none
    MDP_DEV int first_of(bool v) const {
        if constexpr (G <= 64) return __ffsll((unsigned long long)votes(v)) - 1;
        const int at = (int)lowest(v ? (float)rank : (float)G);
        return at < G ? at : -1;
    }
    MDP_DEV int last_of(bool v) const {
        if constexpr (G <= 64) return 63 - __clzll((long long)votes(v));
        return (int)highest(v ? (float)rank : -1.0f);
    }
    MDP_DEV bool some(bool v) const {
        if constexpr (G <= 64) return votes(v) != 0;
        else return __syncthreads_or(v) != 0;
    }
    MDP_DEV void sync() const {
        if constexpr (G <= 64) wave_sync();
        else __syncthreads();
    }
    // over the lanes that run a loop in step: a wave's groups; a block's lanes all say the same
    MDP_DEV bool any(bool v) const {
        if constexpr (G <= 64) return __any(v && good) != 0;
        else return v && good;
    }
    // the buckets of the entries, a byte each
    uint32_t ids[4];
    template <class B, class F>
    MDP_DEV void sort_in(B&& bucket, F&& f) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t four = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int k = (4 * q + e) / N, l = (4 * q + e) % N;
                const int b = bucket(x[k][l]);
                four |= (uint32_t)b << 8 * e;
                f(b, [&] { return w[k][l]; });
            }
            ids[q] = four;
        }
    }
    template <class B, class F>
    MDP_DEV void each_sorted(B&&, F&& f) const {
        int base = rank * N - shift;
        anew(base);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int k = i / N, l = i % N;
            f(x[k][l], base + k * G * N + l, [&] { return w[k][l]; }, (int)(ids[i / 4] >> 8 * (i % 4) & 0xffu));
        }
    }
    MDP_DEV void clear_list() const { if (rank == 0) sh->n = 0; }
    MDP_DEV int listed() const { return shared_by_all(sh->n); }
    template <bool COUNT>
    MDP_DEV void put(float v, int i, double value) const {
        anew(v);
        const int to = atomicAdd(&sh->n, 1);           // in any order: what is asked of the list goes by value and place
        if (to < capacity) sh->list[to] = Listed{word_of(v, i), value};
    }
    template <bool COUNT>
    MDP_DEV Border last_kept(int n, double above, double aim) const {
        const bool in = rank < n;
        const Listed mine = in ? sh->list[rank] : Listed{~0ull, 0.0};
        int order = 0;
        for (int j = 0; G <= 64 ? __any(j < n) != 0 : j < n; ++j) order += j < n && sh->list[j].word < mine.word;
        sync();
        if (in) sh->list[order] = mine;                // in order now, however they came
        sync();
        const Listed at = in ? sh->list[rank] : Listed{~0ull, 0.0};
        const double before = above + (scan(at.value) - at.value);
        int kept = sum((int)(in && before < aim));
        kept = kept ? kept : 1;
        const bool me = in && rank == kept - 1;
        return Border{highest(me ? value_of(at.word) : -kInf), sum(me ? (int)(uint32_t)at.word : 0)};
    }
    MDP_DEV int nth_equal(float v, int r) const {
        int seen = 0, at = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            int equal = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) equal += x[k][e] == v;
            const int upto = scan(equal);
            int rank_of = seen + upto - equal;
            seen += sum(equal);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                rank_of += x[k][e] == v;
                if (x[k][e] == v && rank_of == r) at = place(k, e);
            }
        }
        return sum(at);
    }
};

template <typename T, bool MASK, int G, int K>
__global__ __launch_bounds__(G > 64 ? G : 256, 4) void k_sample_short(SampleArgs g) {
    using R = ShortRow<T, G, K>;
    constexpr int N = Chunk<T>::N, ROWS = G > 64 ? 1 : 256 / G;
    __shared__ typename R::Shared shared[ROWS];
    // of a row that takes whole waves, what its lanes share stands in scalar registers
    const int in_block = threadIdx.x / G;
    const int64_t mine = (int64_t)blockIdx.x * ROWS + (G < 64 ? in_block : __builtin_amdgcn_readfirstlane(in_block));
    const int64_t row = mine < g.rows ? mine : g.rows - 1;             // lanes without a row of their own repeat the last
    const int lane = threadIdx.x % G;
    const Row<T> r(g.logits, g.ld, g.mask, g.ld_mask, g.vocab, row);
    R q;
#pragma unroll
    for (int k = 0; k < K; ++k) r.template load<MASK>(k * G + lane, q.x[k]);
    const Settings s(g, row);
    float m = -kInf;
    bool broken = false;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            broken |= !(q.x[k][e] < kInf);
            m = larger(q.x[k][e], m);
        }
    q.rank = lane;
    q.shift = r.shift;
    q.sh = &shared[threadIdx.x / G];
    q.hist = q.sh->hist;
    q.s = &s;
    m = q.highest(m);
    if (lane == 0) q.sh->top = m;                      // for the end, where no register holds it: the same wave reads it, or behind barriers
    broken = q.some(broken) || s.c != s.c;
    const bool empty = m == -kInf;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e) q.w[k][e] = s.weight(q.x[k][e], empty ? 0.0f : m);
    q.good = !broken && !empty;
    q.m = m;
    if (q.any(!s.all())) {
        if (q.any(s.k > 0 || s.p < 1.0)) {
            double total = 0.0;
            int allowed = 0;
            q.bottom = m;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    total += q.w[k][e];
                    q.bottom = smaller(q.x[k][e] > -kInf ? q.x[k][e] : m, q.bottom);
                }
            total = q.sum(total);
            q.bottom = q.lowest(q.bottom);
            if (q.any(s.k > 0)) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int e = 0; e < N; ++e) allowed += q.x[k][e] > -kInf;
                allowed = q.sum(allowed);
            }
            const Border b = border_of(q, s, m, total, allowed);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < N; ++e) q.w[k][e] = b.keeps(q.x[k][e], q.place(k, e)) ? q.w[k][e] : 0.0;
        }
        if (q.any(s.mp > 0.0)) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < N; ++e) q.w[k][e] = q.w[k][e] >= s.mp ? q.w[k][e] : 0.0;
        }
    }
    // masses by chunk index; the chunk row k that holds the aim, the lane in it, the entry in that
    double part[K], mass = 0.0, sums[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        part[k] = 0.0;
#pragma unroll
        for (int e = 0; e < N; ++e) part[k] += q.w[k][e];
        sums[k] = q.sum(part[k]);
        mass += sums[k];
    }
    const double aim = s.u * mass;
    double before = 0.0, run = 0.0;
    int pick = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (sums[k] > 0.0 && run <= aim) { pick = k; before = run; }
        run += sums[k];
    }
    double v[N], own = 0.0;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = 0.0;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (k == pick) {
            own = part[k];
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = q.w[k][e];
        }
    const double upto = before + q.scan(own);
    // rounding may leave the aim at the end of the last mass: its lane, and its last entry, then
    int winner = q.first_of(own > 0.0 && upto > aim);
    const int end = q.last_of(own > 0.0);
    if (winner < 0) winner = end < 0 ? 0 : end;
    if (lane != winner || mine >= g.rows) return;
    double sum = upto - own, found_w = 1.0;
    int found = -1;
    bool open = true;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        sum += v[e];
        if (open && v[e] > 0.0) {
            found = q.place(pick, e);
            found_w = v[e];
            open = !(sum > aim);
        }
    }
    g.actions[mine] = q.good ? found : -1;
    g.log_prob[mine] = q.good ? (float)log(found_w / mass) : broken ? __builtin_nanf("") : 0.0f;
    if (__builtin_expect(q.good && found_w < kLight, 0)) {      // what it takes is read again, and kept in no register until here
        const Row<T> again(g.logits, g.ld, g.mask, g.ld_mask, g.vocab, mine);
        g.log_prob[mine] = log_share_of_light(to_f32(again.x[found]), q.sh->top, Settings(g, mine).c, mass);
    }
}

// Longer rows: a block a row.  Each wave owns a contiguous piece of the row, so that running sums follow the index; of it every
// lane holds up to H chunks in registers, and what does not fit is read again for each question.
//
// A question over a long row is dear (131072 bfloat16 entries: 9 us of a CU in 32 bits), so what k, p and min_p keep is looked for
// among few candidates: the threads' own largest entries are a part of the row, so a value above which THEY already are k, or
// already hold a share p of the row's mass, is not above the border.  The entries from there on -- a few more than are kept -- are
// listed and sorted, and everything exact happens on them.  Where no such value exists or too many entries lie above it (flat rows),
// the border is searched over the whole row.
//
// 1024 x 131072 bfloat16 with top_p and min_p: 140 us for 268 MB (57 at the copy rate).  A row fills the registers of a CU, so while
// it arrives (13 us of its share of the memory rate) nothing is left to do but its maxima and 32-bit mass, and the 15 us after it --
// bound, list, sort -- load nothing.  Uncut rows of that size: 160 us, 64-bit weights of every entry; rows that the list leaves:
// 642 us (scale 0.5), one pass for the list and four over the row, most of it from the caches.
template <typename T, bool MASK, int THREADS, int H>
struct LongRow {
    static constexpr int N = Chunk<T>::N, W = THREADS / 64, size = THREADS, capacity = THREADS;
    static constexpr int per_lane = 4;
    static constexpr float window = 24.0f;
    static constexpr bool total_known = false;
    // What the mass in 32 bits may be off, as a share: 2^-16 for the weights (three roundings of an exponent of 20 binary orders, the
    // orders that hold the mass of 2^18 entries, make 2.4e-6, sums of chunks as much again), and two roundings for each time that a
    // thread's largest entry changed.
    MDP_DEV double rough() const { return 1.53e-5 + 2.4e-7 * (double)steps; }
    struct Shared {
        double d[W + 1];
        int n[W + 1];
        float f[W];
        union {
            struct { float top[THREADS]; } maxima;
            struct { uint64_t key[THREADS]; double value[THREADS]; } list;
        };
        uint32_t hist[per_lane * THREADS];
        Border border;
        float bound;
        int found, last, listed;
    };
    const Row<T> r;
    Shared& sh;
    const Settings& s;
    const int tid, lane, wave, steps;                  // chunks of a wave: (wave steps + step) 64 + lane
    const int rank;
    uint32_t* const hist;
    Chunk<T> held[H ? H : 1];
    float m, bottom;

    MDP_DEV LongRow(const SampleArgs& g, int64_t row, const Settings& settings, Shared& shared)
        : r(g.logits, g.ld, g.mask, g.ld_mask, g.vocab, row), sh(shared), s(settings), tid(threadIdx.x), lane(threadIdx.x & 63),
          wave(threadIdx.x >> 6), steps((r.chunks() + THREADS - 1) / THREADS), rank(threadIdx.x), hist(shared.hist) {
#pragma unroll
        for (int h = 0; h < H; ++h) held[h] = chunk(wave, h);
    }
    MDP_DEV int place(int of, int step) const { return ((of * steps + step) * 64 + lane) * N - r.shift; }
    MDP_DEV Chunk<T> chunk(int of, int step) const {   // of wave `of`'s piece
        const int j = (of * steps + step) * 64 + lane;
        if (step >= steps || j >= r.chunks()) return Chunk<T>::lowest();
        if (!MASK && r.full(j)) return r.chunk(j);
        float v[N];
        r.template load<MASK>(j, v);
        return Chunk<T>::of(v);
    }
    // f(step, entries) for each of this thread's chunks
    template <class F>
    MDP_DEV void each_chunk(F&& f) const {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if (h < steps) {
                float v[N];
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = held[h].at(e);
                f(h, v);
            }
            __builtin_amdgcn_sched_barrier(0);         // one chunk's arithmetic at a time: all of them at once would not fit the registers
        }
        each_chunk_again(f, H);
    }
    // the same with every chunk read again: a loop, where the registers would need the code once for each chunk that they hold
    template <class F>
    MDP_DEV void each_chunk_again(F&& f, int from = 0) const {
        Chunk<T> next = chunk(wave, from);
        for (int h = from; h < steps; ++h) {
            const Chunk<T> q = next;
            next = chunk(wave, h + 1);                 // on its way while this one is worked on
            float v[N];
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = q.at(e);
            f(h, v);
        }
    }
    // what find_border asks for
    template <class F>
    MDP_DEV void each(F&& f) const {
        each_chunk_again([&](int step, const float (&v)[N]) {
            const int i0 = place(wave, step);
#pragma unroll
            for (int e = 0; e < N; ++e) f(v[e], i0 + e, [&] { return s.weight(v[e], m); });
        });
    }
    MDP_DEV double weight(float x) const { return s.weight(x, m); }
    MDP_DEV void sync() const { __syncthreads(); }
    MDP_DEV bool any(bool v) const { return v; }       // the same for the whole block
    MDP_DEV double sum(double v) const { return block_sum(v); }
    MDP_DEV int sum(int v) const { return block_sum(v); }
    MDP_DEV float highest(float v) const { return block_max(v); }
    MDP_DEV float lowest(float v) const { return -block_max(-v); }
    MDP_DEV uint32_t scan(uint32_t v) const {
        v = group_scan<64>(v);
        __syncthreads();
        if (lane == 63) sh.n[wave] = (int)v;
        __syncthreads();
        for (int w = 0; w < wave; ++w) v += (uint32_t)sh.n[w];
        return v;
    }

    MDP_DEV double block_sum(double v) const {
        v = group_sum<64>(v);
        __syncthreads();
        if (lane == 0) sh.d[wave] = v;
        __syncthreads();
        double t = 0.0;
        for (int w = 0; w < W; ++w) t += sh.d[w];
        return t;
    }
    MDP_DEV int block_sum(int v) const {
        v = group_sum<64>(v);
        __syncthreads();
        if (lane == 0) sh.n[wave] = v;
        __syncthreads();
        int t = 0;
        for (int w = 0; w < W; ++w) t += sh.n[w];
        return t;
    }
    MDP_DEV float block_max(float v) const {
        v = group_max<64>(v);
        __syncthreads();
        if (lane == 0) sh.f[wave] = v;
        __syncthreads();
        float t = sh.f[0];
        for (int w = 1; w < W; ++w) t = larger(sh.f[w], t);
        return t;
    }
    // sum over the threads up to and with this one; `all` over every thread
    MDP_DEV double block_scan(double v, double& all) const {
        v = group_scan<64>(v);
        __syncthreads();
        if (lane == 63) sh.d[wave] = v;
        __syncthreads();
        double before = 0.0;
        all = 0.0;
        for (int w = 0; w < W; ++w) {
            if (w < wave) before += sh.d[w];
            all += sh.d[w];
        }
        return before + v;
    }
    MDP_DEV double exact_mass() const {
        double t = 0.0;
        each([&](float, int, auto&& w) { t += w(); });
        return block_sum(t);
    }

    // A value not above the border, from the threads' largest entries, or -inf.  `mass`: the row's, in 32 bits.
    MDP_DEV float bound_of(float top, float mass) const {
        __syncthreads();
        sh.maxima.top[tid] = top;
        __syncthreads();
        if (wave == 0) {
            float v[W], w[W];
            const float c = s.c32();
#pragma unroll
            for (int i = 0; i < W; ++i) {
                v[i] = sh.maxima.top[i * 64 + lane];
                w[i] = __builtin_amdgcn_exp2f(larger((v[i] - m) * c, -300.0f));
            }
            const float aim = (float)s.p * mass * (1.0001f + 1e-6f * (float)steps);    // above p S whatever 32 bits made of the sums
            float bound = -kInf;
            if (s.k > 0 || s.p < 1.0) {
                const auto enough = [&](float from) {
                    float q = 0.0f;
#pragma unroll
                    for (int i = 0; i < W; ++i) q += v[i] >= from ? (s.k > 0 ? 1.0f : w[i]) : 0.0f;
                    q = group_sum<64>(q);
                    return s.k > 0 ? q >= (float)s.k : q >= aim;
                };
                float lo = (float)((double)m - 60.0 / s.c), hi = m;
                if (enough(lo)) {
                    // ten halvings: 60 binary orders of magnitude down to 1/17 of one, a few entries more than needed
                    for (int it = 0; it < 10; ++it) {
                        const float mid = 0.5f * lo + 0.5f * hi;
                        if (enough(mid)) lo = mid; else hi = mid;
                    }
                    bound = lo;
                }
            }
            if (s.k == 0 && s.mp > 0.0) {
                // lighter than min_p: never kept
                const float light = (float)((double)m + log2((double)s.mp) / s.c);
                bound = larger(light - 1e-3f * fabsf(light) - 1e-3f, bound);
            }
            if (lane == 0) sh.bound = bound;
        }
        __syncthreads();
        return sh.bound;
    }

    // Lists the entries >= bound as words, in any order; their number, of which no more than THREADS are listed.
    MDP_DEV int gather(float bound) const {
        __syncthreads();
        clear_list();
        __syncthreads();
        each_chunk([&](int step, const float (&v)[N]) {
            const int i0 = place(wave, step);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (v[e] >= bound) put<true>(v[e], i0 + e, 1.0);
        });
        __syncthreads();
        return sh.listed;
    }
    template <class B, class F>
    MDP_DEV void sort_in(B&& bucket, F&& f) const {
        each([&](float x, int, auto&& w) { f(bucket(x), w); });
    }
    template <class B, class F>
    MDP_DEV void each_sorted(B&& bucket, F&& f) const {
        each([&](float x, int i, auto&& w) { f(x, i, w, bucket(x)); });
    }
    MDP_DEV void clear_list() const { if (tid == 0) sh.listed = 0; }
    MDP_DEV int listed() const { return sh.listed; }
    template <bool COUNT>
    MDP_DEV void put(float x, int i, double) const {
        const int to = atomicAdd(&sh.listed, 1);       // in any order: it is sorted
        if (to < capacity) sh.list.key[to] = word_of(x, i);
    }
    template <bool COUNT>
    MDP_DEV Border last_kept(int n, double above, double aim) const {
        const uint64_t word = tid < n ? sh.list.key[tid] : ~0ull;
        __syncthreads();
        const uint64_t sorted = sort(word, n);
        const double v = tid < n ? (COUNT ? 1.0 : s.weight(value_of(sorted), m)) : 0.0;
        double all;
        const double before = above + (block_scan(v, all) - v);
        const int kept = max(1, block_sum((int)(tid < n && before < aim)));
        if (tid == kept - 1) sh.border = Border{value_of(sorted), (int)(uint32_t)sorted};
        __syncthreads();
        return sh.border;
    }
    MDP_DEV int nth_equal(float x, int r) const {
        int mine = 0;
        each([&](float v, int, auto&&) { mine += v == x; });
        mine = group_sum<64>(mine);
        __syncthreads();
        if (lane == 0) sh.n[wave] = mine;
        __syncthreads();
        int seen = 0;
        for (int w = 0; w < wave; ++w) seen += sh.n[w];
        if (seen < r && seen + mine >= r)
            each_chunk_again([&](int step, const float (&v)[N]) {
                int equal = 0;
#pragma unroll
                for (int e = 0; e < N; ++e) equal += v[e] == x;
                const int upto = group_scan<64>(equal);
                int rank_of = seen + upto - equal;
                seen += of_lane(upto, 63);
                const int i0 = place(wave, step);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    rank_of += v[e] == x;
                    if (v[e] == x && rank_of == r) sh.found = i0 + e;
                }
            });
        __syncthreads();
        return sh.found;
    }

    // sorts the threads' words, rising with the thread
    MDP_DEV uint64_t sort(uint64_t v, int n) const {
        int padded = 64;
        while (padded < n) padded <<= 1;
        const bool works = tid < padded;               // waves beyond only keep the barriers
        for (int size = 2; size < 2 * padded; size <<= 1)
            for (int stride = size >> 1; stride; stride >>= 1) {
                if (stride >= 64) {
                    __syncthreads();
                    if (works) sh.list.key[tid] = v;
                    __syncthreads();
                }
                if (!works) continue;
                const uint64_t o = stride < 64 ? (uint64_t)__shfl_xor((unsigned long long)v, stride) : sh.list.key[tid ^ stride];
                const bool low = !(tid & stride), rising = !(tid & size);
                v = (o < v) == (low == rising) ? o : v;
            }
        return v;
    }
    MDP_DEV static int votes(bool v) { return __popcll(__ballot(v)); }
    // how many of a wave's sorted entries are kept, by what `held` weighs; -1 if that is only the 32-bit mass and too near to tell
    MDP_DEV int kept_of_few(int n, double ws, double before, double held, bool in_32) const {
        const double off = rough();
        int kept = s.k > 0 ? min(s.k, n) : n;
        if (s.p < 1.0) {
            const int short_of = votes(lane < kept && before < s.p * held);
            if (in_32 && (votes(lane < kept && before < s.p * held * (1.0 - off)) != short_of || votes(lane < kept && before < s.p * held * (1.0 + off)) != short_of)) return -1;
            kept = min(kept, short_of);
        }
        return max(1, min(kept, votes(lane < n && ws >= s.mp)));
    }
    // the draw among n <= 64 candidates: the first wave's
    MDP_DEV void draw_from_few(const SampleArgs& g, int64_t row, int n, double mass32) const {
        uint64_t sorted = ~0ull;
        double ws = 0.0, before = 0.0;
        int kept = 1;
        if (wave == 0) {
            sorted = sort(lane < n ? sh.list.key[lane] : ~0ull, 64);
            ws = lane < n ? s.weight(value_of(sorted), m) : 0.0;
            const double upto = group_scan<64>(ws);
            before = upto - ws;
            kept = kept_of_few(n, ws, before, s.k > 0 ? of_lane(upto, min(s.k, n) - 1) : mass32, s.k == 0);
            if (lane == 0) sh.found = kept;
        }
        if (s.p < 1.0 && s.k == 0) {
            __syncthreads();
            if (sh.found < 0) {
                const double held = exact_mass();
                if (wave == 0) kept = kept_of_few(n, ws, before, held, false);
            }
        }
        if (wave) return;
        const uint64_t by_place = sort(lane < kept ? sorted << 32 | (uint32_t)lane : ~0ull, 64);
        const double from = __shfl(ws, (int)(uint32_t)by_place & 63);
        const double kw = lane < kept ? from : 0.0;
        const double line = group_scan<64>(kw), sum = of_lane(line, 63);
        const double aim = s.u * sum;
        const uint64_t over = __ballot(kw > 0.0 && line > aim), some = __ballot(kw > 0.0);
        const int who = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)some);
        if (lane == who) answer(g, row, (int)(by_place >> 32), kw, sum);
    }

    MDP_DEV void answer(const SampleArgs& g, int64_t row, int i, double w, double mass) const {
        g.actions[row] = i;
        g.log_prob[row] = (float)log(w / mass);
    }

    // the draw among n listed candidates, among which is everything that k, p and min_p keep
    MDP_DEV void draw_from_list(const SampleArgs& g, int64_t row, int n, double mass32) const {
        const uint64_t word = tid < n ? sh.list.key[tid] : ~0ull;
        __syncthreads();
        const uint64_t sorted = sort(word, n);
        const double ws = tid < n ? s.weight(value_of(sorted), m) : 0.0;
        double all;
        const double upto = block_scan(ws, all), before = upto - ws;
        int kept = s.k > 0 ? min(s.k, n) : n;
        if (s.p < 1.0) {
            double held = mass32;
            if (s.k > 0) held = block_sum(tid == kept - 1 ? upto : 0.0);
            int short_of = block_sum((int)(tid < kept && before < s.p * held));
            if (s.k == 0) {
                // the row's mass in 32 bits decides unless the border is within its error of the aim
                const double off = rough();
                const int low = block_sum((int)(tid < kept && before < s.p * held * (1.0 - off)));
                const int high = block_sum((int)(tid < kept && before < s.p * held * (1.0 + off)));
                if (low != high) {
                    held = exact_mass();
                    short_of = block_sum((int)(tid < kept && before < s.p * held));
                }
            }
            kept = min(kept, short_of);
        }
        kept = min(kept, block_sum((int)(tid < n && ws >= s.mp)));
        kept = max(kept, 1);
        // those that are kept, by place
        sh.list.value[tid] = ws;
        __syncthreads();
        const uint64_t by_place = sort(tid < kept ? sorted << 32 | (uint32_t)tid : ~0ull, kept);
        const double kw = tid < kept ? sh.list.value[(uint32_t)by_place] : 0.0;
        double sum;
        const double line = block_scan(kw, sum);
        const double aim = s.u * sum;
        if (tid == 0) { sh.found = THREADS; sh.last = 0; }
        __syncthreads();
        if (kw > 0.0) {
            if (line > aim) atomicMin(&sh.found, tid);
            atomicMax(&sh.last, tid);
        }
        __syncthreads();
        const int who = sh.found < THREADS ? sh.found : sh.last;
        if (tid == who) answer(g, row, (int)(by_place >> 32), kw, sum);
    }

    MDP_DEV double kept_mass(const Border& b, const float (&v)[N], int i0, double (&w)[N]) const {
        double t = 0.0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            w[e] = b.keeps(v[e], i0 + e) ? s.weight(v[e], m) : 0.0;
            w[e] = w[e] >= s.mp ? w[e] : 0.0;
            t += w[e];
        }
        return t;
    }
    MDP_DEV double kept_mass(const Border& b, int of, int step, double (&w)[N]) const {
        const Chunk<T> q = chunk(of, step);
        float v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = q.at(e);
        return kept_mass(b, v, place(of, step), w);
    }
    // The draw over the whole row: the masses of the waves' pieces, then of the steps of the piece that holds the aim (a wave each),
    // then the entries of that step.
    template <bool CUT>
    MDP_DEV void draw_from_row(const SampleArgs& g, int64_t row, const Border& b) const {
        double mass = 0.0;
        if (!CUT)
            each_chunk([&](int, const float (&v)[N]) {
#pragma unroll
                for (int e = 0; e < N; ++e) mass += s.weight(v[e], m);
            });
        else
            each_chunk_again([&](int h, const float (&v)[N]) {
                double w[N];
                mass += kept_mass(b, v, place(wave, h), w);
            });
        mass = group_sum<64>(mass);
        __syncthreads();
        if (lane == 0) sh.d[wave] = mass;
        __syncthreads();
        double total = 0.0, before = 0.0, run = 0.0;
        for (int w = 0; w < W; ++w) total += sh.d[w];
        const double aim = s.u * total;
        int target = 0;
        for (int w = 0; w < W; ++w) {
            if (sh.d[w] > 0.0 && run <= aim) { target = w; before = run; }
            run += sh.d[w];
        }
        int at = 0;
        run = before;
        for (int h0 = 0; h0 < steps; h0 += W) {
            double w[N];
            const double part = group_sum<64>(kept_mass(b, target, h0 + wave, w));
            __syncthreads();
            if (lane == 0) sh.d[wave] = part;
            __syncthreads();
            for (int h = 0; h < W; ++h) {
                if (sh.d[h] > 0.0 && run <= aim) { at = h0 + h; before = run; }
                run += sh.d[h];
            }
            if (run > aim) break;                      // uniform
        }
        if (wave) return;
        double w[N];
        const double own = kept_mass(b, target, at, w);
        const double upto = before + group_scan<64>(own);
        const uint64_t over = __ballot(own > 0.0 && upto > aim), some = __ballot(own > 0.0);
        const int winner = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)some);   // see the short rows
        if (lane != winner) return;
        double sum = upto - own, found_w = 1.0;
        int found = -1;
        bool open = true;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            sum += w[e];
            if (open && w[e] > 0.0) {
                found = place(target, at) + e;
                found_w = w[e];
                open = !(sum > aim);
            }
        }
        answer(g, row, found, found_w, total);
        if (found_w < kLight) g.log_prob[row] = log_share_of_light(r.entry(found), m, s.c, total);     // the list's entries are heavier
    }
};

// While the row arrives: each thread's largest entry and its mass about that in 32 bits; then the row's.  False for a row without a
// draw (answered here).  A NaN or +inf makes the mass a NaN.
template <class L>
MDP_DEV bool first_pass(L& q, const SampleArgs& g, int64_t row, float& top, double& total) {
    constexpr int N = L::N;
    const float c = q.s.c32();
    top = -__FLT_MAX__;
    double part = 0.0;                                 // sums of chunks: a long row has many
    q.each_chunk([&](int, const float (&v)[N]) {
        float to = top;
#pragma unroll
        for (int e = 0; e < N; ++e) to = larger(v[e], to);
        if (to > top) {
            part *= (double)__builtin_amdgcn_exp2f(larger((top - to) * c, -300.0f));
            top = to;
        }
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) sum += __builtin_amdgcn_exp2f((v[e] - top) * c);
        part += sum;
    });
    q.m = q.block_max(top);
    total = q.block_sum(part * (double)__builtin_amdgcn_exp2f(larger((top - q.m) * c, -300.0f)));
    const bool broken = total != total || q.s.c != q.s.c;
    if (total > 0.0 && !broken) return true;
    if (threadIdx.x == 0) {
        g.actions[row] = -1;
        g.log_prob[row] = broken ? __builtin_nanf("") : 0.0f;
    }
    return false;
}

// A row that is still to be drawn: its action holds this and the bits of its mass in 32 bits, its log_prob its largest entry.
constexpr int64_t kLeft = INT64_MIN;

// Rows that k, p or min_p cut, by the list of candidates.  Rows that it does not decide are left to the kernel below: a kernel of its
// own, so that what it needs does not take registers from this one.
template <typename T, bool MASK, int THREADS, int H>
__global__ __launch_bounds__(THREADS) void k_sample_list(SampleArgs g) {
    using L = LongRow<T, MASK, THREADS, H>;
    __shared__ typename L::Shared sh;
    const int64_t row = blockIdx.x;
    const Settings s(g, row);
    L q(g, row, s, sh);
    float top;
    double total;
    if (!first_pass(q, g, row, top, total)) return;
    if (!s.all()) {
        const float bound = q.bound_of(top, (float)total);
        if (bound > -kInf) {
            const int n = q.gather(bound);
            if (n <= THREADS) {
                if (n <= 64) q.draw_from_few(g, row, n, total);
                else q.draw_from_list(g, row, n, total);
                return;
            }
        }
    }
    if (threadIdx.x == 0) {
        g.actions[row] = kLeft | (int64_t)__float_as_uint((float)total);
        g.log_prob[row] = q.m;
    }
}

// Whole rows: those that nothing cuts (CUT false: each of the launch), or those that the list left.
template <typename T, bool MASK, int THREADS, int H, bool CUT>
__global__ __launch_bounds__(THREADS) void k_sample_whole(SampleArgs g) {
    using L = LongRow<T, MASK, THREADS, H>;
    constexpr int N = L::N;
    __shared__ typename L::Shared sh;
    const int64_t row = blockIdx.x;
    const int64_t left = CUT ? g.actions[row] : 0;
    if (CUT && left >= -1) return;
    const Settings s(g, row);
    L q(g, row, s, sh);
    double total;
    if (CUT) {
        q.m = g.log_prob[row];
        total = (double)__uint_as_float((uint32_t)left);
    } else {
        float top;
        if (!first_pass(q, g, row, top, total)) return;
    }
    Border b = everything();
    if (CUT && (s.k > 0 || s.p < 1.0)) {
        int allowed = 0;
        if (s.k > 0) {
            q.each_chunk_again([&](int, const float (&v)[N]) {
#pragma unroll
                for (int e = 0; e < N; ++e) allowed += v[e] > -kInf;
            });
            allowed = q.block_sum(allowed);
        }
        q.bottom = -__FLT_MAX__;                       // not looked for: the window decides
        b = border_of(q, s, q.m, total, allowed);
    }
    q.template draw_from_row<CUT>(g, row, b);
}

template <typename T, bool MASK>
void launch_sample(const SampleArgs& g, hipStream_t s) {
    const int chunks = most_chunks<T>(g.logits, g.ld, g.rows, g.vocab);
    constexpr int K = 16 / Chunk<T>::N;                // 16 entries a lane
#define SHORT(G)                                                                                                                \
    if (chunks <= G * K) {                                                                                                      \
        constexpr int ROWS = G > 64 ? 1 : 256 / G;                                                                              \
        hipLaunchKernelGGL((k_sample_short<T, MASK, G, K>), dim3((unsigned)((g.rows + ROWS - 1) / ROWS)), dim3(G > 64 ? G : 256), 0, s, g); \
        return;                                                                                                                 \
    }
    SHORT(4) SHORT(8) SHORT(16) SHORT(32) SHORT(64)
    // From here to 4096 entries a row fits the registers of a block just as well; only a small top_k is quicker by the list of
    // candidates (float32, 2^26 entries in rows of 1028 / 2048 / 4096: top_p 412 / 220 / 240 us against 1130 / 590 / 433 by list and
    // whole row, top_k 40 385 / 197 / 209 against 273 / 144 / 90).
    const bool few = !g.top_k && g.top_k_s > 0 && g.top_k_s <= 64;
    if (!few) { SHORT(128) SHORT(256) }
#undef SHORT
    const dim3 grid((unsigned)g.rows);
    const bool all = !g.temperature && !g.top_k && !g.top_p && !g.min_p && g.rate != kGreedy && g.rate == g.rate && g.top_k_s <= 0 && g.top_p_s >= 1.0f && !(g.min_p_s > 0.0f);
#define LONG(THREADS, H)                                                                                                        \
    if (all) {                                                                                                                  \
        hipLaunchKernelGGL((k_sample_whole<T, MASK, THREADS, H, false>), grid, dim3(THREADS), 0, s, g);                         \
    } else {                                                                                                                    \
        hipLaunchKernelGGL((k_sample_list<T, MASK, THREADS, H>), grid, dim3(THREADS), 0, s, g);                                 \
        hipLaunchKernelGGL((k_sample_whole<T, MASK, THREADS, 0, true>), grid, dim3(THREADS), 0, s, g);                          \
    }
    // Four blocks of 256 threads on a CU work on four rows in turn, one of 1024 on one: with many rows the former hide each other's
    // waits (bfloat16 rows of 32000, top_p: 1024 of them 162 us against 216), with fewer than two a CU the latter is done sooner (256
    // of them 55 us against 83).
    if (chunks <= 256 * 4) { LONG(256, 4) }
    else if (chunks <= 256 * 16 && g.rows >= 512) { LONG(256, 16) }
    else if (chunks <= 1024 * 4) { LONG(1024, 4) }
    else { LONG(1024, 16) }
#undef LONG
}

}  // namespace mdp

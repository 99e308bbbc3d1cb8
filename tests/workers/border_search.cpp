// The search of a draw's border (categorical_border_device.hpp) on the host, run by one lane: tests count its passes over the row
// and give it sums that come out differently in another order.  C++17, no GPU headers.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <vector>

#define MDP_DEV inline
namespace mdp {
using std::fmax;
using std::fmin;
constexpr float kInf = __builtin_inff();
inline float fmaxf(float a, float b) { return std::fmax(a, b); }
inline float fminf(float a, float b) { return std::fmin(a, b); }
inline uint32_t key_of(float x) {
    x += 0.0f;
    uint32_t u;
    std::memcpy(&u, &x, 4);
    return (u >> 31) ? ~u : u | 0x80000000u;
}
inline float of_key(uint32_t k) {
    const uint32_t u = (k >> 31) ? k & 0x7fffffffu : ~k;
    float x;
    std::memcpy(&x, &u, 4);
    return x;
}
template <typename V>
inline void anew(V&) {}
inline void atomicAdd(uint32_t* to, uint32_t v) { *to += v; }
}  // namespace mdp
#include "categorical_border_device.hpp"

namespace {

struct TooMany {};

struct HostSettings {
    double c, p;
    int k;
    float c32() const { return (float)fmax(fmin(c, 3e38), 1e-38); }
};

// One lane, `PER` buckets; weights are given, or come from the values.
template <int PER, int CAP, bool KNOWN>
struct HostRow {
    static constexpr int size = 1, per_lane = PER, capacity = CAP;
    static constexpr float window = KNOWN ? 14.0f : 24.0f;
    static constexpr bool total_known = KNOWN;
    const int rank = 0;
    const float* x;
    const double* w;
    long n;
    float m, bottom;
    double c;
    long passes = 0, most;
    uint32_t hist[PER];
    struct Listed { float x; int place; double w; };
    std::vector<Listed> list;
    int number = 0;

    double weight_at(long i) const { return w ? w[i] : weight(x[i]); }
    double weight(float v) const { return std::exp2(((double)v - (double)m) * c); }
    template <class F>
    void each(F&& f) {
        if (++passes > most) throw TooMany{};
        for (long i = 0; i < n; ++i) f(x[i], (int)i, [&] { return weight_at(i); });
    }
    template <class B, class F>
    void sort_in(B&& bucket, F&& f) { each([&](float v, int, auto&& w) { f(bucket(v), w); }); }
    template <class B, class F>
    void each_sorted(B&& bucket, F&& f) { each([&](float v, int i, auto&& w) { f(v, i, w, bucket(v)); }); }
    template <typename V>
    V sum(V v) const { return v; }
    float highest(float v) const { return v; }
    float lowest(float v) const { return v; }
    uint32_t scan(uint32_t v) const { return v; }
    void sync() const {}
    bool any(bool v) const { return v; }
    void clear_list() { list.clear(); number = 0; }
    int listed() const { return number; }
    template <bool COUNT>
    void put(float v, int i, double value) {
        if (number++ < CAP) list.push_back({v, i, value});
    }
    template <bool COUNT>
    mdp::Border last_kept(int count, double above, double aim) {
        if (count <= 0) return {NAN, -1};              // nothing to choose from
        std::vector<Listed> q(list.begin(), list.begin() + count);
        std::sort(q.begin(), q.end(), [](const Listed& a, const Listed& b) { return a.x > b.x || (a.x == b.x && a.place < b.place); });
        int kept = 0;
        double before = above;
        for (const Listed& l : q) {
            if (before < aim) ++kept;
            before += COUNT ? 1.0 : l.w;
        }
        const Listed& last = q[kept ? kept - 1 : 0];
        return {last.x, last.place};
    }
    int nth_equal(float v, int r) {
        ++passes;
        for (long i = 0; i < n; ++i)
            if (x[i] == v && --r == 0) return (int)i;
        return -1;
    }
};

template <int PER, int CAP, bool KNOWN>
long run(const float* x, const double* w, long n, double c, double p, int k, double aim, long most, float* tau, int* place) {
    HostRow<PER, CAP, KNOWN> row;
    row.x = x;
    row.w = w;
    row.n = n;
    row.c = c;
    row.most = most;
    row.m = -FLT_MAX;
    row.bottom = FLT_MAX;
    for (long i = 0; i < n; ++i) {
        row.m = std::fmax(row.m, x[i]);
        if (x[i] > -INFINITY) row.bottom = std::fmin(row.bottom, x[i]);
    }
    if (!KNOWN) row.bottom = -FLT_MAX;
    double total = 0.0;
    int allowed = 0;
    for (long i = 0; i < n; ++i) {
        total += row.weight_at(i);
        allowed += x[i] > -INFINITY;
    }
    if (!KNOWN) total = (float)total;                  // what 32 bits make of it
    const HostSettings s{c, p, k};
    mdp::Border b;
    try {
        b = aim > 0.0 ? mdp::find_border<false>(row, s, row.m, aim, total, false, true) : mdp::border_of(row, s, row.m, total, allowed);
    } catch (TooMany) {
        return -1;
    }
    *tau = b.tau;
    *place = b.place;
    return row.passes;
}

}  // namespace

// The border of a row (weights w, or exp2((x - max) c) where w is null), by k and p, or by an aim > 0; passes over the row, or -1 for
// more than `most`.  form: 0 a long row's block, 1 a short row's wave, 2 four lanes, 3 few places in the list.
extern "C" long border_search(int form, const float* x, const double* w, long n, double c, double p, int k, double aim, long most,
                              float* tau, int* place) {
    switch (form) {
        case 0: return run<4096, 1024, false>(x, w, n, c, p, k, aim, most, tau, place);
        case 1: return run<256, 64, true>(x, w, n, c, p, k, aim, most, tau, place);
        case 2: return run<64, 4, true>(x, w, n, c, p, k, aim, most, tau, place);
        default: return run<64, 8, false>(x, w, n, c, p, k, aim, most, tau, place);
    }
}

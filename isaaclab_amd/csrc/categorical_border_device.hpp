// Where a row's draw is cut: the last entry that top_k and top_p keep.  Includes nothing: what this needs besides a row (key_of, of_key,
// kInf, anew, atomicAdd, MDP_DEV, integer types) comes from who includes it, so that the search also runs on a host, by one lane.
#pragma once

namespace mdp {

// What is kept is a prefix of the row sorted by (value falling, place rising): everything up to and with one entry.
struct Border {
    float tau;
    int place;
    MDP_DEV bool keeps(float x, int i) const { return x > tau || (x == tau && i <= place); }
};
MDP_DEV Border everything() { return Border{-__FLT_MAX__, 0x7fffffff}; }

// Finds the last entry of the shortest prefix that holds `aim`, counting entries (COUNT) or their weights.  C is what searches a row
// together -- a group of lanes or a block -- and gives
//   each(f): f(x, place, w) for each of this lane's entries, w() its weight; sort_in(bucket, f): f(bucket of x, w) for each, and
//   each_sorted(bucket, f): f(x, place, w, bucket of x) after it; weight(x); sum, highest, lowest over all; scan: the sum over the
//   lanes up to and with this one; sync; any: over the lanes that run this loop in step; size, rank: lanes and this lane's number;
//   hist[per_lane size] in shared memory, and there a list of up to `capacity` entries: put<COUNT>(x, place, w) adds one, listed()
//   tells how many were put, last_kept<COUNT>(n, above, aim) finds the border among the n listed, with `above` before them;
//   nth_equal(x, r): the place of the r-th entry equal to x (r from 1); bottom: the row's lowest entry.
// Entries are sorted into buckets that fall with the value: about the maximum first, a bucket a small part of a binary order of
// magnitude or of what the row spans (entries more than `window` orders below share the last).  The bucket in which the aim is
// reached, by 32-bit fixed point, is confirmed in 64 bits while its few entries are listed, and these are looked at one by one.  If
// it is not the one -- entries lighter than a unit of the fixed point add up, or are lost --, its neighbour is looked at, then the
// middle of what is left.  If its entries are too many, the bucket is cut again, by keys and in units of what it weighs, which ends
// with one value.  A peak of 23 above 131071 entries of N(0, 0.1) takes 21 passes at top_p 0.99999, an ordinary row 2 to 5; one
// bucket after the other, where the units stay the row's, took ten thousand.  Where `total`, the mass of the row, is known in 32
// bits only (C::total_known false) and the aim is a share of it (share_of_total), the first pass sums it up in 64.
template <bool COUNT, class C, class S>
MDP_DEV Border find_border(C& c, const S& s, float m, double aim, double total, bool share_of_total, bool active) {
    constexpr int PER = C::per_lane, LAST = PER * C::size - 2, NONE = PER * C::size - 1;   // the last bucket; an entry that is in none
    Border border = everything();
    aim = fmax(aim, 1e-300);                           // the first entry reaches a share of 0
    float per = (float)LAST / fmaxf(fminf(C::window / s.c32(), m - c.bottom), 1e-30f);   // buckets for a difference of 1
    double scale = COUNT ? 1.0 : 2147483648.0 / total;                  // all weights together: half of what 32 bits hold
    float top = m, bottom = -__FLT_MAX__;
    double above = 0.0;
    int shift = -1;                                    // by value; later by key >> shift
    const auto by_value = [&](float x) { return x > -kInf ? (int)fminf((top - x) * per, (float)LAST) : NONE; };
    const auto bucket = [&](float x) {
        if (shift < 0) return by_value(x);
        float again = x;
        anew(again);
        return x <= top && x >= bottom ? (int)((key_of(top) - key_of(again)) >> shift) : NONE;
    };
    while (c.any(active)) {
        c.sync();
        for (int i = 0; i < PER; ++i) c.hist[c.rank * PER + i] = 0u;
        c.sync();
        anew(per);
        anew(scale);
        double weighed = 0.0;
        const auto count_in = [&](int b, auto&& w) {
            const double v = COUNT ? 1.0 : w();
            if (!COUNT && !C::total_known) weighed += v;
            if (active && b != NONE) atomicAdd(&c.hist[b], COUNT ? 1u : (uint32_t)fma(v, scale, 0.5));
        };
        if (c.any(active && shift >= 0)) c.sort_in(bucket, count_in);
        else c.sort_in(by_value, count_in);
        c.sync();
        if (!COUNT && !C::total_known && share_of_total) {
            aim = fmax(s.p * c.sum(weighed), 1e-300);
            share_of_total = false;
        }
        const double need_d = fmin(fmax((aim - above) * scale, 1.0), 4294967295.0);
        const uint32_t need = (uint32_t)__builtin_ceil(need_d);
        uint32_t q[PER], mine = 0u;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            q[i] = c.hist[c.rank * PER + i];
            mine += q[i];
        }
        uint32_t run = c.scan(mine) - mine;
        int b = NONE, full = -1;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            run += q[i];
            if (b == NONE && run >= need) b = c.rank * PER + i;
            if (q[i]) full = c.rank * PER + i;
        }
        b = (int)c.lowest((float)b);
        if (c.any(active && b == NONE)) {              // the aim in the rounding of the last ones: the last that holds anything
            full = (int)c.highest((float)full);
            if (b == NONE) b = full < 0 ? LAST : full;
        }
        // confirm: the bucket is not the one while the entries above it reach the aim by themselves, or fall short of it with its own
        int count;
        double more, in;
        bool sure = !active, few = false;
        int from = 0, to = LAST;                       // the buckets among which it is
        bool tried = false;
        for (;;) {
            more = 0.0;
            in = 0.0;
            c.sync();
            c.clear_list();
            c.sync();
            c.each_sorted(bucket, [&](float x, int i, auto&& w, int at) {
                const double v = COUNT ? 1.0 : w();
                more += at < b ? v : 0.0;
                if (at == b) {
                    in += v;
                    if (active) c.template put<COUNT>(x, i, v);
                }
            });
            c.sync();
            more = c.sum(more);
            in = c.sum(in);
            count = c.listed();
            int go = 0;
            if (above + more >= aim && b > from) go = -1;
            else if (above + more + in < aim && b < to) go = 1;
            if (go == 0) sure = true;
            if (!c.any(active && !sure)) break;
            if (go < 0) to = b - 1;
            else if (go > 0) from = b + 1;
            if (!sure) b = tried ? (from + to) / 2 : b + go;
            tried = true;
        }
        few = (unsigned)(count - 1) < (unsigned)C::capacity;
        if (c.any(active && few)) {
            const Border found = c.template last_kept<COUNT>(active && few ? count : 0, above + more, aim);
            if (active && few) border = found;
        }
        if (c.any(active && !few)) {
            float hi = -kInf, lo = kInf;
            c.each_sorted(bucket, [&](float x, int, auto&&, int at) {
                if (at == b) { hi = fmaxf(hi, x); lo = fminf(lo, x); }
            });
            hi = c.highest(hi);
            lo = c.lowest(lo);
            const bool one = hi == lo;
            if (c.any(active && !few && one)) {
                const double v = COUNT ? 1.0 : c.weight(hi), want = (aim - (above + more)) / v;
                const int r = want < 1.0 ? 1 : want < (double)count ? (int)__builtin_ceil(want) : count;
                const int place = c.nth_equal(hi, r);
                if (active && !few && one) border = Border{hi, place};
            }
            if (!few && !one) {
                if (count) {
                    top = hi;
                    bottom = lo;
                    above += more;
                    if (!COUNT) scale = 2147483648.0 / in;
                } else if (shift < 0) {
                    // an empty bucket: the aim lies between two others, in the last bits of sums of another order.  All by keys,
                    top = m;
                    bottom = -__FLT_MAX__;
                } else {
                    // which tell where it starts
                    const uint64_t lost = (uint64_t)b << shift, all = key_of(top) - key_of(bottom);
                    if (active) border = Border{of_key(key_of(top) - (uint32_t)(lost <= all ? lost - 1 : all)), 0x7fffffff};
                    active = false;
                }
                const uint32_t range = key_of(top) - key_of(bottom);
                shift = 0;
                while (range >> shift > (uint32_t)LAST) ++shift;
            }
            active = active && !few && !one;
        } else active = false;
    }
    return border;
}

// The border that k and p draw together, of `allowed` entries that weigh `total`.
template <class C, class S>
MDP_DEV Border border_of(C& c, const S& s, float m, double total, int allowed) {
    Border b = everything();
    const bool by_k = s.k > 0 && s.k < allowed, by_p = s.p < 1.0;
    double held = total;
    if (c.any(by_k)) {
        const Border f = find_border<true>(c, s, m, (double)s.k, 1.0, false, by_k);
        if (by_k) b = f;
        if (c.any(by_k && by_p)) {
            double kept = 0.0;
            c.each([&](float x, int i, auto&& w) { kept += b.keeps(x, i) ? w() : 0.0; });
            held = c.sum(kept);
        }
    }
    if (c.any(by_p)) {
        const Border f = find_border<false>(c, s, m, s.p * held, total, !by_k, by_p);
        if (by_p && (f.tau > b.tau || (f.tau == b.tau && f.place < b.place))) b = f;
    }
    return b;
}

}  // namespace mdp

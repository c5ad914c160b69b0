// A step's logits to its next codes on gfx950 (the C ABI's navi_sample_rows and navi_draft_accept): one token for every row under its
// own rule, and the drafted rows that the sampled codes confirm.
//
// Sampling. A row's tokens stand in the order of their logits x (the lowest index first among equals). Their weights are
// 2^(4 c (x - max) / 4) with c = log2 e / temperature; a rule keeps a prefix of the order, and the token is the first, in the order of the
// indexes, at which the kept weights' running sum passes u of their total. So that the token is the definition's and not that of the
// sums' rounding, weights are computed in 64 bits (2^-43) and summed as integers or in 64 bits.
//
//  * The order is cut into bins of a quarter of a power of two, bin floor(4 c x), 256 of them below the largest (2^-64: what is
//    below has no weight). One pass counts the tokens and sums the weights of every bin, one LDS atomic a token: the weight in
//    units of 2^-31 of its bin's edge below bit 48, the count above.
//  * The sums over the bins say in which bin top-k and top-p end. Only that bin's tokens are looked at again: a radix
//    select over (logit, index) as one 64-bit key, by count or by weight, gives the last key that is kept.
//  * Then the kept weights are summed in the order of the indexes, and the wave that holds the border names the token.
//
// Up to 16384 tokens a block has its row in registers and does all of this in one launch. Longer rows are cut into chunks: a launch makes
// the chunks' bins, a second copies the tokens of the bins in question, a third does the rest, reading again only the chunk that
// the number falls into.
#include "host_util.h"
#include "kv.h"
#include "sampler.h"

#include <algorithm>
#include <cfloat>

// 4 c x is rounded once wherever it is used, so that a token's bin, its place in it and what it is compared with fit together: a product
// fused into the difference after it would differ from the rounded one by more than a bin for logits near the largest number.
#pragma clang fp contract(off)

namespace navi_amd {
namespace sample {

constexpr int BINS = 256;
constexpr int CAP = 8192;              // tokens of the bins in question that are kept in LDS; more are read from the row again
constexpr int ROW_MOST = 16384;        // tokens of a row that a block has in registers
constexpr int MAXC = 64;               // most chunks of a row
constexpr int PER = 16;                // tokens of a thread of a chunk

struct Args {
    const void *x;
    const navi_sample_rule *rules;
    const float *u;
    const uint32_t *allowed, *seen;
    int32_t *token;
    float *logprob;
    uint64_t *bins, *best, *list;      // the workspace (ws_of): [row][chunk][BINS], [row][chunk], [row][CAP]
    int32_t *listed;                   // [row]
    int rows, vocab, ld, n_rules, ld_allowed, ld_seen, ld_token, chunks;
};

// A token's place in the order as a number, the first the largest. 0 comes after all of them.
__device__ __forceinline__ uint64_t key_of(float x, int i) { return static_cast<uint64_t>(float_key(x)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(i)); }
__device__ __forceinline__ float logit_of(uint64_t key) { return key_float(static_cast<unsigned>(key >> 32)); }
__device__ __forceinline__ int index_of(uint64_t key) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key)); }

struct Rule {
    double c4;                         // 4 log2 e / temperature
    double p, m;                       // top_p; log2 min_p
    float penalty;
    int k;                             // 0: off, as p of 1 and m of -inf are
    bool greedy;
    __device__ __forceinline__ bool cuts() const { return k > 0 || p < 1.0 || m != -INFINITY; }
};
__device__ __forceinline__ Rule rule_of(const Args &a, int row) {
    const navi_sample_rule *s = a.rules + (a.n_rules == 1 ? 0 : row);
    Rule r;
    const float t = gld(&s->temperature), p = gld(&s->top_p), m = gld(&s->min_p), pen = gld(&s->repetition_penalty);
    r.greedy = !(t > 0.f);
    r.c4 = r.greedy ? 0.0 : 4.0 * 1.44269504088896340736 / static_cast<double>(t);
    r.k = max(gld(&s->top_k), 0);
    r.p = p < 1.f ? fmax(static_cast<double>(p), 0.0) : 1.0;
    r.m = m > 0.f ? log2(fmin(static_cast<double>(m), 1.0)) : -INFINITY;
    r.penalty = pen > 0.f ? pen : 1.f;
    return r;
}

// A row's logits as its rule sees them: -inf for what is not allowed, NaN and -inf; no -0; at most the largest finite number.
template <class T>
struct Row {
    const T *x;
    const uint32_t *allowed, *seen;
    float penalty;
    int vocab;
    bool vec;                          // four at a time are aligned
    __device__ __forceinline__ Row(const Args &a, int row, float pen) {
        x = static_cast<const T *>(a.x) + static_cast<size_t>(row) * a.ld;
        allowed = a.allowed ? a.allowed + static_cast<size_t>(row) * a.ld_allowed : nullptr;
        seen = a.seen && pen != 1.f ? a.seen + static_cast<size_t>(row) * a.ld_seen : nullptr;
        penalty = pen;
        vocab = a.vocab;
        vec = (reinterpret_cast<uintptr_t>(x) & (4 * sizeof(T) - 1)) == 0;
    }
    __device__ __forceinline__ float as_seen(float v, int i, uint32_t allow, uint32_t see) const {
        if (see >> (i & 31) & 1u) v = v > 0.f ? v / penalty : v * penalty;
        v = v != v ? -INFINITY : fminf(v, FLT_MAX) + 0.f;
        return allow >> (i & 31) & 1u ? v : -INFINITY;
    }
    __device__ __forceinline__ float at(int i) const {
        return as_seen(static_cast<float>(gld(x + i)), i, allowed ? gld(allowed + (i >> 5)) : ~0u, seen ? gld(seen + (i >> 5)) : 0u);
    }
    // tokens i .. i + 3, i a multiple of 4; -inf past the last
    __device__ __forceinline__ void four(int i, float *v) const {
        if (i >= vocab) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = -INFINITY;
            return;
        }
        if (vec && i + 4 <= vocab) {
            typedef T T4 __attribute__((ext_vector_type(4)));
            const T4 t = *(const NAVI_GLOBAL T4 *) (x + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(t[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = i + e < vocab ? static_cast<float>(gld(x + i + e)) : -INFINITY;
        }
        const uint32_t allow = allowed ? gld(allowed + (i >> 5)) : ~0u, see = seen ? gld(seen + (i >> 5)) : 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = as_seen(v[e], i + e, allow, see);
    }
};

// 2^(f / 4) for 0 <= f < 1: e^g about the middle, g = (f / 4 - 1 / 8) ln 2; the eighth power that is left out is 2^-43.
__device__ __forceinline__ double quarter(double f) {
    const double g = fma(f, 0.25 * 0.693147180559945309417, -0.125 * 0.693147180559945309417);
    double s = 1.0 / 5040;
    s = fma(s, g, 1.0 / 720);
    s = fma(s, g, 1.0 / 120);
    s = fma(s, g, 1.0 / 24);
    s = fma(s, g, 1.0 / 6);
    s = fma(s, g, 0.5);
    s = fma(s, g, 1.0);
    s = fma(s, g, 1.0);
    return s * 1.09050773266525765921;                            // 2^(1 / 8)
}
// 2^(-j / 4)
__device__ __forceinline__ double bin_edge(int j) {
    const double q[4] = {1.0, 0.840896415253714543031, 0.707106781186547524401, 0.594603557501360533359};
    const double f = (j & 3) == 0 ? q[0] : (j & 3) == 1 ? q[1] : (j & 3) == 2 ? q[2] : q[3];
    return ldexp(f, -(j >> 2));
}

constexpr double UNIT = 2147483648.0;  // 2^31: a weight at its bin's edge

// A token's bin below the row's (or chunk's) first, BINS or more: none, and its weight over the bin's edge.
struct Place {
    int j;
    double w;
};
__device__ __forceinline__ int bin_of(float x, double c4, double top) {
    return x == -INFINITY ? BINS : static_cast<int>(fmin(top - floor(static_cast<double>(x) * c4), static_cast<double>(BINS)));
}
__device__ __forceinline__ Place place_of(float x, double c4, double top) {
    const double q = static_cast<double>(x) * c4, b = floor(q);
    Place p;
    p.j = x == -INFINITY ? BINS : static_cast<int>(fmin(top - b, static_cast<double>(BINS)));
    p.w = quarter(q - b);
    return p;
}
__device__ __forceinline__ uint64_t units(double w) { return static_cast<uint64_t>(static_cast<uint32_t>(w * UNIT + 0.5)); }

__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) v = max(v, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(v), o)));
    return v;
}
__device__ __forceinline__ double wave_scan(double v) {           // inclusive
    const int l = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const double x = __shfl_up(v, o);
        if (l >= o) v += x;
    }
    return v;
}

template <int BT>
struct Lds {
    static constexpr int NW = BT / WAVE;
    unsigned long long w[BINS];        // sums of the weights of the bins, then of a radix digit's tokens
    unsigned n[BINS];                  // and their counts
    double upto[BINS];                 // weights and counts of the bins up to each, in units of the first bin's edge
    int count[BINS];
    unsigned long long red[2][NW];
    double seg[64], part[4];
    int partn[4];
    unsigned long long key;
    int listed, kb, pb;
};

// The block's largest; `slot` 0 or 1 of red, free until the call after the next with the same one.
template <int BT>
__device__ __forceinline__ uint64_t block_max(uint64_t v, Lds<BT> &q, int slot) {
    v = wave_max64(v);
    if ((threadIdx.x & 63) == 0) q.red[slot][threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t m = q.red[slot][0];
#pragma unroll
    for (int i = 1; i < Lds<BT>::NW; ++i) m = max(m, static_cast<uint64_t>(q.red[slot][i]));
    return m;
}

// upto and count from w and n.
template <int BT>
__device__ __forceinline__ void sum_bins(Lds<BT> &q) {
    const int t = threadIdx.x, wv = t >> 6;
    double w = 0.0;
    int n = 0;
    if (t < BINS) {
        w = wave_scan(static_cast<double>(q.w[t]) * (bin_edge(t) / UNIT));
        n = wave_incl_scan(static_cast<int>(q.n[t]));
        if ((t & 63) == 63) {
            q.part[wv] = w;
            q.partn[wv] = n;
        }
    }
    __syncthreads();
    if (t < BINS) {
        double before = 0.0;
        int first = 0;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            before += i < wv ? q.part[i] : 0.0;
            first += i < wv ? q.partn[i] : 0;
        }
        q.upto[t] = before + w;
        q.count[t] = first + n;
    }
    __syncthreads();
}

// The bin in which a rule's top_k ends (BINS: it keeps all), and the one in which the weights up to it reach `mass`. All threads.
template <int BT>
__device__ __forceinline__ int bin_of_count(Lds<BT> &q, int k) {
    const int t = threadIdx.x;
    if (k < 1 || k >= q.count[BINS - 1]) return BINS;             // the same for all
    if (t < BINS && q.count[t] >= k && (t == 0 || q.count[t - 1] < k)) q.kb = t;
    __syncthreads();
    return q.kb;
}
template <int BT>
__device__ __forceinline__ int bin_of_mass(Lds<BT> &q, double mass) {
    const int t = threadIdx.x;
    __syncthreads();                                              // the readers of the call before are done
    if (t < BINS) {
        const int here = q.count[t], before = t ? q.count[t - 1] : 0;
        if (here > before && (q.upto[t] >= mass || here == q.count[BINS - 1]) && (before == 0 || q.upto[t - 1] < mass)) q.pb = t;
    }
    __syncthreads();
    return q.pb;
}

// The bins whose tokens are looked at again: those in which top_k and min_p end, and p0 .. p1, in one of which top_p does.
struct Marks {
    int kb, mb, p0, p1;
    __device__ __forceinline__ bool any() const { return kb < BINS || mb < BINS || p0 <= p1; }
    __device__ __forceinline__ bool has(int j) const { return j < BINS && (j == kb || j == mb || (j >= p0 && j <= p1)); }
};

// Tokens to look at again: keys in LDS, or, where they are too many, the row.
struct List {
    const unsigned long long *key;
    int n;
    template <int BT, class F>
    __device__ __forceinline__ void each(F f) const {
        for (int i = threadIdx.x; i < n; i += BT) f(static_cast<uint64_t>(key[i]));
    }
};
template <class T>
struct Whole {
    const Row<T> &row;
    template <int BT, class F>
    __device__ __forceinline__ void each(F f) const {
        for (int i = threadIdx.x; i < row.vocab; i += BT) {
            const float x = row.at(i);
            if (x != -INFINITY) f(key_of(x, i));
        }
    }
};

// Of the tokens in bin `bin`, largest key first: the key at which their count reaches `need`, or (need 0) their weights' sum `mass` in
// units. `sum`: the weights up to it and with it. A digit of 8 bits at a time, from the highest in which the keys differ, until one token is left.
// q.w and q.n are used. All threads.
template <int BT, class S>
__device__ uint64_t select(const S &s, Lds<BT> &q, double c4, double top, int bin, int need, double mass, uint64_t &sum) {
    const int t = threadIdx.x, l = t & 63;
    uint64_t hi = 0, lo = 0;                                      // lo: of the complements
    s.template each<BT>([&](uint64_t k) {
        if (bin_of(logit_of(k), c4, top) == bin) {
            hi = max(hi, k);
            lo = max(lo, ~k);
        }
    });
    __syncthreads();
    hi = block_max(hi, q, 0);
    lo = ~block_max(lo, q, 1);
    sum = 0;
    if (hi == 0) return 0;                                        // no token
    int h = hi == lo ? 0 : 64 - __builtin_clzll(hi ^ lo);         // bits from h on are settled
    uint64_t prefix = h < 64 ? hi >> h : 0;
    if (h == 0) {
        sum = units(place_of(logit_of(hi), c4, top).w);
        return hi;
    }
    while (true) {
        const int width = min(h, 8), at = h - width;
        __syncthreads();
        if (t < BINS) {
            q.w[t] = 0;
            q.n[t] = 0;
        }
        __syncthreads();
        s.template each<BT>([&](uint64_t k) {
            const Place p = place_of(logit_of(k), c4, top);
            if (p.j != bin || (h < 64 ? k >> h : 0) != prefix) return;
            const unsigned d = static_cast<unsigned>(k >> at) & ((1u << width) - 1u);
            atomicAdd(&q.n[d], 1u);
            atomicAdd(&q.w[d], static_cast<unsigned long long>(units(p.w)));
        });
        __syncthreads();
        // lane l has digits 255 - 4 l .. 252 - 4 l; every wave finds the digit itself
        int c[4], cs = 0;
        uint64_t w[4], ws = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c[i] = static_cast<int>(q.n[255 - 4 * l - i]);
            w[i] = q.w[255 - 4 * l - i];
            cs += c[i];
            ws += w[i];
        }
        int cb = wave_incl_scan(cs) - cs;
        uint64_t wb = ws;
#pragma unroll
        for (int o = 1; o < WAVE; o <<= 1) {
            const uint64_t x = __shfl_up(static_cast<unsigned long long>(wb), o);
            if (l >= o) wb += x;
        }
        wb -= ws;
        int d = -1, dc = 0, dn = 0, last = -1, lc = 0, ln = 0;
        uint64_t dw = 0, db = 0, lw = 0, lb = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool reached = need > 0 ? cb + c[i] >= need : static_cast<double>(wb + w[i]) >= mass;
            if (c[i] > 0) {
                if (d < 0 && reached) { d = 255 - 4 * l - i; dc = cb; dn = c[i]; dw = w[i]; db = wb; }
                last = 255 - 4 * l - i; lc = cb; ln = c[i]; lw = w[i]; lb = wb;
            }
            cb += c[i];
            wb += w[i];
        }
        uint64_t hit = __ballot(d >= 0);
        int src;
        if (hit) {
            src = __builtin_ctzll(hit);
        } else {                                                  // the sum falls short of the mass by its rounding: the last one
            src = 63 - __builtin_clzll(__ballot(last >= 0));
            d = last; dc = lc; dn = ln; dw = lw; db = lb;
        }
        d = __shfl(d, src);
        dn = __shfl(dn, src);
        dc = __shfl(dc, src);
        dw = __shfl(static_cast<unsigned long long>(dw), src);
        db = __shfl(static_cast<unsigned long long>(db), src);
        need -= need > 0 ? dc : 0;
        mass -= static_cast<double>(db);
        sum += db;
        prefix = prefix << width | static_cast<uint64_t>(d);
        h = at;
        if (dn == 1 || h == 0) {
            sum += dw;
            if (h == 0) return prefix;
            s.template each<BT>([&](uint64_t k) {
                if (k >> h == prefix && bin_of(logit_of(k), c4, top) == bin) q.key = k;
            });
            __syncthreads();
            return q.key;
        }
    }
}

// The last of the order that is kept: all bins before `bin`, and of it the keys from `key` on. bin BINS: all.
struct Cut {
    int bin;
    uint64_t key;
    __device__ __forceinline__ void narrow(int b, uint64_t k) {
        if (b < bin || (b == bin && k > key)) {
            bin = b;
            key = k;
        }
    }
    __device__ __forceinline__ bool keeps(int j, uint64_t k) const { return j < bin || (j == bin && k >= key); }
};

// From the bins' sums (sum_bins). best4: 4 c times the row's largest logit. All threads.
template <int BT>
__device__ __forceinline__ Marks marks_of(Lds<BT> &q, const Rule &r, double best4, double top) {
    Marks k{bin_of_count(q, r.k), BINS, BINS, -1};
    if (r.m != -INFINITY) k.mb = static_cast<int>(fmin(top - floor(best4 + 4.0 * r.m), static_cast<double>(BINS)));
    if (r.p < 1.0) {
        const double least = k.kb == BINS ? q.upto[BINS - 1] : k.kb ? q.upto[k.kb - 1] : 0.0, most = q.upto[min(k.kb, BINS - 1)];
        k.p0 = bin_of_mass(q, r.p * least);
        k.p1 = bin_of_mass(q, r.p * most);
    }
    return k;
}

// What a rule keeps, from the bins' sums and the tokens of the bins in question.
template <int BT, class S>
__device__ Cut cut_of(const S &s, Lds<BT> &q, const Rule &r, double best4, double top, const Marks &marks) {
    const int kb = marks.kb, mb = marks.mb;
    Cut cut{BINS, 0};
    double all = q.upto[BINS - 1];
    uint64_t sum;
    if (kb < BINS) {
        const double before = kb ? q.upto[kb - 1] : 0.0;
        cut.narrow(kb, select(s, q, r.c4, top, kb, r.k - (kb ? q.count[kb - 1] : 0), 0.0, sum));
        all = before + static_cast<double>(sum) * (bin_edge(kb) / UNIT);
    }
    if (r.p < 1.0) {
        const double mass = r.p * all;
        const int pb = min(max(bin_of_mass(q, mass), marks.p0), marks.p1);
        const double before = pb ? q.upto[pb - 1] : 0.0;
        cut.narrow(pb, select(s, q, r.c4, top, pb, 0, (mass - before) * (UNIT / bin_edge(pb)), sum));
    }
    if (mb < BINS) {
        // the least key that reaches min_p, or, where none of the bin does, one more than all of them
        uint64_t least = 0, most = 0;                             // least: of the complements
        s.template each<BT>([&](uint64_t k) {
            const float x = logit_of(k);
            if (bin_of(x, r.c4, top) != mb) return;
            most = max(most, k);
            if ((static_cast<double>(x) * r.c4 - best4) * 0.25 >= r.m) least = max(least, ~k);
        });
        __syncthreads();
        least = block_max(least, q, 0);
        most = block_max(most, q, 1);
        cut.narrow(mb, least ? ~least : most + 1);
    }
    return cut;
}

// The first token of the block's BT x N (from i0 on, in registers: thread t has 4 from i0 + 4 (k BT + t)) at which the kept weights'
// sum passes `number` (FROM_U: that part of the sum); none passes it: the last kept one. `total`: the sum of all kept weights of the row, for the
// log probability (FROM_U: the block's).
template <int BT, int N, bool FROM_U>
__device__ __forceinline__ void draw(const Args &a, int row, const float (&v)[N], int i0, Lds<BT> &q, const Rule &r, double top, const Cut &cut, double number,
                                     double total) {
    constexpr int K = N / 4, NW = BT / WAVE;
    static_assert(K * NW <= 64, "a segment a lane");
    const int t = threadIdx.x, l = t & 63, wv = t >> 6;
    double own[K];
    __syncthreads();
    if (K * NW < 64 && t < 64) q.seg[t] = 0.0;
    if (K * NW < 64) __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        own[k] = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const Place p = place_of(v[4 * k + e], r.c4, top);
            if (p.j < BINS && cut.keeps(p.j, key_of(v[4 * k + e], i0 + (k * BT + t) * 4 + e))) own[k] += p.w * bin_edge(p.j);
        }
        const double sum = wave_scan(own[k]);
        if (l == 63) q.seg[k * NW + wv] = sum;
    }
    __syncthreads();
    const double mine = q.seg[l], upto = wave_scan(mine);
    if (FROM_U) {
        total = __shfl(upto, 63);
        number *= total;
    }
    const uint64_t past = __ballot(upto > number), some = __ballot(mine > 0.0);
    if (!some) return;                                            // nothing is kept here
    const int seg = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
    if (seg % NW != wv) return;
    const double before = seg ? __shfl(upto, seg - 1) : 0.0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (seg / NW != k) continue;
        const double sum = before + wave_scan(own[k]);
        const uint64_t over = __ballot(own[k] > 0.0 && sum > number), any = __ballot(own[k] > 0.0);
        const int lane = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
        if (l == lane) {
            double run = sum - own[k], weight = 0.0;
            int pick = -1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = i0 + (k * BT + t) * 4 + e;
                const Place p = place_of(v[4 * k + e], r.c4, top);
                if (p.j < BINS && cut.keeps(p.j, key_of(v[4 * k + e], i)) && (pick < 0 || run <= number)) {
                    pick = i;
                    weight = p.w * bin_edge(p.j);
                    run += weight;
                }
            }
            gst(a.token + static_cast<size_t>(row) * a.ld_token, pick);
            if (a.logprob) gst(a.logprob + row, static_cast<float>(log(weight / total)));
        }
    }
}

__device__ __forceinline__ void put(const Args &a, int row, int token, float logprob) {
    gst(a.token + static_cast<size_t>(row) * a.ld_token, token);
    if (a.logprob) gst(a.logprob + row, logprob);
}
__device__ __forceinline__ double number_of(const Args &a, int row) {
    const float u = gld(a.u + row);
    return u > 0.f ? static_cast<double>(fminf(u, 0x1.fffffep-1f)) : 0.0;
}

// ---- a row a block ---------------------------------------------------------------------------

template <class T, int BT, int N>
__global__ void __launch_bounds__(BT) k_row(Args a) {
    __shared__ Lds<BT> q;
    constexpr int HELD = BT * N < CAP ? BT * N : CAP;
    __shared__ unsigned long long list[HELD];
    const int row = blockIdx.x, t = threadIdx.x;
    const Rule r = rule_of(a, row);
    const Row<T> x(a, row, r.penalty);
    float v[N];
    uint64_t best = 0;
    if (t < BINS) {
        q.w[t] = 0;
        q.n[t] = 0;
    }
    if (t == 0) q.listed = 0;
#pragma unroll
    for (int k = 0; k < N / 4; ++k) x.four((k * BT + t) * 4, v + 4 * k);
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (v[i] != -INFINITY) best = max(best, key_of(v[i], (i / 4 * BT + t) * 4 + i % 4));
    best = block_max(best, q, 0);
    if (best == 0 || r.greedy) {
        if (t == 0) put(a, row, best ? index_of(best) : -1, best ? 0.f : -INFINITY);
        return;
    }
    const double best4 = static_cast<double>(logit_of(best)) * r.c4, top = floor(best4);
    Cut cut{BINS, 0};
    if (r.cuts()) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const Place p = place_of(v[i], r.c4, top);
            if (p.j < BINS) atomicAdd(&q.w[p.j], 1ull << 48 | units(p.w));
        }
        __syncthreads();
        if (t < BINS) {
            q.n[t] = static_cast<unsigned>(q.w[t] >> 48);
            q.w[t] &= (1ull << 48) - 1;
        }
        __syncthreads();
        sum_bins(q);
        const Marks marks = marks_of(q, r, best4, top);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (marks.has(bin_of(v[i], r.c4, top))) {
                const int at = atomicAdd(&q.listed, 1);
                if (at < HELD) list[at] = key_of(v[i], (i / 4 * BT + t) * 4 + i % 4);
            }
        }
        __syncthreads();
        if (q.listed <= HELD) cut = cut_of(List{list, q.listed}, q, r, best4, top, marks);
        else cut = cut_of(Whole<T>{x}, q, r, best4, top, marks);
    }
    draw<BT, N, true>(a, row, v, 0, q, r, top, cut, number_of(a, row), 0.0);
}

// ---- a row in chunks -------------------------------------------------------------------------

// A chunk's bins below its own largest token's, and that token's key.
template <class T, int BT>
__global__ void __launch_bounds__(BT) k_bins(Args a) {
    __shared__ unsigned long long w[4][BINS];
    __shared__ Lds<BT> q;
    const int chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks, t = threadIdx.x, i0 = chunk * BT * PER;
    const Rule r = rule_of(a, row);
    const Row<T> x(a, row, r.penalty);
    float v[PER];
    for (int i = t; i < 4 * BINS; i += BT) w[i / BINS][i % BINS] = 0;
    if (chunk == 0 && t == 0) gst(a.listed + row, 0);
#pragma unroll
    for (int k = 0; k < PER / 4; ++k) x.four(i0 + (k * BT + t) * 4, v + 4 * k);
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (v[i] != -INFINITY) best = max(best, key_of(v[i], i0 + (i / 4 * BT + t) * 4 + i % 4));
    best = block_max(best, q, 0);
    const size_t at = static_cast<size_t>(row) * a.chunks + chunk;
    if (t == 0) gst(a.best + at, best);
    if (r.greedy) return;
    if (best) {
        const double top = floor(static_cast<double>(logit_of(best)) * r.c4);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const Place p = place_of(v[i], r.c4, top);
            if (p.j < BINS) atomicAdd(&w[t & 3][p.j], 1ull << 48 | units(p.w));
        }
    }
    __syncthreads();
    for (int i = t; i < BINS; i += BT) gst(a.bins + at * BINS + i, static_cast<uint64_t>(w[0][i] + w[1][i] + w[2][i] + w[3][i]));
}

// A row's largest token and its bins from its chunks'; q.w, q.n, upto and count are set where it is not greedy. false: no token.
struct Merged {
    uint64_t best;
    double best4, top;
};
template <int BT>
__device__ __forceinline__ Merged merge(const Args &a, int row, const Rule &r, Lds<BT> &q) {
    const int t = threadIdx.x;
    const size_t at = static_cast<size_t>(row) * a.chunks;
    if (t < BINS) {
        q.w[t] = 0;
        q.n[t] = 0;
    }
    Merged m;
    m.best = block_max(t < a.chunks ? gld(a.best + at + t) : uint64_t(0), q, 0);
    m.best4 = static_cast<double>(logit_of(m.best)) * r.c4;
    m.top = floor(m.best4);
    if (m.best == 0 || r.greedy) return m;
    for (int i = t; i < a.chunks * BINS; i += BT) {
        const uint64_t b = gld(a.best + at + i / BINS), x = gld(a.bins + at * BINS + i);
        if (!b || !x) continue;
        const double j = m.top - floor(static_cast<double>(logit_of(b)) * r.c4) + i % BINS;
        if (j < BINS) {
            atomicAdd(&q.n[static_cast<int>(j)], static_cast<unsigned>(x >> 48));
            atomicAdd(&q.w[static_cast<int>(j)], static_cast<unsigned long long>(x & ((1ull << 48) - 1)));
        }
    }
    __syncthreads();
    sum_bins(q);
    return m;
}

// The tokens of the bins in question, in any order.
template <class T, int BT>
__global__ void __launch_bounds__(BT) k_list(Args a) {
    __shared__ Lds<BT> q;
    const int chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks, t = threadIdx.x, i0 = chunk * BT * PER;
    const Rule r = rule_of(a, row);
    if (r.greedy || !r.cuts()) return;
    const Row<T> x(a, row, r.penalty);
    const Merged m = merge(a, row, r, q);
    if (m.best == 0) return;
    const Marks marks = marks_of(q, r, m.best4, m.top);
    if (!marks.any()) return;
    float v[PER];
#pragma unroll
    for (int k = 0; k < PER / 4; ++k) x.four(i0 + (k * BT + t) * 4, v + 4 * k);
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (marks.has(bin_of(v[i], r.c4, m.top))) {
            const int at = atomicAdd(a.listed + row, 1);
            if (at < CAP) gst(a.list + static_cast<size_t>(row) * CAP + at, key_of(v[i], i0 + (i / 4 * BT + t) * 4 + i % 4));
        }
}

constexpr int FT = 1024;
// What is kept, the chunk into which the number falls, and the token. CHUNK: tokens of a chunk.
template <class T, int CHUNK>
__global__ void __launch_bounds__(FT) k_pick(Args a) {
    __shared__ Lds<FT> q;
    __shared__ unsigned long long list[CAP];
    __shared__ unsigned long long part[MAXC];                     // of the last kept bin, in units
    __shared__ double mass[MAXC];
    const int row = blockIdx.x, t = threadIdx.x, l = t & 63, wv = t >> 6;
    const Rule r = rule_of(a, row);
    const Merged m = merge(a, row, r, q);
    if (m.best == 0 || r.greedy) {
        if (t == 0) put(a, row, m.best ? index_of(m.best) : -1, m.best ? 0.f : -INFINITY);
        return;
    }
    const Row<T> x(a, row, r.penalty);
    const Marks marks = marks_of(q, r, m.best4, m.top);
    const int n = marks.any() ? gld(a.listed + row) : 0;
    const bool held = n <= CAP;
    if (held)
        for (int i = t; i < n; i += FT) list[i] = gld(a.list + static_cast<size_t>(row) * CAP + i);
    if (t < MAXC) part[t] = 0;
    __syncthreads();
    Cut cut{BINS, 0};
    if (marks.any()) cut = held ? cut_of(List{list, n}, q, r, m.best4, m.top, marks) : cut_of(Whole<T>{x}, q, r, m.best4, m.top, marks);
    if (cut.bin < BINS) {
        auto add = [&](uint64_t k) {
            const Place p = place_of(logit_of(k), r.c4, m.top);
            if (p.j == cut.bin && k >= cut.key) atomicAdd(&part[index_of(k) / CHUNK], static_cast<unsigned long long>(units(p.w)));
        };
        if (held) List{list, n}.each<FT>(add);
        else Whole<T>{x}.template each<FT>(add);
    }
    __syncthreads();
    // the chunks' kept weights, a wave a chunk
    const size_t at = static_cast<size_t>(row) * a.chunks;
    for (int c = wv; c < a.chunks; c += FT / WAVE) {
        const uint64_t b = gld(a.best + at + c);
        double sum = 0.0;
        if (b) {
            const double off = m.top - floor(static_cast<double>(logit_of(b)) * r.c4);
#pragma unroll
            for (int i = 0; i < BINS / WAVE; ++i) {
                const double j = off + (i * WAVE + l);
                if (j < cut.bin)
                    sum += static_cast<double>(gld(a.bins + (at + c) * BINS + i * WAVE + l) & ((1ull << 48) - 1)) * (bin_edge(static_cast<int>(j)) / UNIT);
            }
        }
        sum = wave_scan(sum);
        if (l == 63) mass[c] = sum + (cut.bin < BINS ? static_cast<double>(part[c]) * (bin_edge(cut.bin) / UNIT) : 0.0);
    }
    __syncthreads();
    const double mine = l < a.chunks ? mass[l] : 0.0, upto = wave_scan(mine), total = __shfl(upto, 63), number = number_of(a, row) * total;
    const uint64_t past = __ballot(upto > number), some = __ballot(mine > 0.0);
    const int chunk = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
    const double before = chunk ? __shfl(upto, chunk - 1) : 0.0;
    constexpr int N = CHUNK / FT;
    float v[N];
#pragma unroll
    for (int k = 0; k < N / 4; ++k) x.four(chunk * CHUNK + (k * FT + t) * 4, v + 4 * k);
    draw<FT, N, false>(a, row, v, chunk * CHUNK, q, r, m.top, cut, number - before, total);
}

// ---- launches --------------------------------------------------------------------------------

// Tokens of a chunk: 4096, 16 of 256 threads, so that few long rows still reach many CUs; 16384 where there are blocks for all of them
// anyway, or more than 64 chunks otherwise.
int chunk_of(int rows, int vocab) {
    const int64_t blocks = static_cast<int64_t>(rows) * ((vocab + 4095) / 4096);
    return blocks <= 1024 && vocab <= MAXC * 4096 ? 4096 : 16384;
}
size_t workspace(int rows, int vocab) {
    if (vocab <= ROW_MOST || rows < 1) return 0;
    const int chunk = chunk_of(rows, vocab), chunks = (vocab + chunk - 1) / chunk;
    return static_cast<size_t>(rows) * (static_cast<size_t>(chunks) * (BINS + 1) * 8 + CAP * 8 + 4);
}

template <class T>
void launch(Args a, void *ws, hipStream_t s) {
    const dim3 rows(static_cast<unsigned>(a.rows));
    if (a.vocab <= 1024) hipLaunchKernelGGL((k_row<T, 256, 4>), rows, dim3(256), 0, s, a);
    else if (a.vocab <= 2048) hipLaunchKernelGGL((k_row<T, 256, 8>), rows, dim3(256), 0, s, a);
    else if (a.vocab <= 4096) hipLaunchKernelGGL((k_row<T, 512, 8>), rows, dim3(512), 0, s, a);
    else if (a.vocab <= 8192) hipLaunchKernelGGL((k_row<T, 1024, 8>), rows, dim3(1024), 0, s, a);
    else if (a.vocab <= ROW_MOST) hipLaunchKernelGGL((k_row<T, 1024, 16>), rows, dim3(1024), 0, s, a);
    else {
        const int chunk = chunk_of(a.rows, a.vocab);
        a.chunks = (a.vocab + chunk - 1) / chunk;
        a.bins = static_cast<uint64_t *>(ws);
        a.best = a.bins + static_cast<size_t>(a.rows) * a.chunks * BINS;
        a.list = a.best + static_cast<size_t>(a.rows) * a.chunks;
        a.listed = reinterpret_cast<int32_t *>(a.list + static_cast<size_t>(a.rows) * CAP);
        const dim3 grid(static_cast<unsigned>(a.rows) * a.chunks);
        if (chunk == 4096) {
            hipLaunchKernelGGL((k_bins<T, 256>), grid, dim3(256), 0, s, a);
            hipLaunchKernelGGL((k_list<T, 256>), grid, dim3(256), 0, s, a);
            hipLaunchKernelGGL((k_pick<T, 4096>), rows, dim3(FT), 0, s, a);
        } else {
            hipLaunchKernelGGL((k_bins<T, 1024>), grid, dim3(1024), 0, s, a);
            hipLaunchKernelGGL((k_list<T, 1024>), grid, dim3(1024), 0, s, a);
            hipLaunchKernelGGL((k_pick<T, 16384>), rows, dim3(FT), 0, s, a);
        }
    }
}

// ---- accepting drafts ------------------------------------------------------------------------

struct AcceptArgs {
    const int32_t *cu, *slot, *planned, *parent, *drafted, *sampled, *last;
    int32_t *path, *accept, *next;
    int n, n_rows, max_new, max_path, codes, ld_drafted, ld_sampled;
};

constexpr int AT = 256;
// A wave a request, a lane a row: whether its codes are those sampled at the row that it follows; then down the tree, one ballot a row.
__global__ void __launch_bounds__(AT) k_accept(AcceptArgs a) {
    const int i = blockIdx.x * (AT / WAVE) + (threadIdx.x >> 6), l = threadIdx.x & 63;
    if (i >= a.n) return;
    const int c0 = max(gld(a.cu + i), 0), count = min(gld(a.cu + i + 1), a.n_rows) - c0;
    const bool none = count > a.max_new || (a.planned && gld(a.planned + i) != 0);
    int parent = -2;
    bool fits = false;
    if (l < count && !none) {
        parent = a.parent ? gld(a.parent + c0 + l) : l - 1;
        fits = parent >= -1 && parent < l && gld(a.slot + c0 + l) >= 0;
        if (fits) {
            const int32_t *d = a.drafted + static_cast<size_t>(c0 + l) * a.ld_drafted;
            const int32_t *g = parent >= 0 ? a.sampled + static_cast<size_t>(c0 + parent) * a.ld_sampled : a.last ? a.last + static_cast<size_t>(i) * a.codes : nullptr;
            if (g) {
                bool same = true;
#pragma unroll 8
                for (int c = 0; c < a.codes; ++c) {
                    const int32_t x = gld(g + c);
                    same = same && x >= 0 && x == gld(d + c);
                }
                fits = same;
            }
        }
    }
    int at = -1, len = 0, mine = 0;
    while (len < a.max_path) {
        const uint64_t m = __ballot(fits && parent == at);
        if (!m) break;
        at = __builtin_ctzll(m);
        if (l == len) mine = at;
        ++len;
    }
    if (l < a.max_path) gst(a.path + static_cast<size_t>(i) * a.max_path + l, mine);
    if (l == 0) gst(a.accept + i, len);
    for (int c = l; c < a.codes; c += WAVE)
        gst(a.next + static_cast<size_t>(i) * a.codes + c, len > 0 ? gld(a.sampled + static_cast<size_t>(c0 + at) * a.ld_sampled + c)
                                                           : a.last ? gld(a.last + static_cast<size_t>(i) * a.codes + c) : -1);
}

} // namespace sample
} // namespace navi_amd

using namespace navi_amd;

extern "C" {

size_t navi_sample_workspace(int32_t n_rows, int32_t vocab) {
    return n_rows < 1 || vocab < 1 || vocab > (1 << 20) ? 0 : sample::workspace(n_rows, vocab);
}

navi_status navi_sample_rows(const void *d_logits, int32_t dtype, int32_t ld, int32_t n_rows, int32_t vocab, const navi_sample_rule *d_rules,
                             int32_t n_rules, const float *d_u, const uint32_t *d_allowed, int32_t ld_allowed, const uint32_t *d_seen,
                             int32_t ld_seen, int32_t *d_token, int32_t ld_token, float *d_logprob, void *d_ws, size_t ws_bytes, void *stream,
                             char *err, size_t errlen) {
    if (dtype != NAVI_DT_F32 && dtype != NAVI_DT_F16 && dtype != NAVI_DT_BF16) {
        set_err(err, errlen, "sample_rows: unsupported type %d (f32, f16 or bf16)", dtype);
        return NAVI_ERR_UNSUPPORTED;
    }
    const int words = (vocab + 31) / 32;
    if (n_rows < 0 || vocab < 1 || vocab > (1 << 20) || ld < vocab || (n_rules != 1 && n_rules != n_rows) || ld_token < 1 ||
        (d_allowed && ld_allowed != 0 && ld_allowed < words) || (d_seen && ld_seen != 0 && ld_seen < words)) {
        set_err(err, errlen, "sample_rows: out of range (rows %d, vocab %d, ld %d, rules %d, ld_allowed %d, ld_seen %d, ld_token %d)", n_rows, vocab, ld, n_rules,
                ld_allowed, ld_seen, ld_token);
        return NAVI_ERR_INVALID;
    }
    const uintptr_t four = reinterpret_cast<uintptr_t>(d_rules) | reinterpret_cast<uintptr_t>(d_u) | reinterpret_cast<uintptr_t>(d_allowed) |
                           reinterpret_cast<uintptr_t>(d_seen) | reinterpret_cast<uintptr_t>(d_token) | reinterpret_cast<uintptr_t>(d_logprob);
    if ((n_rows > 0 && (!d_logits || !d_rules || !d_u || !d_token)) || (four & 3u) || (reinterpret_cast<uintptr_t>(d_logits) & (dtype == NAVI_DT_F32 ? 3u : 1u))) {
        set_err(err, errlen, "sample_rows: a null or misaligned pointer");
        return NAVI_ERR_INVALID;
    }
    for (const void *out : {static_cast<const void *>(d_token), static_cast<const void *>(d_logprob)})
        for (const void *in : {d_logits, static_cast<const void *>(d_rules), static_cast<const void *>(d_u), static_cast<const void *>(d_allowed), static_cast<const void *>(d_seen)})
            if (out && out == in) {
                set_err(err, errlen, "sample_rows: d_token or d_logprob is one of the inputs, which other blocks still read");
                return NAVI_ERR_INVALID;
            }
    if (d_logprob && static_cast<const void *>(d_token) == d_logprob) {
        set_err(err, errlen, "sample_rows: d_token and d_logprob are one array");
        return NAVI_ERR_INVALID;
    }
    // up to 1024 threads a row, or a chunk of 16384 tokens, and a launch has less than 2^32
    if (static_cast<int64_t>(n_rows) * ((vocab + 16383) / 16384) * 1024 > UINT32_MAX) {
        set_err(err, errlen, "sample_rows: %d rows of %d tokens are too many for one call", n_rows, vocab);
        return NAVI_ERR_INVALID;
    }
    const size_t need = sample::workspace(n_rows, vocab);
    if (need > 0 && (!d_ws || !kv::aligned16(d_ws) || ws_bytes < need)) {
        set_err(err, errlen, "sample_rows: the workspace is null, misaligned or smaller than %zu bytes (%zu)", need, ws_bytes);
        return NAVI_ERR_INVALID;
    }
    kv::OnDevice dev;
    const navi_status st = dev.enter(stream, "sample_rows", err, errlen);
    if (st != NAVI_OK) return st;
    if (n_rows == 0) return NAVI_OK;
    sample::Args a{};
    a.x = d_logits;
    a.rules = d_rules;
    a.u = d_u;
    a.allowed = d_allowed;
    a.seen = d_seen;
    a.token = d_token;
    a.logprob = d_logprob;
    a.rows = n_rows;
    a.vocab = vocab;
    a.ld = ld;
    a.n_rules = n_rules;
    a.ld_allowed = ld_allowed;
    a.ld_seen = ld_seen;
    a.ld_token = ld_token;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == NAVI_DT_F32) sample::launch<float>(a, d_ws, s);
    else if (dtype == NAVI_DT_F16) sample::launch<_Float16>(a, d_ws, s);
    else sample::launch<__bf16>(a, d_ws, s);
    NAVI_TRY_HIP(hipGetLastError(), err, errlen);
    return NAVI_OK;
}

navi_status navi_draft_accept(const navi_kv_pages *pages, const int32_t *d_parent, const int32_t *d_drafted, int32_t ld_drafted, const int32_t *d_sampled,
                              int32_t ld_sampled, int32_t n_codes, const int32_t *d_last, int32_t *d_path, int32_t max_path, int32_t *d_accept,
                              int32_t *d_next, void *stream, char *err, size_t errlen) {
    navi_status st = kv::check_pages("draft_accept", pages, err, errlen);
    if (st != NAVI_OK) return st;
    if (!d_path || !d_accept || !d_next || (pages->n_rows > 0 && (!d_drafted || !d_sampled))) {
        set_err(err, errlen, "draft_accept: null argument");
        return NAVI_ERR_INVALID;
    }
    if (pages->max_new > 64 || max_path < 1 || max_path > 64 || n_codes < 1 || n_codes > 4096 || ld_drafted < n_codes || ld_sampled < n_codes) {
        set_err(err, errlen, "draft_accept: out of range (max_new %d, max_path %d, codes %d, ld_drafted %d, ld_sampled %d)", pages->max_new, max_path, n_codes,
                ld_drafted, ld_sampled);
        return NAVI_ERR_INVALID;
    }
    for (const int32_t *out : {d_path, d_accept, d_next})
        for (const int32_t *in : {static_cast<const int32_t *>(pages->cu_rows), static_cast<const int32_t *>(pages->row_slot), pages->status, d_parent, d_drafted, d_sampled})
            if (out == in) {
                set_err(err, errlen, "draft_accept: a result is one of the inputs, which other blocks still read");
                return NAVI_ERR_INVALID;
            }
    if (d_path == d_accept || d_path == d_next || d_accept == d_next || d_path == d_last || d_accept == d_last) {
        set_err(err, errlen, "draft_accept: d_path, d_accept and d_next are three arrays, and only d_next may be d_last");
        return NAVI_ERR_INVALID;
    }
    kv::OnDevice dev;
    if ((st = dev.enter(stream, "draft_accept", err, errlen)) != NAVI_OK) return st;
    const sample::AcceptArgs a{pages->cu_rows, pages->row_slot, pages->status, d_parent, d_drafted, d_sampled, d_last, d_path, d_accept, d_next, pages->n_requests,
                               pages->n_rows, pages->max_new, max_path, n_codes, ld_drafted, ld_sampled};
    const int per = sample::AT / WAVE;
    hipLaunchKernelGGL(sample::k_accept, dim3((pages->n_requests + per - 1) / per), dim3(sample::AT), 0, static_cast<hipStream_t>(stream), a);
    NAVI_TRY_HIP(hipGetLastError(), err, errlen);
    return NAVI_OK;
}

} // extern "C"

// A step's logits to its next codes on gfx950 (the C ABI's navi_sample_rows and navi_draft_accept): one token for every row under its
// own rule, and the drafted rows that the sampled codes confirm.
//
// Sampling. A row's tokens stand in the order of their logits x (the lowest index first among equals). Their weights are 2^(c (x - max)) with
// c = log2 e / temperature; a rule keeps the beginning of the order, and the token is the first, in the order of the indexes, at which the
// kept weights' running sum passes u of their total. So that the token is the definition's and not that of the sums' rounding, weights have few
// enough bits that a block's sums of equal ones are exact in 64: integers in units of 2^-31 of a bin's edge (2^-32 off at most) for the cuts and for rows
// in chunks, whose chunk and token are then found on one scale; 39 bits (computed to 2^-43) for the draw from a row that a block has whole.
//
//  * The order is cut into bins of a quarter of a power of two, floor(4 c x), 256 of them from the largest on (what is below 2^-63 has
//    no weight). One pass counts the tokens and sums the weights of every bin, one LDS atomic a token: the weight below bit 48, the count above.
//  * Sums over the bins, in a wave's registers, say in which bin top_k and top_p end. Only that bin's tokens are looked at again, by their
//    64-bit keys (logit, then index): down to 64 by digits of the key, and these each against all.
//  * Then the kept weights are summed in the order of the indexes, and the wave that holds the border names the token.
//
// Up to 16384 tokens a block has its row in LDS and does all of this in one launch: a chain of some twenty dependent steps, whose latencies bound it
// (one row of 2048 tokens with top_k 10 us, 512 rows 14.5, 8192 rows 98, a CU's instructions by then). Longer rows are cut into chunks of
// 4096 or 16384 tokens, in four launches: the chunks' bins (k_bins), the rows' (k_rows), the marked bins' tokens copied side by side (k_list),
// and one block a row for the rest, which reads again only the chunk that the number falls into (k_pick). 256 rows of 151936 f32 tokens, each
// with a rule of its own, take 91 us, of which k_bins 42 (156 MB at 3.7 TB/s; 20 instructions a token, all SIMDs issuing), k_rows 6,
// k_list 17 and k_pick 27, as long as its slowest row: a nucleus that ends among thousands of tokens of one bin. One row 30 to 45 us.
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
constexpr int CAP = 8192;              // tokens of the marked bins that are kept in LDS; where there are more, the row is read again
constexpr int ROW_MOST = 16384;        // tokens of a row that a block has in LDS
constexpr int MAXC = 64;               // most chunks of a row
constexpr int COPIES = 4;
constexpr unsigned long long ONE = 1ull << 48;   // a token in a sum of weights

struct Record;
struct Args {
    const void *x;
    const navi_sample_rule *rules;
    const float *u;
    const uint32_t *allowed, *seen;
    int32_t *token;
    float *logprob;
    // the workspace (launch): chunks' bins and largest keys; rows' sums and marked tokens; chunks' running sums of weights, and the largest logit of each
    // part of a chunk
    uint64_t *bins, *best, *sums, *list;
    double *upto;
    float *most;
    Record *record;
    int rows, vocab, ld, n_rules, ld_allowed, ld_seen, ld_token, chunks;
};

// A token's place in the order as a number, the first the largest. 0 comes after all of them.
__device__ __forceinline__ uint64_t key_of(float x, int i) { return static_cast<uint64_t>(float_key(x + 0.f)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(i)); }
__device__ __forceinline__ float logit_of(uint64_t key) { return key_float(static_cast<unsigned>(key >> 32)); }
__device__ __forceinline__ int index_of(uint64_t key) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key)); }

struct Rule {
    double c4;                         // 4 log2 e / temperature
    double inv;                        // 1 / c4
    double p, m;                       // top_p; log2 min_p
    double over, times;                // what a seen token's logit is multiplied with above 0 and below
    int k;                             // 0: off, as p of 1 and m of -inf are
    bool greedy, penal;
    __device__ __forceinline__ bool cuts() const { return k > 0 || p < 1.0 || m != -INFINITY; }
    // In 64 bits and rounded once: the product as it is, and the quotient too, since a quotient of two f32 lies at least 2^-49 of itself
    // from the middle between two others (below 2^-126, where they are further apart than that, the last bit may differ).
    __device__ __forceinline__ float seen(float v) const { return static_cast<float>(static_cast<double>(v) * (v > 0.f ? over : times)); }
};
__device__ __forceinline__ Rule rule_of(const Args &a, int row) {
    const navi_sample_rule *s = a.rules + (a.n_rules == 1 ? 0 : row);
    Rule r;
    const float t = gld(&s->temperature), p = gld(&s->top_p), m = gld(&s->min_p), pen = gld(&s->repetition_penalty);
    r.greedy = !(t > 0.f);
    // above 0 even for an infinite temperature, so that it times -inf is no NaN, and times the least number not 0
    r.c4 = r.greedy ? 1.0 : fmax(4.0 * 1.44269504088896340736 / static_cast<double>(t), 1e-60);
    r.k = max(gld(&s->top_k), 0);
    r.inv = 1.0 / r.c4;
    r.p = p < 1.f ? fmax(static_cast<double>(p), 0.0) : 1.0;
    r.m = -INFINITY;
    if (m > 0.f) r.m = log2(fmin(static_cast<double>(m), 1.0));
    r.penal = pen > 0.f && pen != 1.f;
    r.times = static_cast<double>(pen);
    r.over = 1.0 / r.times;
    return r;
}

// A row's logits: as they stand in memory, and as its rule sees them: -inf for what is not allowed, NaN and -inf; at most the
// largest finite number. (-0 is ordered as 0: key_of.)
template <class T>
struct Row {
    const T *x;
    const uint32_t *allowed, *seen;
    int vocab;
    bool vec;                          // four at a time are aligned
    __device__ __forceinline__ Row(const Args &a, int row) {
        x = static_cast<const T *>(a.x) + static_cast<size_t>(row) * a.ld;
        allowed = a.allowed ? a.allowed + static_cast<size_t>(row) * a.ld_allowed : nullptr;
        seen = a.seen ? a.seen + static_cast<size_t>(row) * a.ld_seen : nullptr;
        vocab = a.vocab;
        vec = (reinterpret_cast<uintptr_t>(x) & (4 * sizeof(T) - 1)) == 0;
    }
    static __device__ __forceinline__ float number(float v) { return v == v ? __builtin_amdgcn_fmed3f(v, -INFINITY, FLT_MAX) : -INFINITY; }
    __device__ __forceinline__ float at(int i, const Rule &r) const {
        float v = static_cast<float>(gld(x + i));
        if (seen && r.penal && gld(seen + (i >> 5)) >> (i & 31) & 1u) v = r.seen(v);
        return allowed && !(gld(allowed + (i >> 5)) >> (i & 31) & 1u) ? -INFINITY : number(v);
    }
    // tokens i .. i + 3, i a multiple of 4; -inf past the last
    __device__ __forceinline__ void load(int i, float *v) const {
        if (vec && i + 4 <= vocab) {
            typedef T T4 __attribute__((ext_vector_type(4)));
            const T4 t = *(const NAVI_GLOBAL T4 *) (x + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(t[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = i + e < vocab ? static_cast<float>(gld(x + i + e)) : -INFINITY;
        }
    }
    __device__ __forceinline__ void see(int i, float *v, const Rule &r) const {
        if (seen && r.penal) {
            const uint32_t w = i < vocab ? gld(seen + (i >> 5)) >> (i & 31) : 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = w >> e & 1u ? r.seen(v[e]) : v[e];
        }
        const uint32_t w = allowed && i < vocab ? gld(allowed + (i >> 5)) >> (i & 31) : 15u;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = w >> e & 1u ? number(v[e]) : -INFINITY;
    }
};
// Thread t's N tokens of a block's: 4 from i0 + 4 (k BT + t).
template <int BT>
__device__ __forceinline__ int token_at(int i0, int i) { return i0 + (i / 4 * BT + static_cast<int>(threadIdx.x)) * 4 + i % 4; }
template <int BT, int N, class T>
__device__ __forceinline__ void load_all(const Row<T> &x, int i0, float (&v)[N]) {
#pragma unroll
    for (int k = 0; k < N; k += 4) x.load(token_at<BT>(i0, k), v + k);
}
template <int BT, int N, class T>
__device__ __forceinline__ void see_all(const Row<T> &x, int i0, float (&v)[N], const Rule &r) {
#pragma unroll
    for (int k = 0; k < N; k += 4) x.see(token_at<BT>(i0, k), v + k, r);
}

// The largest key of a block's tokens, 0 without one, and for each part of a wave's (256 tokens) its largest logit. `index`: whether the key's
// index is wanted (else that of some token).
template <int BT, int PARTS>
__device__ __forceinline__ uint64_t block_best(const float (&v)[4 * PARTS], int i0, float (&most)[PARTS], bool index, float *red, int *red_at) {
    const int l = threadIdx.x & 63, wv = threadIdx.x >> 6;
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
        most[k] = wave_max(fmaxf(fmaxf(v[4 * k], v[4 * k + 1]), fmaxf(v[4 * k + 2], v[4 * k + 3])));
        m = fmaxf(m, most[k]);
    }
    if (l == 0) red[wv] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int i = 1; i < BT / WAVE; ++i) m = fmaxf(m, red[i]);
    if (m == -INFINITY) return 0;
    if (!index) return key_of(m, i0);
    int at = INT32_MAX;
#pragma unroll
    for (int i = 4 * PARTS - 1; i >= 0; --i) at = v[i] == m ? token_at<BT>(i0, i) : at;
    at = wave_min_int(at);
    if (l == 0) red_at[wv] = at;
    __syncthreads();
    at = red_at[0];
#pragma unroll
    for (int i = 1; i < BT / WAVE; ++i) at = min(at, red_at[i]);
    return key_of(m, at);
}
// The block's 4 BT PARTS tokens from i0 on into LDS as the rule sees them. A thread uses only those that it has put there (token_at) until the
// next barrier.
template <int BT, int PARTS, class T>
__device__ __forceinline__ void keep(const float (&v)[4 * PARTS], float *xs) {
#pragma unroll
    for (int k = 0; k < PARTS; ++k) *reinterpret_cast<f32x4_t *>(xs + token_at<BT>(0, 4 * k)) = f32x4_t{v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
}

// A weight over its bin's edge, 2^(f / 4) for 0 <= f < 1: Taylor's polynomial about the middle, its eighth power 2^-43. In units of 2^-31 and
// rounded: one through Chebyshev's points, 2^-35 at most from it, its mean 2^-40.
constexpr double UNIT = 2147483648.0;
constexpr double LN = 0.25 * 0.693147180559945309417;
__device__ __forceinline__ double quarter(double f) {
    const double g = f - 0.5;
    constexpr double M = 1.09050773266525765921;                  // 2^(1 / 8)
    constexpr double C1 = LN, C2 = C1 * LN / 2, C3 = C2 * LN / 3, C4 = C3 * LN / 4, C5 = C4 * LN / 5, C6 = C5 * LN / 6, C7 = C6 * LN / 7;
    double s = C7 * M;
    s = fma(s, g, C6 * M);
    s = fma(s, g, C5 * M);
    s = fma(s, g, C4 * M);
    s = fma(s, g, C3 * M);
    s = fma(s, g, C2 * M);
    s = fma(s, g, C1 * M);
    return fma(s, g, M);
}
// The constants in registers that the compiler takes as they come: written as such, it moves each into the sum's register first, three
// instructions a step.
struct Units {
    double c[6];
    __device__ __forceinline__ Units() {
        const double k[6] = {0.9999999999802172 * UNIT + 0.5, 0.1732867965638913 * UNIT,    0.015014140101979987 * UNIT,
                             0.0008673221940371589 * UNIT,    3.743580564591298e-05 * UNIT, 1.4203366711186339e-06 * UNIT};
#pragma unroll
        for (int i = 0; i < 6; ++i) {
            c[i] = k[i];
            if (i < 5) asm("" : "+s"(c[i]));
            else asm("" : "+v"(c[i]));
        }
    }
    __device__ __forceinline__ uint32_t of(double f) const {
        double s = fma(c[5], f, c[4]);
        s = fma(s, f, c[3]);
        s = fma(s, f, c[2]);
        s = fma(s, f, c[1]);
        return static_cast<uint32_t>(fma(s, f, c[0]));
    }
};
__device__ __forceinline__ uint32_t units(double f) { return Units().of(f); }
// 2^(-j / 4)
__device__ __forceinline__ double bin_edge(int j) {
    const double q[4] = {1.0, 0.840896415253714543031, 0.707106781186547524401, 0.594603557501360533359};
    const double f = (j & 3) == 0 ? q[0] : (j & 3) == 1 ? q[1] : (j & 3) == 2 ? q[2] : q[3];
    return ldexp(f, -(j >> 2));
}

// A token's bin below the row's (or chunk's) first, BINS: none of them, and its place in it.
struct Place {
    int j;
    double f;
};
__device__ __forceinline__ Place place_of(float x, double c4, double top) {
    const double q = static_cast<double>(x) * c4, b = floor(q);   // -inf: in no bin
    return Place{static_cast<int>(fmin(top - b, static_cast<double>(BINS))), q - b};
}
__device__ __forceinline__ int bin_of(float x, double c4, double top) { return place_of(x, c4, top).j; }

// The least float key whose logit reaches a border: reaches(x) is true from some x on. One more than the largest's: none does. Halving from the
// two keys beside the guess, which hold the border unless the guess is poor; 35 steps at most.
constexpr uint32_t KEY_LEAST = 0x00800000u, KEY_MOST = 0xFF7FFFFFu;   // of -FLT_MAX and FLT_MAX
template <class F>
__device__ __forceinline__ uint32_t least_key(double guess, F reaches) {
    const uint32_t k = float_key(static_cast<float>(fmin(fmax(guess, -static_cast<double>(FLT_MAX)), static_cast<double>(FLT_MAX))));
    uint32_t lo = KEY_LEAST, hi = KEY_MOST + 1u;                  // the border lies within
    auto probe = [&](uint32_t at) {
        if (reaches(key_float(at))) hi = at;
        else lo = at + 1u;
    };
    if (k - 2u > lo) probe(k - 2u);
    if (k + 2u >= lo && k + 2u < hi) probe(k + 2u);
    while (lo < hi) probe(lo + (hi - lo) / 2u);
    return lo;
}
__device__ __forceinline__ uint32_t bin_start(int j, const Rule &r, double top) {
    const double b = top - j;
    return j < 0 ? KEY_MOST + 1u : least_key(b * r.inv, [&](float x) { return floor(static_cast<double>(x) * r.c4) >= b; });
}
// Keys from lo on, len of them.
struct Keys {
    uint64_t lo, len;
    __device__ __forceinline__ bool have(uint64_t k) const { return k - lo < len; }
    // those of them from `from` on, n at most: a part, or a digit's keys, may reach past a bin's ends
    __device__ __forceinline__ Keys part(uint64_t from, uint64_t n) const {
        const uint64_t first = max(lo, from), last = min(lo + (len - 1), from + (n - 1));
        return Keys{first, first <= last ? last - first + 1 : 0};
    }
};
__device__ __forceinline__ Keys between(uint32_t lo, uint32_t hi) { return Keys{static_cast<uint64_t>(lo) << 32, static_cast<uint64_t>(hi - lo) << 32}; }
// The least float key that min_p leaves (m > -inf).
__device__ __forceinline__ uint32_t least_of(const Rule &r, double best4) {
    return least_key((best4 + 4.0 * r.m) * r.inv, [&](float x) { return (static_cast<double>(x) * r.c4 - best4) * 0.25 >= r.m; });
}

// Adds a token to its bin, if it has one. The instructions are what bounds a pass over a row: 15 vector ones a token, four scalar ones and its atomic. (The conversion
// takes numbers past its range to its ends; so written, since C++ leaves them undefined.)
struct Adder {
    double c4, top;
    Units un;
    __device__ __forceinline__ void add(unsigned long long *w, float x) const {
        const double q = static_cast<double>(x) * c4, b = floor(q), d = top - b;
        int j;
        asm("v_cvt_i32_f64 %0, %1" : "=v"(j) : "v"(d));
        if (static_cast<unsigned>(j) < BINS) atomicAdd(w + j, ONE + un.of(q - b));
    }
};

// ---- 64 bits over a wave: DPP moves of both halves (dev_common.h has the patterns) --------------

template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xF, false);
    return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, int l) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), l), hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), l);
    return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ double as_double(uint64_t v) { return __longlong_as_double(static_cast<long long>(v)); }
__device__ __forceinline__ uint64_t as_bits(double v) { return static_cast<uint64_t>(__double_as_longlong(v)); }
__device__ __forceinline__ double lane_double(double v, int l) { return as_double(lane64(as_bits(v), l)); }

// Inclusive sums over the lanes; what a move does not reach adds 0.
template <int CTRL, int ROWS>
__device__ __forceinline__ void scan_step(double &v) { v += as_double(dpp64<CTRL, ROWS>(as_bits(v))); }
template <int CTRL, int ROWS>
__device__ __forceinline__ void scan_step(uint64_t &v) { v += dpp64<CTRL, ROWS>(v); }
template <class V>
__device__ __forceinline__ V wave_scan(V v) {
    scan_step<0x111, 0xF>(v);
    scan_step<0x112, 0xF>(v);
    scan_step<0x114, 0xF>(v);
    scan_step<0x118, 0xF>(v);
    scan_step<0x142, 0xA>(v);
    scan_step<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
    v = max(v, dpp64<0x111, 0xF>(v));
    v = max(v, dpp64<0x112, 0xF>(v));
    v = max(v, dpp64<0x114, 0xF>(v));
    v = max(v, dpp64<0x118, 0xF>(v));
    v = max(v, dpp64<0x142, 0xA>(v));
    v = max(v, dpp64<0x143, 0xC>(v));
    return lane64(v, 63);
}

template <int BT>
struct Lds {
    static constexpr int NW = BT / WAVE;
    unsigned long long w[COPIES][BINS];    // sums of the bins' weights, counts above bit 48, by lane: fewer of an instruction meet; then of a digit's tokens
    unsigned n[BINS];                  // counts that may pass 16 bits
    unsigned long long red[2][NW];
    int at[NW];                        // of block_best
    float most[NW];
    double seg[64];
    unsigned long long few[WAVE];      // the tokens that are left to rank
    uint32_t unit[WAVE];
    unsigned long long key, sum;
    int listed;
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

// A row's bins in a wave's registers, lane l with bins 4 l .. 4 l + 3, and their sums: every wave looks for itself, without barriers.
struct Edge {
    int bin, count, own;               // BINS: none; the tokens before it, and in it
    double before, upto;               // weights before it, and with it, in units of the first bin's edge
};
struct Bins {
    int n[4], first;
    double w[4], before, all;
    int tokens;
    __device__ __forceinline__ Bins(const int (&count)[4], const uint64_t (&mass)[4]) {
        const int l = threadIdx.x & 63;
        int c = 0;
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            n[i] = count[i];
            w[i] = static_cast<double>(mass[i]) * ldexp(bin_edge(i) / UNIT, -l);
            c += n[i];
            s += w[i];
        }
        first = wave_incl_scan(c) - c;
        const double upto = wave_scan(s);
        all = lane_double(upto, 63);
        before = __shfl_up(upto, 1);
        if (l == 0) before = 0.0;
        tokens = __builtin_amdgcn_readlane(first + c, 63);
    }
    // the bin in which the first k tokens end
    __device__ __forceinline__ Edge of_count(int k) const {
        Edge e{BINS, 0, 0, 0.0, all};
        if (k < 1 || k >= tokens) return e;
        int c = first, bin = -1, cb = 0, own = 0;
        double s = before, sb = 0.0, su = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (c < k && c + n[i] >= k) { bin = 4 * static_cast<int>(threadIdx.x & 63) + i; cb = c; own = n[i]; sb = s; su = s + w[i]; }
            c += n[i];
            s += w[i];
        }
        return take(__builtin_ctzll(__ballot(bin >= 0)), bin, cb, own, sb, su);
    }
    // the one in which the weights reach `mass`; where rounding keeps their sum below it, the last that has a token
    __device__ __forceinline__ Edge of_mass(double mass) const {
        int bin = -1, cb = 0, own = 0, last = -1, lc = 0, ln = 0, c = first;
        double sb = 0.0, su = 0.0, lb = 0.0, lu = 0.0, s = before;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double u = s + w[i];
            if (n[i] > 0) {
                last = 4 * static_cast<int>(threadIdx.x & 63) + i; lc = c; ln = n[i]; lb = s; lu = u;
                if (bin < 0 && u >= mass) { bin = last; cb = c; own = n[i]; sb = s; su = u; }
            }
            c += n[i];
            s = u;
        }
        const uint64_t hit = __ballot(bin >= 0);
        if (hit) return take(__builtin_ctzll(hit), bin, cb, own, sb, su);
        return take(63 - __builtin_clzll(__ballot(last >= 0)), last, lc, ln, lb, lu);
    }
    static __device__ __forceinline__ Edge take(int lane, int bin, int c, int own, double b, double u) {
        return Edge{__builtin_amdgcn_readlane(bin, lane), __builtin_amdgcn_readlane(c, lane), __builtin_amdgcn_readlane(own, lane), lane_double(b, lane),
                    lane_double(u, lane)};
    }
};

// The bins whose tokens are looked at again: the one in which top_k ends, and p0 .. p1, in one of which top_p does.
struct Marks {
    Edge k;
    int p0, p1, own;                   // own: the tokens in p0
    __device__ __forceinline__ Marks(const Bins &b, const Rule &r) {
        k = b.of_count(r.k);
        p0 = BINS;
        p1 = -1;
        own = 0;
        if (r.p < 1.0) {
            const Edge e = b.of_mass(r.p * (k.bin < BINS ? k.before : b.all));
            p0 = e.bin;
            own = e.own;
            p1 = k.bin < BINS ? b.of_mass(r.p * k.upto).bin : p0;
        }
    }
    // whether the parts' sums are made of top_k's bin, and of top_p's if that is one: where the tokens are too many to rank at once
    __device__ __forceinline__ bool fine_k() const { return k.bin < BINS && k.own > WAVE; }
    __device__ __forceinline__ bool fine_p() const { return p0 == p1 && own > WAVE; }
};

// Tokens to look at again: keys in LDS, or, where they are too many, all of the row's, SPAN at a time in LDS as the rule sees them (WHOLE: there already).
// A thread reads back those that it has put there. Rows so flat are slow, since one block goes over all of the row several times: 151936 normal logits with
// sigma 0.3, of which the largest bin has a quarter, 310 us, 256 such rows 430 to 540 (418 and 726 with the logits loaded one by one); all alike 530.
template <class T, int BATCH, int SPAN, bool WHOLE>
struct Tokens {
    typedef uint64_t Batch[BATCH];
    const unsigned long long *key;
    float *xs;
    int n;
    bool held;
    const Row<T> &row;
    const Rule &r;
    double top;
    // tokens i0 .. i0 + SPAN - 1 into xs
    template <int BT>
    __device__ __forceinline__ void bring(int i0) const {
        if constexpr (!WHOLE) {
            float v[SPAN / BT];
            load_all<BT>(row, i0, v);
            see_all<BT>(row, i0, v, r);
            keep<BT, SPAN / BT / 4, T>(v, xs);
        }
    }
    // the key of the thread's j-th of these, 0: none
    template <int BT>
    __device__ __forceinline__ uint64_t brought(int i0, int j) const {
        const int i = token_at<BT>(0, j);
        const float x = xs[i];
        return x == -INFINITY ? 0 : key_of(x, i0 + i);
    }
    // f(keys) of the thread's tokens, BATCH at a time (0: none), so that their loads and sums overlap
    template <int BT, class F>
    __device__ __forceinline__ void each(F f) const {
        const int end = held ? n - (threadIdx.x & ~63) : row.vocab, step = held ? BATCH * BT : SPAN;
#pragma unroll 1
        for (int i0 = 0; i0 < end; i0 += step) {
            if (!held) bring<BT>(i0);
#pragma unroll 1
            for (int b = 0; b < (held ? BATCH : SPAN / BT); b += BATCH) {
                Batch k;
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    if (held) {
                        const int i = i0 + j * BT + threadIdx.x;
                        k[j] = i < n ? key[i] : 0;
                    } else {
                        k[j] = brought<BT>(i0, b + j);
                    }
                }
                f(k);
            }
        }
    }
    __device__ __forceinline__ uint32_t units_of(uint64_t k) const { return units(place_of(logit_of(k), r.c4, top).f); }
};

// Of the n <= 64 keys q.few (weights q.unit), largest first: the one at which their count reaches `need`, or (need 0) their weights' sum `mass` in
// units; none: the last. `sum`: plus the weights up to it and with it. Each key against all of them, BT / 64 lanes a key. All threads, after a barrier.
template <int BT>
__device__ __forceinline__ uint64_t rank(Lds<BT> &q, int n, int need, double mass, uint64_t &sum) {
    constexpr int G = BT / WAVE;
    static_assert(G == 4 || G == 8, "");
    const int i = threadIdx.x / G;
    const uint64_t key = i < n ? q.few[i] : 0;
    int place = 0;
    uint64_t before = 0;
#pragma unroll 4
    for (int j = threadIdx.x % G; j < n; j += G) {
        const bool ahead = q.few[j] > key;
        place += ahead;
        before += ahead ? q.unit[j] : 0u;
    }
    auto all = [&](auto move) {                                   // the sum with the lanes that `move` takes from
        place += static_cast<int>(move(static_cast<uint64_t>(place)));
        before += move(before);
    };
    all([](uint64_t v) { return dpp64<0xB1, 0xF>(v); });          // quad_perm [1,0,3,2]
    all([](uint64_t v) { return dpp64<0x4E, 0xF>(v); });          // quad_perm [2,3,0,1]
    if (G == 8) all([](uint64_t v) { return dpp64<0x141, 0xF>(v); });   // row_half_mirror
    const uint64_t upto = before + (key ? q.unit[i] : 0u);
    const bool reached = need > 0 ? place == need - 1 : static_cast<double>(upto) >= mass && (place == 0 || static_cast<double>(before) < mass);
    const bool last = place == n - 1 && (need > 0 ? need > n : static_cast<double>(upto) < mass);
    if (threadIdx.x % G == 0 && key && (reached || last)) {
        q.key = key;
        q.sum = upto;
    }
    __syncthreads();
    sum += n > 0 ? q.sum : 0;
    return n > 0 ? q.key : 0;
}

// Sums of weights and counts of 256 parts of a marked bin's float keys, of 2^shift keys each; or null.
struct Fine {
    const uint64_t *sums;
    int shift;
};
__device__ __forceinline__ int fine_shift(uint32_t len) { return len > 256u ? 24 - __builtin_clz(len - 1u) : 0; }

// The digit in which the count reaches `need`, or (need 0) the weights `mass`; these and `sum` then without the digits above, n: its count. Lane l has
// the counts and weights of digits 255 - 4 l .. 252 - 4 l; every wave finds it for itself.
__device__ __forceinline__ int digit_of(const int (&c)[4], const uint64_t (&w)[4], int &n, int &need, double &mass, uint64_t &sum) {
    const int l = threadIdx.x & 63, cs = c[0] + c[1] + c[2] + c[3];
    const uint64_t ws = w[0] + w[1] + w[2] + w[3];
    int cb = wave_incl_scan(cs) - cs;
    uint64_t wb = wave_scan(ws) - ws;
    int d = -1, dc = 0, dn = 0, last = -1, lc = 0, ln = 0;
    uint64_t db = 0, lb = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool reached = need > 0 ? cb + c[i] >= need : static_cast<double>(wb + w[i]) >= mass;
        if (c[i] > 0) {
            if (d < 0 && reached) { d = 255 - 4 * l - i; dc = cb; dn = c[i]; db = wb; }
            last = 255 - 4 * l - i; lc = cb; ln = c[i]; lb = wb;
        }
        cb += c[i];
        wb += w[i];
    }
    const uint64_t hit = __ballot(d >= 0);
    const uint64_t any = __ballot(last >= 0);
    int src;
    if (hit) {
        src = __builtin_ctzll(hit);
    } else if (!any) {
        n = 0;
        return 0;
    } else {                                                      // the sum falls short of the mass by its rounding: the last one
        src = 63 - __builtin_clzll(any);
        d = last; dc = lc; dn = ln; db = lb;
    }
    need -= need > 0 ? __builtin_amdgcn_readlane(dc, src) : 0;
    db = lane64(db, src);
    mass -= static_cast<double>(db);
    sum += db;
    n = __builtin_amdgcn_readlane(dn, src);
    return __builtin_amdgcn_readlane(d, src);
}

// The same as rank for the n tokens of `in`; all threads. Up to 64 are ranked. More: first by the fine sums, if there are any; then the block narrows
// them by a digit of 8 bits, from the highest in which their keys differ (f16 logits have few different values, and indexes few
// different bits). q.w, q.n and q.few are used.
template <int BT, class S>
__device__ __forceinline__ uint64_t select(const S &s, Lds<BT> &q, Keys in, int n, const Fine &fine, int need, double mass, uint64_t &sum) {
    const int t = threadIdx.x, l = t & 63;
    sum = 0;
    if (fine.sums) {
        int c[4];
        uint64_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = gld(fine.sums + 255 - 4 * l - i);
            c[i] = static_cast<int>(gld(fine.sums + BINS + 255 - 4 * l - i));
        }
        const int d = digit_of(c, w, n, need, mass, sum);
        in = in.part(in.lo + (static_cast<uint64_t>(d) << (32 + fine.shift)), uint64_t(1) << (32 + fine.shift));
    }
#pragma unroll 1
    while (n > WAVE) {
        __syncthreads();                                          // what the round before, or the caller, has left here has been read
        for (int i = t; i < COPIES * BINS; i += BT) q.w[0][i] = 0;
        if (t < BINS) q.n[t] = 0;
        uint64_t hi = 0, lo = 0;                                  // lo: of the complements
        s.template each<BT>([&](const typename S::Batch &k) {
#pragma unroll
            for (const uint64_t x : k) {
                const bool on = in.have(x);
                hi = max(hi, on ? x : 0);
                lo = max(lo, on ? ~x : 0);
            }
        });
        hi = wave_max64(hi);
        lo = wave_max64(lo);
        if (l == 63) {
            q.red[0][t >> 6] = hi;
            q.red[1][t >> 6] = lo;
        }
        __syncthreads();
        hi = lo = 0;
#pragma unroll
        for (int i = 0; i < Lds<BT>::NW; ++i) {
            hi = max(hi, static_cast<uint64_t>(q.red[0][i]));
            lo = max(lo, static_cast<uint64_t>(q.red[1][i]));
        }
        lo = ~lo;
        if (hi <= lo) break;                                      // one token, or (where the counts cannot be right) none
        const int h = 64 - __builtin_clzll(hi ^ lo), width = min(h, 8), at = h - width;   // bits from h on are alike
        s.template each<BT>([&](const typename S::Batch &k) {
#pragma unroll
            for (const uint64_t x : k) {
                if (!in.have(x)) continue;
                const unsigned d = static_cast<unsigned>(x >> at) & ((1u << width) - 1u);
                atomicAdd(&q.w[t & (COPIES - 1)][d], (s.held ? ONE : 0ull) + s.units_of(x));
                if (!s.held) atomicAdd(&q.n[d], 1u);
            }
        });
        __syncthreads();
        int c[4];
        uint64_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 255 - 4 * l - i;
            w[i] = 0;
#pragma unroll
            for (int j = 0; j < COPIES; ++j) w[i] += q.w[j][d];
            c[i] = s.held ? static_cast<int>(w[i] >> 48) : static_cast<int>(q.n[d]);
            if (s.held) w[i] &= ONE - 1;
        }
        const uint64_t above = h < 64 ? hi >> h << h : 0;
        in = in.part(above | static_cast<uint64_t>(digit_of(c, w, n, need, mass, sum)) << at, uint64_t(1) << at);
    }
    __syncthreads();
    if (t == 0) q.listed = 0;
    __syncthreads();
    s.template each<BT>([&](const typename S::Batch &k) {
#pragma unroll
        for (const uint64_t x : k)
            if (in.have(x)) {
                const int at = atomicAdd(&q.listed, 1);
                if (at < WAVE) {                                  // as many as there are
                    q.few[at] = x;
                    q.unit[at] = s.units_of(x);
                }
            }
    });
    __syncthreads();
    return rank(q, min(q.listed, WAVE), need, mass, sum);
}

// The last of the order that is kept: keys from `key` on, the last of them in `bin` (BINS: all are kept).
struct Cut {
    uint64_t key;
    int bin;
    __device__ __forceinline__ Cut() : key(static_cast<uint64_t>(KEY_LEAST) << 32), bin(BINS) {}
    __device__ __forceinline__ void narrow(int b, uint64_t k) {
        if (k > key) {
            key = k;
            bin = b;
        }
    }
};

// The float keys of the marked bins, a lane a border.
struct Ranges {
    uint32_t k0, k1, p0, p1;           // top_k's bin, top_p's bins: first key, one past the last
    __device__ __forceinline__ Ranges(const Marks &m, const Rule &r, double top) {
        const int l = threadIdx.x & 3, j = l == 0 ? m.k.bin : l == 1 ? m.k.bin - 1 : l == 2 ? m.p1 : m.p0 - 1;
        const uint32_t start = bin_start(j, r, top);
        k0 = __builtin_amdgcn_readlane(start, 0);
        k1 = __builtin_amdgcn_readlane(start, 1);
        p0 = __builtin_amdgcn_readlane(start, 2);
        p1 = __builtin_amdgcn_readlane(start, 3);
        if (m.k.bin >= BINS) k0 = k1 = 0u;
        if (m.p0 > m.p1) p0 = p1 = 0u;
    }
    __device__ __forceinline__ bool has(uint32_t k) const { return k - k0 < k1 - k0 || k - p0 < p1 - p0; }
    __device__ __forceinline__ uint32_t least() const { return min(k0 < k1 ? k0 : ~0u, p0 < p1 ? p0 : ~0u); }
};

// What top_k and top_p keep, from the bins' sums and the tokens of the marked bins.
template <int BT, class S>
__device__ __forceinline__ void cut_tokens(Cut &cut, const S &s, Lds<BT> &q, const Rule &r, const Bins &bins, double top, const Marks &marks, const Ranges &ranges,
                                           const uint64_t *fine) {
    double all = bins.all;
#pragma unroll 1
    for (int by = 0; by < 2; ++by) {                              // top_k, then top_p of what it leaves: one copy of the code
        if (by == 0 ? marks.k.bin >= BINS : r.p >= 1.0) continue;
        Keys in = between(ranges.k0, ranges.k1);
        int bin = marks.k.bin, n = marks.k.own, need = r.k - marks.k.count;
        double mass = 0.0;
        if (by == 1) {
            // between p0 and p1 whatever the rounding of the sums
            mass = r.p * all;
            Edge e = bins.of_mass(mass);
            if (e.bin < marks.p0 || e.bin > marks.p1) e = bins.of_mass(r.p * (marks.k.bin < BINS ? marks.k.upto : bins.all));
            bin = e.bin;
            n = e.own;
            need = 0;
            mass = (mass - e.before) * (UNIT / bin_edge(bin));
            in = marks.p0 == marks.p1 ? between(ranges.p0, ranges.p1) : between(bin_start(bin, r, top), bin_start(bin - 1, r, top));
        }
        uint64_t sum;
        const bool parts = fine && (by == 0 ? marks.fine_k() : marks.fine_p());
        cut.narrow(bin, select(s, q, in, n, Fine{parts ? fine + by * 2 * BINS : nullptr, fine_shift(static_cast<uint32_t>(in.len >> 32))}, need, mass, sum));
        if (by == 0) all = marks.k.before + static_cast<double>(sum) * (bin_edge(bin) / UNIT);
    }
}

// log x of 2^-64 < x < 2^64 in 64 bits (2^-41): a 32-bit logarithm l, and with x 2^-l = 1 + d, |d| < 2^-18, the series of log(1 + d).
__device__ __forceinline__ double log_of(double x) {
    const double l = static_cast<double>(__builtin_amdgcn_logf(static_cast<float>(x))), q = -4.0 * l, b = floor(q);
    const double d = x * quarter(q - b) * bin_edge(-static_cast<int>(b)) - 1.0;
    return l * (4.0 * LN) + d * (1.0 - d * (0.5 - d * (1.0 / 3.0)));
}

__device__ __forceinline__ void put(const Args &a, int row, int token, float logprob) {
    gst(a.token + static_cast<size_t>(row) * a.ld_token, token);
    if (a.logprob) gst(a.logprob + row, logprob);
}

// The first token of the 4 BT PARTS in LDS (from i0 on) at which the kept weights' sum passes `number` (FROM_U: that part of the sum); none
// passes it: the last kept one. `total`: the sum of all kept weights of the row, for the log probability (FROM_U: of those here).
// Equal tokens, which 16-bit logits often have, are on a border between them for many a u: there the sums have to be those of real numbers. FROM_U: 39 bits
// of a weight leave 14 for the 16384 tokens of a row. Else the weights are those of which `number` and `total` were made, the chunks' units: two
// roundings of one weight, 2^-32 apart, would put the number on the wrong side.
template <int BT, int PARTS, bool FROM_U>
__device__ __forceinline__ void draw(const Args &a, int row, const float *xs, int i0, Lds<BT> &q, const Rule &r, double top, const Cut &cut, double number,
                                     double total) {
    constexpr int NW = BT / WAVE;
    static_assert(PARTS * NW <= 64, "a segment a lane");
    const int t = threadIdx.x, l = t & 63, wv = t >> 6;
    const Units un;
    auto weight = [&](float x, int i) {                           // of token i, 0 where it is not kept
        double w = 0.0;
        if (key_of(x, i0 + i) >= cut.key) {
            const Place p = place_of(x, r.c4, top);
            if (p.j < BINS) w = FROM_U ? as_double(as_bits(quarter(p.f) * bin_edge(p.j)) & ~uint64_t(0x3FFF)) : un.of(p.f) * (bin_edge(p.j) / UNIT);
        }
        return w;
    };
    auto four = [&](int k, f32x4_t &x) {                          // of the thread's four in part k
        const int i = token_at<BT>(0, 4 * k);
        x = *reinterpret_cast<const f32x4_t *>(xs + i);
        double w = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w += weight(x[e], i + e);
        return w;
    };
    f32x4_t x;
    constexpr int AT_ONCE = PARTS < 4 ? PARTS : 4;                // that many parts' sums overlap
#pragma unroll 1
    for (int k = 0; k < PARTS; k += AT_ONCE) {
        double sum[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) sum[j] = four(k + j, x);
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            sum[j] = wave_scan(sum[j]);
            if (l == 63) q.seg[(k + j) * NW + wv] = sum[j];
        }
    }
    __syncthreads();
    const double mine = l < PARTS * NW ? q.seg[l] : 0.0, upto = wave_scan(mine);
    if (FROM_U) {
        total = lane_double(upto, 63);
        number *= total;
    }
    // only where something is kept: the lanes' sums associate differently, so that one that adds nothing can be a rounding above the one before it
    const uint64_t past = __ballot(mine > 0.0 && upto > number), some = __ballot(mine > 0.0);
    if (!some) {                                                  // nothing is: the logits have been written to meanwhile
        if (t == 0) put(a, row, -1, -INFINITY);
        return;
    }
    const int seg = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
    if (seg % NW != wv) return;
    const double before = seg ? lane_double(upto, seg - 1) : 0.0, log_total = a.logprob ? log_of(total) : 0.0;
    const double own = four(seg / NW, x), sum = before + wave_scan(own);
    const uint64_t over = __ballot(own > 0.0 && sum > number), any = __ballot(own > 0.0);
    if (l != (over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any))) return;
    double run = sum - own;
    float y = 0.f;
    int pick = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int i = token_at<BT>(0, 4 * (seg / NW)) + e;
        const double w = weight(x[e], i);
        if (w > 0.0 && (pick < 0 || run <= number)) {
            pick = i0 + i;
            y = x[e];
            run += w;
        }
    }
    // the logarithm of a weight is what it was made from; the sum's rounding can put a lone token's above 0
    put(a, row, pick, fminf(static_cast<float>((static_cast<double>(y) * r.c4 - top) * LN - log_total), 0.f));
}

__device__ __forceinline__ double number_of(const Args &a, int row) {
    const float u = gld(a.u + row);
    return u > 0.f ? static_cast<double>(fminf(u, 0x1.fffffep-1f)) : 0.0;
}

// ---- a row a block ---------------------------------------------------------------------------

template <class T, int BT, int PARTS>
__global__ void __launch_bounds__(BT) k_row(Args a) {
    constexpr int MOST = 4 * BT * PARTS, HELD = MOST < CAP ? MOST : CAP;
    __shared__ Lds<BT> q;
    __shared__ __align__(16) float xs[MOST];
    __shared__ unsigned long long list[HELD];
    const int row = blockIdx.x, t = threadIdx.x, l = t & 63;
    const Row<T> x(a, row);
    uint64_t best;
    Rule r;
    double number;
    {
        float v[4 * PARTS];
        load_all<BT>(x, 0, v);
        number = number_of(a, row);
        r = rule_of(a, row);
        for (int i = t; i < COPIES * BINS; i += BT) q.w[0][i] = 0;
        if (t == 0) q.listed = 0;
        see_all<BT>(x, 0, v, r);
        keep<BT, PARTS, T>(v, xs);
        float most[PARTS];
        best = block_best<BT, PARTS>(v, 0, most, r.greedy, q.most, q.at);
    }
    if (best == 0 || r.greedy) {
        if (t == 0) put(a, row, best ? index_of(best) : -1, best ? 0.f : -INFINITY);
        return;
    }
    const double best4 = static_cast<double>(logit_of(best)) * r.c4, top = floor(best4);
    Cut cut;
    if (r.m != -INFINITY) cut.narrow(0, static_cast<uint64_t>(least_of(r, best4)) << 32);
    if (r.k > 0 || r.p < 1.0) {
        const Adder to{r.c4, top, Units()};
#pragma unroll 2
        for (int k = 0; k < PARTS; ++k) {
            const f32x4_t v = *reinterpret_cast<const f32x4_t *>(xs + token_at<BT>(0, 4 * k));
#pragma unroll
            for (int e = 0; e < 4; ++e) to.add(q.w[t & (COPIES - 1)], v[e]);
        }
        __syncthreads();
        int n[4];
        uint64_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = 0;
#pragma unroll
            for (int j = 0; j < COPIES; ++j) w[i] += q.w[j][4 * l + i];
            n[i] = static_cast<int>(w[i] >> 48);
            w[i] &= ONE - 1;
        }
        const Bins bins(n, w);
        const Marks marks(bins, r);
        const Ranges ranges(marks, r, top);
#pragma unroll 2
        for (int k = 0; k < PARTS; ++k) {
            const int i = token_at<BT>(0, 4 * k);
            const f32x4_t v = *reinterpret_cast<const f32x4_t *>(xs + i);
            if (float_key(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]))) < ranges.least()) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (ranges.has(float_key(v[e]))) {
                    const int at = atomicAdd(&q.listed, 1);
                    if (at < HELD) list[at] = key_of(v[e], i + e);
                }
        }
        __syncthreads();
        const int listed = q.listed;
        cut_tokens(cut, Tokens<T, 2, MOST, true>{list, xs, listed, listed <= HELD, x, r, top}, q, r, bins, top, marks, ranges, nullptr);
    }
    draw<BT, PARTS, true>(a, row, xs, 0, q, r, top, cut, number, 0.0);
}

// ---- a row in chunks -------------------------------------------------------------------------

// What the launches tell each other about a row.
struct Record {
    uint64_t best;                     // its largest key
    uint32_t lo[3], len[3];            // float keys of the marked bins (top_k's, top_p's, min_p's): lo .. lo + len - 1
    int32_t listed, fine;              // keys copied; bit 0, 1: the sums of parts of top_k's bin, of top_p's, are wanted
};

// A chunk's bins below its own largest token's, and that token's key.
template <class T, int BT, int PER>
__global__ void __launch_bounds__(BT) k_bins(Args a) {
    constexpr int EIGHT = 8;           // copies of the bins
    __shared__ unsigned long long w[EIGHT][BINS + 1];
    const int chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks, t = threadIdx.x, i0 = chunk * BT * PER;
    const Row<T> x(a, row);
    float v[PER];
    load_all<BT>(x, i0, v);
    const Rule r = rule_of(a, row);
    for (int i = t; i < EIGHT * (BINS + 1); i += BT) w[0][i] = 0;
    see_all<BT>(x, i0, v, r);
    __shared__ float red[BT / WAVE];
    __shared__ int red_at[BT / WAVE];
    float most[PER / 4];
    const uint64_t best = block_best<BT, PER / 4>(v, i0, most, r.greedy, red, red_at);
    const size_t at = static_cast<size_t>(row) * a.chunks + chunk;
    if (t == 0) gst(a.best + at, best);
    if ((t & 63) == 0) {
#pragma unroll
        for (int k = 0; k < PER / 4; ++k) gst(a.most + (at * (PER / 4) + k) * (BT / WAVE) + (t >> 6), most[k]);
    }
    if (r.greedy) return;
    if (best) {
        const Adder to{r.c4, floor(static_cast<double>(logit_of(best)) * r.c4), Units()};
#pragma unroll
        for (int i = 0; i < PER; ++i) to.add(w[t & (EIGHT - 1)], v[i]);
    }
    __syncthreads();
    for (int i = t; i < BINS; i += BT) {
        unsigned long long sum = 0;
#pragma unroll
        for (int c = 0; c < EIGHT; ++c) sum += w[c][i];
        gst(a.bins + at * BINS + i, static_cast<uint64_t>(sum));
        // and the weights up to each bin, in units of the first one's edge
        const double upto = wave_scan(static_cast<double>(sum & (ONE - 1)) * (bin_edge(i) / UNIT));
        w[0][i] = as_bits(upto);
    }
    __syncthreads();
    for (int i = t; i < BINS; i += BT) {
        double before = 0.0;
#pragma unroll
        for (int j = 0; j < BINS / WAVE - 1; ++j) before += j < i / WAVE ? as_double(w[0][j * WAVE + WAVE - 1]) : 0.0;
        gst(a.upto + at * BINS + i, before + as_double(w[0][i]));
    }
}

// A row's bins from its chunks', in the wave's registers.
__device__ __forceinline__ Bins bins_of(const Args &a, int row) {
    const int l = threadIdx.x & 63;
    const uint64_t *s = a.sums + static_cast<size_t>(row) * 6 * BINS;
    int n[4];
    uint64_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = gld(s + 4 * l + i);
        n[i] = static_cast<int>(gld(s + BINS + 4 * l + i));
    }
    return Bins(n, w);
}

constexpr int MT = 1024;
// The rows' bins and records.
__global__ void __launch_bounds__(MT) k_rows(Args a) {
    __shared__ Lds<MT> q;
    __shared__ int first[MAXC];
    const int row = blockIdx.x, t = threadIdx.x;
    const size_t at = static_cast<size_t>(row) * a.chunks;
    // all chunks' bins on their way at once (of a greedy row: nothing of use); a chunk without a token has none
    uint64_t got[MAXC * BINS / MT];
#pragma unroll
    for (int i = 0; i < MAXC * BINS / MT; ++i) got[i] = i * (MT / BINS) + t / BINS < a.chunks ? gld(a.bins + at * BINS + i * MT + t) : uint64_t(0);
    const Rule r = rule_of(a, row);
    if (t < BINS) {
        q.w[0][t] = 0;
        q.n[t] = 0;
    }
    const uint64_t mine = t < a.chunks ? gld(a.best + at + t) : uint64_t(0), best = block_max(mine, q, 0);
    Record *rec = a.record + row;
    if (t == 0) {
        gst(&rec->best, best);
        gst(&rec->listed, 0);
    }
    if (t < 3) gst(&rec->len[t], 0u);
    if (t == 0) gst(&rec->fine, 0);
    if (best == 0 || r.greedy) return;
    const double best4 = static_cast<double>(logit_of(best)) * r.c4, top = floor(best4);
    // a chunk's first bin among the row's
    if (t < MAXC) first[t] = mine ? bin_of(logit_of(mine), r.c4, top) : BINS;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MAXC * BINS / MT; ++i) {
        if (i * (MT / BINS) >= a.chunks) break;
        const int j = first[i * (MT / BINS) + t / BINS] + t % BINS;
        if (got[i] && j < BINS) {
            atomicAdd(&q.n[j], static_cast<unsigned>(got[i] >> 48));
            atomicAdd(&q.w[0][j], static_cast<unsigned long long>(got[i] & (ONE - 1)));
        }
    }
    __syncthreads();
    uint64_t *s = a.sums + static_cast<size_t>(row) * 6 * BINS;   // weights, counts; the same of parts of top_k's bin; of top_p's
    gst(s + 2 * BINS + t, uint64_t(0));
    if (t < BINS) {
        gst(s + t, static_cast<uint64_t>(q.w[0][t]));
        gst(s + BINS + t, static_cast<uint64_t>(q.n[t]));
    }
    if (t >= WAVE || !r.cuts()) return;
    int n[4];
    uint64_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = q.w[0][4 * t + i];
        n[i] = static_cast<int>(q.n[4 * t + i]);
    }
    const Bins bins(n, w);
    const Marks m(bins, r);
    if (t < 3) {
        int first = t == 0 ? m.k.bin : m.p0, last = t == 0 ? m.k.bin : m.p1;
        if (t == 2) first = last = r.m == -INFINITY ? BINS : bin_of(key_float(least_of(r, best4)), r.c4, top);
        if (first < BINS && first <= last) {
            const uint32_t lo = bin_start(last, r, top);
            gst(&rec->lo[t], lo);
            gst(&rec->len[t], bin_start(first - 1, r, top) - lo);
        }
        if (t == 0) gst(&rec->fine, (m.fine_k() ? 1 : 0) | (m.fine_p() ? 2 : 0));
    }
}

// The tokens of the bins in question, in any order.
template <class T, int BT, int PER>
__global__ void __launch_bounds__(BT) k_list(Args a) {
    constexpr int NW = BT / WAVE;
    __shared__ int part[NW], s_at;
    __shared__ unsigned long long w[2][BINS];                     // count above bit 48
    const int chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks, t = threadIdx.x, l = t & 63, wv = t >> 6, i0 = chunk * BT * PER;
    Record *rec = a.record + row;
    uint32_t lo[3], len[3], least = ~0u;
    const float *most = a.most + static_cast<size_t>(blockIdx.x) * (PER / 4) * NW + wv;
    float top_of[PER / 4];
#pragma unroll
    for (int k = 0; k < PER / 4; ++k) top_of[k] = gld(most + k * NW);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        len[i] = gld(&rec->len[i]);
        lo[i] = gld(&rec->lo[i]);
        if (len[i]) least = min(least, lo[i]);
    }
    if (least == ~0u) return;
    const Row<T> x(a, row);
    float v[PER];
    // parts of a wave whose largest logit is below all marked bins are not read again
#pragma unroll
    for (int k = 0; k < PER / 4; ++k)
        if (float_key(top_of[k]) >= least) x.load(token_at<BT>(i0, 4 * k), v + 4 * k);
    const int fine = gld(&rec->fine);
    const uint64_t best = gld(&rec->best);
    const Rule r = rule_of(a, row);
    for (int i = t; i < 2 * BINS; i += BT) w[0][i] = 0;
    uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < PER / 4; ++k) {
        if (float_key(top_of[k]) < least) continue;
        float *f = v + 4 * k;
        x.see(token_at<BT>(i0, 4 * k), f, r);
        if (!__ballot(float_key(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]))) >= least)) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t y = float_key(f[e]);
            mine |= static_cast<uint32_t>(y - lo[0] < len[0] || y - lo[1] < len[1] || y - lo[2] < len[2]) << (4 * k + e);
        }
    }
    const int n = __popc(mine), upto = wave_incl_scan(n);
    if (l == 63) part[wv] = upto;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        before += i < wv ? part[i] : 0;
        all += part[i];
    }
    if (all == 0) return;
    if (t == 0) s_at = atomicAdd(&rec->listed, all);
    __syncthreads();
    int at = s_at + before + upto - n;
    const double top = floor(static_cast<double>(logit_of(best)) * r.c4);
    const int s0 = fine_shift(len[0]), s1 = fine_shift(len[1]);
    // few of a thread's tokens, read again: a loop over registers would be as long a piece of code as there are tokens
#pragma unroll 1
    for (; mine; mine &= mine - 1, ++at) {
        const int i = token_at<BT>(i0, __builtin_ctz(mine));
        const float y = x.at(i, r);
        if (at < CAP) gst(a.list + static_cast<size_t>(row) * CAP + at, key_of(y, i));
        if (!fine) continue;
        const uint32_t k = float_key(y + 0.f);                    // -0 where its key is, at 0
        const unsigned long long one = ONE + units(place_of(y, r.c4, top).f);
        if ((fine & 1) && k - lo[0] < len[0]) atomicAdd(&w[0][(k - lo[0]) >> s0], one);
        if ((fine & 2) && k - lo[1] < len[1]) atomicAdd(&w[1][(k - lo[1]) >> s1], one);
    }
    if (!fine) return;
    __syncthreads();
    for (int i = t; i < 2 * BINS; i += BT) {
        const unsigned long long y = w[0][i];
        if (!y) continue;
        unsigned long long *to = reinterpret_cast<unsigned long long *>(a.sums + (static_cast<size_t>(row) * 3 + 1 + i / BINS) * 2 * BINS + i % BINS);
        atomicAdd(to, y & (ONE - 1));
        atomicAdd(to + BINS, y >> 48);
    }
}

// What is kept, the chunk into which the number falls, and the token. CHUNK: tokens of a chunk.
template <class T, int CHUNK, int FT>
__global__ void __launch_bounds__(FT) k_pick(Args a) {
    constexpr int PARTS = CHUNK / (4 * FT);
    __shared__ Lds<FT> q;
    __shared__ __align__(16) unsigned long long list[CAP];        // and then the chunk's logits
    __shared__ unsigned long long part[MAXC];                     // of the last kept bin, in units
    static_assert(CAP * 8 >= CHUNK * 4, "");
    float *xs = reinterpret_cast<float *>(list);
    const int row = blockIdx.x, t = threadIdx.x, l = t & 63;
    const uint64_t best = gld(&a.record[row].best);
    const int n = gld(&a.record[row].listed);
    const double u = number_of(a, row);
    const Rule r = rule_of(a, row);
    if (best == 0 || r.greedy) {
        if (t == 0) put(a, row, best ? index_of(best) : -1, best ? 0.f : -INFINITY);
        return;
    }
    const Row<T> x(a, row);
    const double best4 = static_cast<double>(logit_of(best)) * r.c4, top = floor(best4);
    const size_t at = static_cast<size_t>(row) * a.chunks;
    const uint64_t own = l < a.chunks ? gld(a.best + at + l) : 0;   // a lane a chunk
    const bool held = n <= CAP;
    if (held)
        for (int i = t; i < n; i += FT) list[i] = gld(a.list + static_cast<size_t>(row) * CAP + i);
    if (t < MAXC) part[t] = 0;
    Cut cut;
    if (r.m != -INFINITY) {
        const uint32_t k = least_of(r, best4);
        cut.narrow(bin_of(key_float(k), r.c4, top), static_cast<uint64_t>(k) << 32);
    }
    __syncthreads();
    const Tokens<T, 8, 2 * CAP, false> tokens{list, xs, n, held, x, r, top};
    if (r.k > 0 || r.p < 1.0) {
        const Bins bins = bins_of(a, row);
        const Marks marks(bins, r);
        cut_tokens(cut, tokens, q, r, bins, top, marks, Ranges(marks, r, top), a.sums + (static_cast<size_t>(row) * 3 + 1) * 2 * BINS);
    }
    // the chunks' weights in the bins before the last kept one
    const double first = top - floor(static_cast<double>(logit_of(own)) * r.c4);   // a chunk's first bin among the row's
    const double upto_bin = static_cast<double>(cut.bin) - 1.0 - first;
    double mine = own && upto_bin >= 0.0 ? gld(a.upto + (at + l) * BINS + min(static_cast<int>(upto_bin), BINS - 1)) : 0.0;
    if (mine > 0.0) mine *= bin_edge(static_cast<int>(first));
    if (cut.bin < BINS) {
        // and of that one's tokens those that are kept, chunk by chunk of a wave's: a chunk's lie side by side in the list
        const Keys in = between(bin_start(cut.bin, r, top), bin_start(cut.bin - 1, r, top));
        // a thread adds up its tokens of a chunk first: of the list's, which lie side by side, consecutive ones
        uint64_t run = 0;
        int chunk = 0;
        auto take = [&](uint64_t k) {
            if (!in.have(k) || k < cut.key) return;
            const int c = index_of(k) / CHUNK;
            if (c != chunk) {
                if (run) atomicAdd(&part[chunk], static_cast<unsigned long long>(run));
                chunk = c;
                run = 0;
            }
            run += tokens.units_of(k);
        };
        if (held) {
            const int share = (n + FT - 1) / FT, end = min(n, (t + 1) * share);
            for (int i = t * share; i < end; ++i) take(list[i]);
        } else {
            for (int i0 = 0; i0 < a.vocab; i0 += 2 * CAP) {
                tokens.template bring<FT>(i0);
                for (int j = 0; j < 2 * CAP / FT; ++j) take(tokens.template brought<FT>(i0, j));
            }
        }
        if (run) atomicAdd(&part[chunk], static_cast<unsigned long long>(run));
        __syncthreads();
        if (l < a.chunks) mine += static_cast<double>(part[l]) * (bin_edge(cut.bin) / UNIT);
    }
    const double upto = wave_scan(mine), total = lane_double(upto, 63), number = u * total;
    const uint64_t past = __ballot(mine > 0.0 && upto > number), some = __ballot(mine > 0.0);   // as in draw
    // none has a weight only if the logits have been written to since the bins were made: a chunk of the row even then
    const int chunk = past ? __builtin_ctzll(past) : some ? 63 - __builtin_clzll(some) : index_of(best) / CHUNK;
    const double before = chunk ? lane_double(upto, chunk - 1) : 0.0;
    __syncthreads();                                              // the list has been read
    {
        float v[4 * PARTS];
        load_all<FT>(x, chunk * CHUNK, v);
        see_all<FT>(x, chunk * CHUNK, v, r);
        keep<FT, PARTS, T>(v, xs);
    }
    draw<FT, PARTS, false>(a, row, xs, chunk * CHUNK, q, r, top, cut, number - before, total);
}

// ---- launches --------------------------------------------------------------------------------

// Tokens of a chunk: 4096, 16 of 256 threads, so that few long rows still reach many CUs; 16384 where there are blocks for all of them
// anyway, or more than 64 chunks otherwise.
constexpr int SHORT_MOST = 1024;       // most chunks of 4096 tokens in a call
int chunk_of(int rows, int vocab) {
    const int64_t blocks = static_cast<int64_t>(rows) * ((vocab + 4095) / 4096);
    return blocks <= SHORT_MOST && vocab <= MAXC * 4096 ? 4096 : 16384;
}
size_t bytes_of(int rows, int chunks, int chunk) {
    return static_cast<size_t>(rows) * (static_cast<size_t>(chunks) * ((2 * BINS + 1) * 8 + chunk / 64) + (6 * BINS + CAP) * 8 + sizeof(Record));
}
// What a call takes of its workspace.
size_t need_of(int rows, int vocab) {
    if (vocab <= ROW_MOST || rows < 1) return 0;
    const int chunk = chunk_of(rows, vocab);
    return bytes_of(rows, (vocab + chunk - 1) / chunk, chunk);
}
// What suffices for every call of up to so many rows and tokens: fewer or shorter rows may be in smaller chunks, and take more.
size_t workspace(int rows, int vocab) {
    size_t most = need_of(rows, vocab);
    if (most > 0)
        for (int chunks = ROW_MOST / 4096 + 1; chunks <= std::min(MAXC, (vocab + 4095) / 4096); ++chunks)
            most = std::max(most, bytes_of(std::min(rows, SHORT_MOST / chunks), chunks, 4096));
    return most;
}

template <class T>
void launch(Args a, void *ws, hipStream_t s) {
    const dim3 rows(static_cast<unsigned>(a.rows));
    if (a.vocab <= 1024) hipLaunchKernelGGL((k_row<T, 256, 1>), rows, dim3(256), 0, s, a);
    else if (a.vocab <= 2048) hipLaunchKernelGGL((k_row<T, 256, 2>), rows, dim3(256), 0, s, a);
    else if (a.vocab <= 4096) hipLaunchKernelGGL((k_row<T, 256, 4>), rows, dim3(256), 0, s, a);
    else if (a.vocab <= 8192) hipLaunchKernelGGL((k_row<T, 512, 4>), rows, dim3(512), 0, s, a);
    else if (a.vocab <= ROW_MOST) hipLaunchKernelGGL((k_row<T, 512, 8>), rows, dim3(512), 0, s, a);
    else {
        const int chunk = chunk_of(a.rows, a.vocab);
        a.chunks = (a.vocab + chunk - 1) / chunk;
        a.bins = static_cast<uint64_t *>(ws);
        a.best = a.bins + static_cast<size_t>(a.rows) * a.chunks * BINS;
        a.sums = a.best + static_cast<size_t>(a.rows) * a.chunks;
        a.upto = reinterpret_cast<double *>(a.sums + static_cast<size_t>(a.rows) * 6 * BINS);
        a.list = reinterpret_cast<uint64_t *>(a.upto + static_cast<size_t>(a.rows) * a.chunks * BINS);
        a.record = reinterpret_cast<Record *>(a.list + static_cast<size_t>(a.rows) * CAP);
        a.most = reinterpret_cast<float *>(a.record + a.rows);
        const dim3 grid(static_cast<unsigned>(a.rows) * a.chunks);
        if (chunk == 4096) {
            hipLaunchKernelGGL((k_bins<T, 256, 16>), grid, dim3(256), 0, s, a);
            hipLaunchKernelGGL(k_rows, rows, dim3(MT), 0, s, a);
            hipLaunchKernelGGL((k_list<T, 256, 16>), grid, dim3(256), 0, s, a);
            hipLaunchKernelGGL((k_pick<T, 4096, 512>), rows, dim3(512), 0, s, a);
        } else {
            hipLaunchKernelGGL((k_bins<T, 512, 32>), grid, dim3(512), 0, s, a);
            hipLaunchKernelGGL(k_rows, rows, dim3(MT), 0, s, a);
            hipLaunchKernelGGL((k_list<T, 512, 32>), grid, dim3(512), 0, s, a);
            hipLaunchKernelGGL((k_pick<T, 16384, 512>), rows, dim3(512), 0, s, a);
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
    const size_t need = sample::need_of(n_rows, vocab);
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

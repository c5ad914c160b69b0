// Attention of drafted rows over a paged K/V cache on gfx950 (the C ABI's navi_tree_attention): every row of
// a request sees all of its cached positions and those of the step's rows that its mask names.
//
// For one request and kv head the rows x grouped heads form M = rows * n_head / n_kv_head query rows over the same L keys:
//   S = scale Q K^T,  p = exp(S - m),  O = p V / sum p.
// K and V (4 D bytes a key and kv head) are read once for all M rows, so with few rows the cache's
// bytes bound it, with many the matrix units.
//
//  * Scores are computed transposed, S^T = K Q^T (v_mfma_f32_16x16x32: 16 keys x 16 query rows): a lane then
//    holds 4 keys of one query row per tile, and two such tiles are, register for register, the B operand
//    of O^T += V^T P^T over 32 keys if V^T's operand takes its keys in that order too. P never leaves
//    its registers (as a hi + lo pair of the cache's type, two products), and a row's maximum, sum and mask are a lane's own values.
//  * V^T's operand is V read from LDS through the transposing load (ds_read_b64_tr_b16: in a
//    16-lane group lane 4r + c fetches columns 4c.. of key r and gets column `lane`, keys 0..3). V rows sit
//    in LDS with their 32-byte chunks XORed by the key, so that the 16 rows such a load touches
//    spread over all banks.
//  * Up to 32 query rows (k_tree) a wave works alone on its own 32-key tiles, every W-th of the block's range, with K from
//    memory in operand form, its own V buffer and no barrier until its range ends; then the waves' results are joined in
//    LDS. 32 requests with one row each over 1024 keys take 25.9 us, 5.20 TB/s: the cache's bytes at the rate of a large
//    read (5.6 TB/s here) are 24.
//  * Above (k_tree_rows) two or four waves with 32 rows each share the K and V tiles, which go through LDS in two buffers with
//    one barrier a tile. 64 requests x 24 rows (48 query rows) over 8192 keys 414 us (412 to 417 in three runs), 5.2 TB/s; without the products 385.
//    64 f32 rows (128 query rows) over 32768 keys 58 us: 39 us for every further 32768 keys, which with the pairs' doubled
//    products are 880 TFLOP/s, and 20 us for the start, the parts' 17 MB and the join.
//  * Softmax against a reference value that moves only when a score passes it by more than SLACK: the
//    rescaling, and the maximum over lanes that it needs, are off the common path. exp2 with the scale folded in.
//  * An e4m3 pool's codes become f16 or bf16, which hold them exactly, on their way to the matrix units: in registers up to 32 query rows (16
//    codes a lane and load, so that a lane's two operands have columns 64 i + 16 (l / 16) .. and q is read in that order), as they are staged
//    above. K's factor goes into the scores' and V's into the sum's inverse, so that the loops are those of the other pools. 32 requests with one
//    row each over 1024 keys take 16.9 us (67.5 MB, 4.0 TB/s); 64 requests x 24 rows over 8192 keys 284 to 305 us from card to card (1.08 GB,
//    3.5 to 3.8 TB/s): half the bytes of f16 under the same products, softmax and barriers (scores alone 208 us), which two waves a SIMD
//    overlap only in part; fewer cycles have come with a lower clock. Loads of 8 codes a lane took 310 us where these take 292.
//  * Requests are cut into even chunks over the blocks, however uneven their lengths (lay_out): 64 requests of lengths spread from
//    1 to 8000 71 us, uncut 145. A second kernel joins the chunks' results (unnormalised sums, reference, sum) in their order.
#include "dev_common.h"
#include "f8.h"
#include "tile_layout.h"
#include "tree.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace navi_amd {
namespace tree {

using kv::Div;
using kv::div_by;

constexpr int NW = 4, BT = NW * WAVE;  // waves of a block of k_tree_join
// Of k_tree: eight, more loads on their way, where a block has a whole request; four, and twice as many blocks, where requests are
// cut (64 ragged ones of up to 8000 keys: 71 us, with eight 84). Eight waves fill a CU, so their gain ends where the blocks are
// more than the CUs: 8 kv heads over 1000 keys, us with eight / four: 24 requests 29.1 / 29.2, 32 25.7 / 27.1, 33 42.6 / 38.4,
// 40 46.6 / 45.0, 48 51.0 / 49.4, 64 56.3 / 55.1.
constexpr int alone_of(bool cut) { return cut ? 4 : 8; }
// Of k_tree_rows, RW waves of which share their query rows' tiles: eight, one block a CU, so that half as many parts of
// a cut request are stored and joined (64 drafted f32 rows over 32768 keys: 59 us, with four 64; 16 x 80 query rows over 4000 78 and
// 80); four where two waves share and the registers allow two blocks a CU (64 requests x 24 rows over 8192 keys: 415 us in each of
// two runs, with eight 432 and 435).
constexpr int waves_of(bool pair, int rw) { return rw == 2 && !pair ? 4 : 8; }
constexpr int KT = 32;                 // keys of a wave's tile
// p = 2^(s - reference + LIFT): at most 2^(SLACK + LIFT) = 2^14, inside f16, and f16's full precision down to
// 2^-24 of the reference instead of 2^-14.
constexpr float SLACK = 4.f, LIFT = 10.f;
constexpr float NONE = -INFINITY;

struct Args {
    const void *q, *k, *v;
    const float *ks, *vs;              // an e4m3 pool's factors of K and V a kv head, or null
    void *out;
    float *po, *pm;                    // the parts of requests that are cut (part_of)
    uint32_t *first;                   // and each group's chunks before every request [groups][n + 1]
    const int32_t *table, *n_past, *cu, *slot;   // slot: null, or rows with slot < 0 see nothing
    const uint64_t *mask;
    int n, hkv, g, blocks, n_pages, n_rows, max_new, ldq, ldkv, ldo, workers, groups, step, parts;
    int tiled;                         // f32 out: in the tile layout of rows.h, heads * D wide
    int flip;                          // scale < 0: the scores' sign goes into q
    Div page, heads_per;               // heads_per: by g
    float scale;                       // |scale| * log2 e
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <class E>
struct Types;
template <>
struct Types<_Float16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ f32x4_t mfma(v8 a, v8 b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static constexpr uint32_t EXPONENT = 0x7C007C00u;
};
template <>
struct Types<__bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ f32x4_t mfma(v8 a, v8 b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static constexpr uint32_t EXPONENT = 0x7F807F80u;
};

// Whether one of the 8 two-byte values is an infinity or NaN (all exponent bits set).
template <class E>
__device__ __forceinline__ bool any_special(u32x4_t x) {
    constexpr uint32_t M = Types<E>::EXPONENT, LO = M & 0xFFFFu, HI = M & 0xFFFF0000u;
    bool b = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) b |= (x[i] & LO) == LO || (x[i] & HI) == HI;
    return b;
}

// What the scores of a kv head's keys are multiplied with, and what its sums of V are. P: the pool's elements; only e4m3 has factors.
template <class P>
__device__ __forceinline__ float score_factor(const Args &a, int kvh) { return sizeof(P) == 1 && a.ks ? a.scale * gld(a.ks + kvh) : a.scale; }
template <class P>
__device__ __forceinline__ float value_factor(const Args &a, int kvh) { return sizeof(P) == 1 && a.vs ? gld(a.vs + kvh) : 1.f; }

// Four consecutive columns of an output row.
template <class E, bool PAIR>
__device__ __forceinline__ void store_out(const Args &a, int row, int col, int width, f32x4_t o) {
    if constexpr (PAIR) {
        st4(static_cast<float *>(a.out) + (a.tiled ? rows::pk_a(row, col, width) : static_cast<size_t>(row) * a.ldo + col), o);
    } else {
        typedef typename Types<E>::v4 v4;
        *(NAVI_GLOBAL v4 *) (static_cast<E *>(a.out) + static_cast<size_t>(row) * a.ldo + col) =
            v4{static_cast<E>(o[0]), static_cast<E>(o[1]), static_cast<E>(o[2]), static_cast<E>(o[3])};
    }
}

template <class T, class U>
__device__ __forceinline__ T bits(const U &u) {
    static_assert(sizeof(T) == sizeof(U), "");
    T t;
    __builtin_memcpy(&t, &u, sizeof(T));
    return t;
}

// The greatest over the four lanes that share a query row (l, l ^ 16, l ^ 32, l ^ 48); their sum.
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float row_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Where request `req` stands: its rows of the step, cached positions and positions in all.
struct Where {
    int c0, rows, past, len;
};
__device__ __forceinline__ Where where_is(const Args &a, int req) {
    const int64_t room = min(static_cast<int64_t>(a.blocks) * a.page.d, static_cast<int64_t>(INT32_MAX - 4 * KT * NW));
    Where w;
    w.c0 = max(gld(a.cu + req), 0);
    const int count = max(min(gld(a.cu + req + 1), a.n_rows) - w.c0, 0), past = gld(a.n_past + req);
    w.rows = min(count, a.max_new);
    w.past = static_cast<int>(min<int64_t>(max(past, 0), room));
    w.len = static_cast<int>(min<int64_t>(static_cast<int64_t>(w.past) + count, room));
    // lengths that a plan refuses: no row of it has a slot
    if (a.slot && (past < 0 || count > a.max_new || static_cast<int64_t>(past) + count > room)) w.rows = w.len = 0;
    return w;
}

// Requests of uneven length over evenly long chunks: with `workers` wanted blocks a kv head and query group, a chunk is
// at most total / workers steps (of a.step 32-key tiles), and a request is cut into as few even chunks of that as it takes:
// at most workers + requests of them, in the requests' order. At most `workers` requests are longer than a chunk, so that
// the chunks of cut requests, whose parts are kept, are at most 2 workers.
constexpr int MAXB = BT;               // most requests of a call that is cut
struct Chunks {
    uint32_t before[MAXB + 1];         // before request i: all chunks, and << 16 those of cut requests
    int steps[MAXB];
    Where at[MAXB];
    int red[NW];
    float sum[NW];
};
__device__ __forceinline__ int steps_of(const Args &a, const Where &w, int qrow0) {
    const int tiles = w.rows * a.g > qrow0 ? (w.len + KT - 1) / KT : 0;
    return (tiles + a.step - 1) / a.step;
}
__device__ __forceinline__ int chunk_steps(const Args &a, float total) {
    // the steps in all, exact below 2^24; above (lengths out of all proportion) rounded up, so that the chunks stay as few, and
    // at most 2^30, more than a request has
    return max(total < 16777216.f ? (static_cast<int>(total) + a.workers - 1) / a.workers
                                  : static_cast<int>(min(total * 1.001f / static_cast<float>(a.workers), 1073741824.f)) + 1, 1);
}
__device__ __forceinline__ uint32_t chunks_of(int steps, int most) {
    const uint32_t n = static_cast<uint32_t>((steps + most - 1) / most);
    return n > 1 ? n << 16 | n : n;
}
// The first BT threads have a request each; all of a block's threads call it.
__device__ __forceinline__ void lay_out(const Args &a, int qrow0, Chunks &q) {
    const int t = threadIdx.x, wv = t >> 6;
    const bool own = t < a.n;
    Where w{0, 0, 0, 0};
    if (own) w = where_is(a, t);
    const int steps = steps_of(a, w, qrow0);
    if (a.n == 1) {                                               // nothing to add up
        if (own) {
            q.before[0] = 0;
            q.before[1] = chunks_of(steps, chunk_steps(a, static_cast<float>(steps)));
            q.steps[0] = steps;
            q.at[0] = w;
        }
        __syncthreads();
        return;
    }
    const float part = wave_sum(static_cast<float>(steps));
    if ((t & 63) == 0 && wv < NW) q.sum[wv] = part;
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) total += q.sum[i];
    const int upto = wave_incl_scan(static_cast<int>(chunks_of(steps, chunk_steps(a, total))));
    if ((t & 63) == 63 && wv < NW) q.red[wv] = upto;
    __syncthreads();
    int off = 0;
#pragma unroll
    for (int i = 0; i < NW - 1; ++i) off += i < wv ? q.red[i] : 0;
    if (t == 0) q.before[0] = 0;
    if (own) {
        q.before[t + 1] = static_cast<uint32_t>(off + upto);
        q.steps[t] = steps;
        q.at[t] = w;
    }
    __syncthreads();
}
// Where a cut chunk's part is kept: the group's rows of [D], and (reference, sum) pairs.
__device__ __forceinline__ size_t part_of(const Args &a, int kvh, int group, int k) {
    return (static_cast<size_t>(kvh) * a.groups + group) * a.parts + k;
}

// A block's share of the work: a request, its tiles t0 .. t_end - 1, and whether these are all it has.
struct Share {
    Where at;
    int kvh, group, req, t0, t_end, part;
    bool whole, none;
};
template <bool CUT>
__device__ __forceinline__ Share share_of(const Args &a, int group_rows) {
    Share s;
    int id = blockIdx.x;
    s.kvh = id % a.hkv;
    id /= a.hkv;
    s.group = id % a.groups;
    const int unit = id / a.groups;
    s.req = unit;
    s.t0 = s.part = 0;
    s.whole = true;
    if constexpr (CUT) {
        __shared__ Chunks c;
        lay_out(a, s.group * group_rows, c);
        if (unit == 0 && s.kvh == 0)                            // for the join
            for (int i = threadIdx.x; i <= a.n; i += blockDim.x) gst(a.first + s.group * (a.n + 1) + i, c.before[i]);
        auto before = [&](int i) { return static_cast<int>(c.before[i] & 0xFFFFu); };
        s.none = unit >= before(a.n);
        if (s.none) return s;
        int lo = 0, hi = a.n;                                     // before[lo] <= unit < before[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (before(mid) <= unit) lo = mid;
            else hi = mid;
        }
        s.req = lo;
        s.at = c.at[lo];
        const int n = before(lo + 1) - before(lo), k = unit - before(lo), steps = c.steps[lo];
        s.whole = n == 1;
        s.part = static_cast<int>(c.before[lo] >> 16) + k;
        s.t0 = static_cast<int>(static_cast<int64_t>(steps) * k / n) * a.step;
        s.t_end = min((s.at.len + KT - 1) / KT, static_cast<int>(static_cast<int64_t>(steps) * (k + 1) / n) * a.step);
    } else {
        s.at = where_is(a, s.req);
        s.none = s.group * group_rows >= s.at.rows * a.g;         // this request has fewer rows
        s.t_end = (s.at.len + KT - 1) / KT;
    }
    return s;
}

// The pages of a request: page_of a position and, from its page, the row of the pool (slot_of): -1 where there is none.
struct Pages {
    const int32_t *table;
    int limit;                         // positions from here on are not the block's
    const Args &a;
    __device__ __forceinline__ int page_of(int key) const { return key < limit ? gld(table + div_by(a.page, key)) : -1; }
    __device__ __forceinline__ int slot_of(int key, int page) const {
        return static_cast<unsigned>(page) < static_cast<unsigned>(a.n_pages)
                   ? page * static_cast<int>(a.page.d) + key - div_by(a.page, key) * static_cast<int>(a.page.d) : -1;
    }
};

// V rows of a tile in LDS: 32-byte piece i of key r at piece i ^ (r & (D / 16 - 1)), so that the rows that a
// transposing load touches spread over the banks. The address of 16-byte half `h` of piece i.
template <int D>
__device__ __forceinline__ unsigned char *v_at(unsigned char *buf, int r, int i, int h) {
    return buf + r * (D * 2) + ((i ^ (r & (D / 16 - 1))) << 5) + (h << 4);
}

// A wave's query rows, 16 a tile; lane l has row l % 16 of each: mask, factor of the scores, and the running
// reference (ref: + SLACK; sub: - LIFT), sum and O^T (columns 16 d + 4 (l / 16) ..).
template <class E, bool PAIR, int D, int NT>
struct Rows {
    typedef typename Types<E>::v8 v8;
    typedef typename Types<E>::v4 v4;
    static constexpr int KS = D / 32, DT = D / 16, QP = PAIR ? 2 : 1;   // MFMA steps of a score, column tiles of O
    f32x4_t acc[NT][DT];
    float ref[NT], sub[NT], sum[NT], fac[NT];
    uint64_t seen[NT];
    uint32_t off[NT];                  // bit r: row r of the tile has no slot (the same in all lanes)

    // Query row m of the request's as it stands in memory (past its rows: zeros), loaded; then its operands, a pair's hi
    // before its lo, and the factor of its scores.
    struct Raw {
        u32x4_t x[QP * KS];
    };
    // Step k of the operands has columns 32 k + 8 (l / 16) .. of the head; WIDE: 64 (k / 2) + 16 (l / 16) + 8 (k % 2) .., as K in 8 bits comes
    // into registers.
    template <bool WIDE>
    static __device__ __forceinline__ void fetch(const Args &a, const Share &s, int m, Raw &r) {
        const int lg = (threadIdx.x & 63) >> 4, j = div_by(a.heads_per, m);
        const bool on = j < s.at.rows;
        const size_t at = static_cast<size_t>(s.at.c0 + (on ? j : 0)) * a.ldq + static_cast<size_t>(s.kvh * a.g + (on ? m - j * a.g : 0)) * D +
                          (WIDE ? 16 : 8) * lg;
        const unsigned char *p = static_cast<const unsigned char *>(a.q) + at * 2 * QP;
#pragma unroll
        for (int i = 0; i < QP * KS; ++i) {
            const int k = i / QP, col = WIDE ? 64 * (k / 2) + 8 * (k % 2) : 32 * k;
            r.x[i] = on ? *(const NAVI_GLOBAL u32x4_t *) (p + 2 * QP * col + 16 * (i % QP)) : u32x4_t{0u, 0u, 0u, 0u};
        }
    }
    static __device__ __forceinline__ float operands(const Args &a, float scale, const Raw &r, v8 (&q)[QP * KS]) {
        float f = scale;
        if constexpr (PAIR) {
            // q times a power of two that puts the row's largest value into [1, 2): pairs keep 22 bits of it
            // whatever its range; the scores get the inverse
            f32x4_t x[KS][2];
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    x[k][h] = bits<f32x4_t>(r.x[2 * k + h]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[k][h][e]));
                }
            top = row_max(top);
            const int ex = top > 0.f && top < INFINITY ? ilogbf(top) : 0;
            f = ldexpf(scale, ex);
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float y = ldexpf(a.flip ? -x[k][e >> 2][e & 3] : x[k][e >> 2][e & 3], -ex);
                    q[k][e] = static_cast<E>(y);
                    q[KS + k][e] = static_cast<E>(y - static_cast<float>(q[k][e]));
                }
        } else {
            const uint32_t sign = a.flip ? 0x80008000u : 0u;
#pragma unroll
            for (int k = 0; k < KS; ++k) q[k] = bits<v8>(r.x[k] ^ sign);
        }
        // a factor of 0 (all scores alike) as the least normal number: -inf, a place not seen, must stay -inf
        return fmaxf(f, 1.17549435e-38f);
    }

    __device__ __forceinline__ void start(const Args &a, const Share &s, int qrow0) {
        const int lr = threadIdx.x & 15;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int j = div_by(a.heads_per, qrow0 + nt * 16 + lr);
            seen[nt] = j < s.at.rows ? gld(a.mask + s.at.c0 + j) : 0;
            off[nt] = a.slot ? static_cast<uint32_t>(__ballot(j < s.at.rows && gld(a.slot + s.at.c0 + j) < 0)) & 0xFFFFu : 0u;
            ref[nt] = NONE;
            sub[nt] = sum[nt] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[nt][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
    }

    // -inf for the scores of keys that a row does not see. Bit k of `there`: key k of the tile exists; the tile begins
    // `ahead` positions after the first drafted one.
    __device__ __forceinline__ void hide(f32x4_t (&sc)[NT][2], uint32_t there, int ahead) {
        const int lg = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            uint32_t vis = ahead >= 64 ? 0u : ahead >= 0 ? static_cast<uint32_t>(seen[nt] >> ahead)
                         : ahead <= -KT ? ~0u : static_cast<uint32_t>(seen[nt] << -ahead) | ((1u << -ahead) - 1u);
            vis = (vis & there) >> (4 * lg);
#pragma unroll
            for (int i = 0; i < 8; ++i) sc[nt][i >> 2][i & 3] = vis >> ((i >> 2) * 16 + (i & 3)) & 1u ? sc[nt][i >> 2][i & 3] : NONE;
        }
    }

    // Scores to p, in place, and O^T += V^T P^T. One test for all query tiles whether a score passes its reference
    // by more than SLACK, so that the rest is one straight run of instructions. p goes into the products as a pair of E whatever
    // q's type (2^-21 of p is left out for f16, 2^-16 for bf16): one E would be off by as much as the output's own rounding. The
    // second product costs 32 requests of 1024 keys 1 %, 64 requests x 24 rows over 8192 keys 1 %, and where the matrix units
    // set the pace (64 f16 rows of two heads over 32768 keys) 45.5 -> 51.7 us.
    __device__ __forceinline__ void add(f32x4_t (&sc)[NT][2], unsigned char *buf) {
        const int l = threadIdx.x & 63, lr = l & 15, lg = l >> 4;
        float top[NT];
        bool passed = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            top[nt] = NONE;
#pragma unroll
            for (int i = 0; i < 8; ++i) top[nt] = fmaxf(top[nt], sc[nt][i >> 2][i & 3]);
            passed |= top[nt] * fac[nt] > ref[nt];
        }
        if (__ballot(passed)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float mx = row_max(top[nt]) * fac[nt];
                const bool up = mx > ref[nt];
                const float f = !up ? 1.f : ref[nt] == NONE ? 0.f : __builtin_amdgcn_exp2f(ref[nt] - SLACK - mx);
                sum[nt] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[nt][d] *= f;
                ref[nt] = up ? mx + SLACK : ref[nt];
                sub[nt] = up ? mx - LIFT : sub[nt];
            }
        }
        v8 va[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const v4 x = bits<v4>(__builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4 *) (v_at<D>(buf, kt * 16 + 4 * lg + (lr >> 2), d, 0) + ((lr & 3) << 3))));
#pragma unroll
                for (int e = 0; e < 4; ++e) va[d][4 * kt + e] = x[e];
            }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            v8 ph, pl;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[nt][i >> 2][i & 3], fac[nt], -sub[nt]));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[nt][i >> 2][(i & 3) + 1], fac[nt], -sub[nt]));
                sc[nt][i >> 2][i & 3] = p0;
                sc[nt][i >> 2][(i & 3) + 1] = p1;
                sum[nt] += p0 + p1;
                if constexpr (std::is_same_v<E, _Float16>) {
                    // hi truncated, two at once; lo is the exact rest, rounded
                    const auto hi = bits<half2_t>(__builtin_amdgcn_cvt_pkrtz(p0, p1));
                    ph[i] = hi[0];
                    ph[i + 1] = hi[1];
                } else {
                    ph[i] = static_cast<E>(p0);
                    ph[i + 1] = static_cast<E>(p1);
                }
                pl[i] = static_cast<E>(p0 - static_cast<float>(ph[i]));
                pl[i + 1] = static_cast<E>(p1 - static_cast<float>(ph[i + 1]));
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                acc[nt][d] = Types<E>::mfma(va[d], ph, acc[nt][d]);
                acc[nt][d] = Types<E>::mfma(va[d], pl, acc[nt][d]);
            }
        }
    }

    // Drafted keys with an infinity or NaN in V (rare; bits `special` of the tile): zeros in the products of add, since 0
    // times one would reach the rows that do not see them. Here the rows that do see them add theirs; sc: p.
    template <class P>
    __device__ __forceinline__ void add_special(const f32x4_t (&sc)[NT][2], uint32_t special, int tile, const Share &s, const Pages &pg) {
        const int l = threadIdx.x & 63, lr = l & 15, lg = l >> 4;
        for (; special; special &= special - 1) {
            const int kin = __builtin_ctz(special), key = tile * KT + kin, ahead = key - s.at.past;
            const int slot = pg.slot_of(key, pg.page_of(key));
            const P *vp = static_cast<const P *>(pg.a.v) + static_cast<size_t>(max(slot, 0)) * pg.a.ldkv + s.kvh * D + 4 * lg;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float p = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) p = (kin >> 4) * 4 + (kin & 3) == i ? sc[nt][i >> 2][i & 3] : p;
                p = __shfl(p, lr + 16 * ((kin & 15) >> 2));
                const bool vis = ahead >= 0 && ahead < 64 && (seen[nt] >> (ahead & 63) & 1);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    v4 x;
                    if constexpr (sizeof(P) == 1) {
                        uint32_t w[2];
                        f8_unpack4<E>(gld(reinterpret_cast<const uint32_t *>(vp + 16 * d)), w);
                        x = bits<v4>(w);
                    } else {
                        x = bits<v4>(*(const NAVI_GLOBAL u32x2_t *) (vp + 16 * d));
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[nt][d][e] = vis ? fmaf(p, static_cast<float>(x[e]), acc[nt][d][e]) : acc[nt][d][e];
                }
            }
        }
    }

    // Rows without a slot, whatever the cache held for them (infinities and NaN included): as rows that see nothing.
    __device__ __forceinline__ void drop() {
        const int lr = threadIdx.x & 15;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            if (off[nt]) {
                const bool no = off[nt] >> lr & 1u;
                ref[nt] = no ? NONE : ref[nt];
                sum[nt] = no ? 0.f : sum[nt];
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[nt][d][e] = no ? 0.f : acc[nt][d][e];
            }
    }

    // Row r of the group, columns col ..: stored, or kept as the chunk's part.
    template <class P>
    static __device__ __forceinline__ void finish(const Args &a, const Share &s, int group_rows, int r, int col, f32x4_t o, float m, float total) {
        const int q = s.group * group_rows + r, j = div_by(a.heads_per, q);
        if (j >= s.at.rows) return;
        if (!s.whole) {
            const size_t at = part_of(a, s.kvh, s.group, s.part) * group_rows + r;
            st4(a.po + at * D + col, o);
            if (col == 0) {
                gst(a.pm + 2 * at, m);
                gst(a.pm + 2 * at + 1, total);
            }
        } else {
            store_out<E, PAIR>(a, s.at.c0 + j, (s.kvh * a.g + q - j * a.g) * D + col, a.hkv * a.g * D, o * (m == NONE ? 0.f : value_factor<P>(a, s.kvh) / total));
        }
    }
};

// Step k's 16 bytes of E from a lane's loads of a pool's row: as they are, or half a load's codes.
template <class E, bool F8, int LD>
__device__ __forceinline__ u32x4_t operand_of(const u32x4_t (&r)[LD], int k) {
    if constexpr (F8) {
        uint32_t lo[2], hi[2];
        f8_unpack4<E>(r[k / 2][2 * (k % 2)], lo);
        f8_unpack4<E>(r[k / 2][2 * (k % 2) + 1], hi);
        return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
    } else {
        return r[k];
    }
}

// Up to 32 query rows: every wave has all of them and works alone on its own tiles, every W-th of the block's, with K from
// memory in operand form and its own V buffer, no barrier until the end; then the W results are joined in LDS.
// CUT: a block takes a chunk of a request's keys, else all of them.
// P: the pool's elements, E or e4m3; these come in 16-byte loads of twice as many columns and become E in registers.
template <class E, bool PAIR, class P, int D, int NT, bool CUT>
__global__ void __launch_bounds__(alone_of(CUT) * WAVE, NT == 1 && CUT ? 3 : 2) k_tree(Args a) {
    constexpr int W = alone_of(CUT);
    constexpr bool F8 = sizeof(P) == 1;
    typedef Rows<E, PAIR, D, NT> R;
    typedef typename R::v8 v8;
    constexpr int KS = R::KS, DT = R::DT, QP = R::QP, VB = KT * D * 2, DP = D + 4;
    constexpr int JOIN = W * NT * 16 * DP * 4, QB = QP * NT * KS * WAVE * 16;
    __shared__ __align__(16) unsigned char sm[W * VB + QB > JOIN ? W * VB + QB : JOIN];
    __shared__ float s_fac[NT * 16], s_ref[W][NT * 16], s_sum[W][NT * 16];
    const int wv = threadIdx.x >> 6, l = threadIdx.x & 63, lr = l & 15, lg = l >> 4;
    // uncut, the first tile's pages do not wait for the request's lengths: a round of memory latency less
    int ahead[2];
    if constexpr (!CUT) {
        const int req = static_cast<int>(blockIdx.x) / a.hkv / a.groups;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const int b = div_by(a.page, wv * KT + kt * 16 + lr);
            ahead[kt] = b < a.blocks ? gld(a.table + static_cast<size_t>(req) * a.blocks + b) : -1;
        }
    }
    const Share s = share_of<CUT>(a, NT * 16);
    if (s.none) return;
    const int qrow0 = s.group * NT * 16;
    const Pages pg{a.table + static_cast<size_t>(s.req) * a.blocks, s.at.len, a};

    constexpr int LD = F8 ? KS / 2 : KS, LC = D / LD;             // loads a key and lane, columns of one over the four lanes
    u32x4_t kr[2][LD], vr[2][LD];
    int slot[2], page[2];
    const P *kb = static_cast<const P *>(a.k) + s.kvh * D + LC / 4 * lg, *vb = static_cast<const P *>(a.v) + s.kvh * D + LC / 4 * lg;
    auto look_up = [&](int t) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) page[kt] = pg.page_of(t * KT + kt * 16 + lr);
    };
    auto load = [&](int t) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            slot[kt] = pg.slot_of(t * KT + kt * 16 + lr, page[kt]);
            const size_t at = static_cast<size_t>(max(slot[kt], 0)) * a.ldkv;
#pragma unroll
            for (int k = 0; k < LD; ++k) kr[kt][k] = *(const NAVI_GLOBAL u32x4_t *) (kb + at + LC * k);
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int k = 0; k < LD; ++k) vr[kt][k] = *(const NAVI_GLOBAL u32x4_t *) (vb + static_cast<size_t>(max(slot[kt], 0)) * a.ldkv + LC * k);
    };
    int t = s.t0 + wv;
    if constexpr (CUT) {
        if (t < s.t_end) look_up(t);
    } else {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) page[kt] = t * KT + kt * 16 + lr < s.at.len ? ahead[kt] : -1;
    }
    // q before K and V, which a wait for it would otherwise include (one row over 256 keys: 8.7 us, after them 10.2)
    typename R::Raw raw;
    if (wv < NT) R::template fetch<F8>(a, s, qrow0 + wv * 16 + lr, raw);
    R rows;
    rows.start(a, s, qrow0);
    if (t < s.t_end) {
        load(t);
        if (t + W < s.t_end) look_up(t + W);                    // pages are looked up two tiles ahead
    }
    // the operands of q into LDS, a wave a query tile
    u32x4_t *s_q = reinterpret_cast<u32x4_t *>(sm + W * VB);
    if (wv < NT) {
        v8 q[QP * KS];
        const float f = R::operands(a, score_factor<P>(a, s.kvh), raw, q);
#pragma unroll
        for (int i = 0; i < QP * KS; ++i) s_q[((i / KS * NT + wv) * KS + i % KS) * WAVE + l] = bits<u32x4_t>(q[i]);
        if (lg == 0) s_fac[wv * 16 + lr] = f;
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) rows.fac[nt] = s_fac[nt * 16 + lr];

    unsigned char *buf = sm + wv * VB;
    for (; t < s.t_end; t += W) {
        // keys of this tile that exist (uniform), and whether any row may not see one
        const uint32_t there =
            static_cast<uint32_t>(__ballot(slot[0] >= 0) & 0xFFFFu) | static_cast<uint32_t>(__ballot(slot[1] >= 0) & 0xFFFFu) << 16;
        // scores, for which V need not have arrived (it is loaded after K: 32 requests of 1024 keys 26.6 us when V came to LDS first);
        // the operands of a step are read while the step before is multiplied
        f32x4_t sc[NT][2];
        asm volatile("" ::: "memory");                            // or the operands would be kept in registers after all
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        v8 qb[2][QP * NT];
        auto load_q = [&](int k) {
#pragma unroll
            for (int i = 0; i < QP * NT; ++i) qb[k & 1][i] = bits<v8>(s_q[(i * KS + k) * WAVE + l]);
        };
        load_q(0);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            if (k + 1 < KS) load_q(k + 1);
            v8 kf[2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) kf[kt] = bits<v8>(operand_of<E, F8>(kr[kt], k));
#pragma unroll
            for (int i = 0; i < QP * NT; ++i)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) sc[i % NT][kt] = Types<E>::mfma(kf[kt], qb[k & 1][i], sc[i % NT][kt]);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, QP * NT, 0);          // LDS reads
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x100, QP * NT, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 2 * QP * NT, 0);  // MFMAs
        }
        const bool masked = (t + 1) * KT > s.at.past || there != 0xFFFFFFFFu;
        uint32_t special = 0;                                     // drafted keys with an infinity or NaN in V
        if (masked) {
            bool sp[2] = {false, false};
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int k = 0; k < LD; ++k) {
                    if (slot[kt] < 0) vr[kt][k] = u32x4_t{0u, 0u, 0u, 0u};
                    if (t * KT + kt * 16 + lr >= s.at.past) sp[kt] |= F8 ? f8_any_nan(vr[kt][k]) : any_special<E>(vr[kt][k]);
                }
            uint64_t b0 = __ballot(sp[0]), b1 = __ballot(sp[1]);
            if (b0 | b1) {
                b0 |= b0 >> 32;
                b1 |= b1 >> 32;
                special = static_cast<uint32_t>((b0 | b0 >> 16) & 0xFFFFu) | static_cast<uint32_t>((b1 | b1 >> 16) & 0xFFFFu) << 16;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int k = 0; k < LD; ++k) vr[kt][k] = special >> (kt * 16 + lr) & 1 ? u32x4_t{0u, 0u, 0u, 0u} : vr[kt][k];
            }
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int k = 0; k < KS; ++k)
                if constexpr (F8) *reinterpret_cast<u32x4_t *>(v_at<D>(buf, kt * 16 + lr, 4 * (k / 2) + lg, k % 2)) = operand_of<E, F8>(vr[kt], k);
                else *reinterpret_cast<u32x4_t *>(v_at<D>(buf, kt * 16 + lr, 2 * k + (lg >> 1), lg & 1)) = vr[kt][k];
        // the next tile's rows, in flight from here
        if (t + W < s.t_end) {
            load(t + W);
            if (t + 2 * W < s.t_end) look_up(t + 2 * W);
        }
        if (masked) rows.hide(sc, there, t * KT - s.at.past);
        rows.add(sc, buf);
        if (special) rows.template add_special<P>(sc, special, t, s, pg);
    }

    rows.drop();
    // join the waves: reference = the greatest, sums and rows scaled to it
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        rows.sum[nt] = row_sum(rows.sum[nt]);
        if (lg == 0) {
            s_ref[wv][nt * 16 + lr] = rows.ref[nt];
            s_sum[wv][nt * 16 + lr] = rows.sum[nt];
        }
    }
    __syncthreads();                                              // and every wave is done with its buffer
    float *js = reinterpret_cast<float *>(sm);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 16 + lr;
        float m = s_ref[0][r];
#pragma unroll
        for (int w = 1; w < W; ++w) m = fmaxf(m, s_ref[w][r]);
        const float own = rows.ref[nt] == NONE ? 0.f : __builtin_amdgcn_exp2f(rows.ref[nt] - m);
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4_t *>(js + (wv * NT * 16 + r) * DP + d * 16 + 4 * lg) = rows.acc[nt][d] * own;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 16 * (D / 4); i += W * WAVE) {
        const int r = i / (D / 4), c = i % (D / 4) * 4;
        f32x4_t o = *reinterpret_cast<f32x4_t *>(js + r * DP + c);
        float m = s_ref[0][r], total = 0.f;
#pragma unroll
        for (int w = 1; w < W; ++w) {
            o += *reinterpret_cast<f32x4_t *>(js + (w * NT * 16 + r) * DP + c);
            m = fmaxf(m, s_ref[w][r]);
        }
#pragma unroll
        for (int w = 0; w < W; ++w) total += s_ref[w][r] == NONE ? 0.f : s_sum[w][r] * __builtin_amdgcn_exp2f(s_ref[w][r] - m);
        R::template finish<P>(a, s, NT * 16, r, c, o, m, total);
    }
}

// More than 32 query rows: a wave has 32 of them (RW waves the block's 32 RW), and the RW waves share the K and V tiles, which
// they bring into LDS together: the cache is read once for 64 or 128 rows. KW such teams take every KW-th tile. Two
// buffers: a tile is written while the one before is multiplied and the one after is on its way from memory; one barrier a tile.
template <class E, bool PAIR, class P, int D, int RW, bool CUT>
__global__ void __launch_bounds__(waves_of(PAIR, RW) * WAVE, 2) k_tree_rows(Args a) {
    constexpr bool F8 = sizeof(P) == 1;
    constexpr int NT = 2, RWV = waves_of(PAIR, RW), KW = RWV / RW;
    typedef Rows<E, PAIR, D, NT> R;
    typedef typename R::v8 v8;
    constexpr int KS = R::KS, DT = R::DT, QP = R::QP, RB = D * 2, TB = KT * RB, DP = D + 4;
    // keys a wave; elements of the pool that a lane loads: 16 bytes of them, or 8 where a wave would have less than a load; lanes a row, rows a load,
    // its loads. In LDS a row is LCH 16-byte pieces of E
    constexpr int KPW = KT / RW, EPL = F8 ? (KPW * D >= 16 * WAVE ? 16 : 8) : 8, LPR = D / EPL, RPI = WAVE / LPR, SI = KPW / RPI, LCH = RB / 16, CPL = LCH / LPR;
    typedef std::conditional_t<F8 && EPL == 8, u32x2_t, u32x4_t> Got;
    static_assert(KW * RW == RWV && SI * RPI * RW == KT, "");
    constexpr int BUFS = 2 * KW * 2 * TB, JOIN = (KW - 1) * RW * 32 * DP * 4;
    __shared__ __align__(16) unsigned char sm[BUFS > JOIN ? BUFS : JOIN];
    // the operands of q stay in registers, but a pair's lo, which would not fit: in LDS, a copy for all teams
    __shared__ u32x4_t s_lo[PAIR ? RW * NT * KS * WAVE : 1];
    __shared__ uint32_t s_there[2][KW][RW], s_special[2][KW][RW];
    __shared__ float s_ref[RWV][NT * 16], s_sum[RWV][NT * 16];
    const int wv = threadIdx.x >> 6, l = threadIdx.x & 63, lr = l & 15, lg = l >> 4, rw = wv % RW, kw = wv / RW;
    const Share s = share_of<CUT>(a, RW * 32);
    if (s.none) return;
    const int qrow0 = s.group * RW * 32 + rw * 32;
    const Pages pg{a.table + static_cast<size_t>(s.req) * a.blocks, min(s.at.len, s.t_end * KT), a};

    // staging: this lane's EPL elements of rows rw KPW + i RPI + l / LPR of the tile
    const int c = l % LPR, r0 = rw * KPW + l / LPR;
    Got kr[SI], vr[SI];
    int slot[SI], page[SI];
    const P *kb = static_cast<const P *>(a.k) + s.kvh * D + EPL * c, *vb = static_cast<const P *>(a.v) + s.kvh * D + EPL * c;
    auto look_up = [&](int t) {
#pragma unroll
        for (int i = 0; i < SI; ++i) page[i] = pg.page_of(t * KT + r0 + i * RPI);
    };
    auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < SI; ++i) {
            slot[i] = pg.slot_of(t * KT + r0 + i * RPI, page[i]);
            const size_t at = static_cast<size_t>(max(slot[i], 0)) * a.ldkv;
            kr[i] = *(const NAVI_GLOBAL Got *) (kb + at);
            vr[i] = *(const NAVI_GLOBAL Got *) (vb + at);
        }
    };
    auto bits_of = [&](uint64_t b, int i) {                       // a ballot over load i's rows as bits of the tile's keys
        uint32_t x = 0;
#pragma unroll
        for (int r = 0; r < RPI; ++r) x |= static_cast<uint32_t>((b >> (r * LPR) & ((uint64_t(1) << LPR) - 1)) != 0) << r;
        return x << (rw * KPW + i * RPI);
    };
    auto as_e = [](const Got &g, int j) {                         // the load's j-th 16 bytes of E
        if constexpr (F8) {
            u32x4_t one[1];
            if constexpr (EPL == 16) one[0] = g;
            else one[0] = u32x4_t{g[0], g[1], 0u, 0u};
            return operand_of<E, true>(one, j);
        } else {
            return g;
        }
    };
    auto put = [&](int b, int t) {
        unsigned char *kd = sm + (b * KW + kw) * 2 * TB, *vd = kd + TB;
        // all of them there and cached: seen by all rows
        bool plain = (t + 1) * KT <= s.at.past;
#pragma unroll
        for (int i = 0; i < SI; ++i) plain = plain && slot[i] >= 0;
        uint32_t there = ((KPW < 32 ? 1u << (KPW & 31) : 0u) - 1u) << (rw * KPW), special = 0;
        if (__ballot(!plain)) {
            there = 0;
#pragma unroll
            for (int i = 0; i < SI; ++i) {
                there |= bits_of(__ballot(slot[i] >= 0), i);
                vr[i] = slot[i] < 0 ? Got(0u) : vr[i];
                bool odd;
                if constexpr (F8 && EPL == 8) odd = f8_any_nan(u32x4_t{vr[i][0], vr[i][1], 0u, 0u});
                else if constexpr (F8) odd = f8_any_nan(vr[i]);
                else odd = any_special<E>(vr[i]);
                const uint32_t x = bits_of(__ballot(t * KT + r0 + i * RPI >= s.at.past && odd), i);
                special |= x;
                vr[i] = x >> (r0 + i * RPI) & 1 ? Got(0u) : vr[i];
            }
        }
#pragma unroll
        for (int i = 0; i < SI; ++i) {
            const int r = r0 + i * RPI;
#pragma unroll
            for (int j = 0; j < CPL; ++j) {
                const int p = c * CPL + j;
                *reinterpret_cast<u32x4_t *>(kd + r * RB + ((p ^ (r & (LCH - 1))) << 4)) = as_e(kr[i], j);
                *reinterpret_cast<u32x4_t *>(v_at<D>(vd, r, p >> 1, p & 1)) = as_e(vr[i], j);
            }
        }
        if (l == 0) {
            s_there[b][kw][rw] = there;
            s_special[b][kw][rw] = special;
        }
    };

    int t = s.t0 + kw;
    const int turns = (s.t_end - s.t0 + KW - 1) / KW;             // the same for all waves: past its tiles a team has none there
    look_up(t);
    R rows;
    rows.start(a, s, qrow0);
    load(t);
    look_up(t + KW);
    v8 q[NT][KS];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        v8 x[QP * KS];
        typename R::Raw raw;
        R::template fetch<false>(a, s, qrow0 + nt * 16 + lr, raw);
        rows.fac[nt] = R::operands(a, score_factor<P>(a, s.kvh), raw, x);
#pragma unroll
        for (int i = 0; i < QP * KS; ++i)
            if (i < KS) q[nt][i] = x[i];
            else if (kw == 0) s_lo[((rw * NT + nt) * KS + i - KS) * WAVE + l] = bits<u32x4_t>(x[i]);
    }
    put(0, t);
    load(t + KW);
    look_up(t + 2 * KW);
    for (int turn = 0; turn < turns; ++turn, t += KW) {
        const int b = turn & 1;
        __syncthreads();                                          // tile t is in LDS, and tile t - KW has been used
        if (turn + 1 < turns) {
            put(b ^ 1, t + KW);
            load(t + 2 * KW);
            look_up(t + 3 * KW);
        }
        uint32_t there = 0, special = 0;
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            there |= s_there[b][kw][i];
            special |= s_special[b][kw][i];
        }
        there = __builtin_amdgcn_readfirstlane(there);
        special = __builtin_amdgcn_readfirstlane(special);
        unsigned char *kd = sm + (b * KW + kw) * 2 * TB;
        f32x4_t sc[NT][2];
        if constexpr (PAIR) asm volatile("" ::: "memory");          // or lo would be kept in registers after all
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            v8 kf[2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const int r = kt * 16 + lr;
                kf[kt] = bits<v8>(*reinterpret_cast<u32x4_t *>(kd + r * RB + (((4 * k + lg) ^ (r & (LCH - 1))) << 4)));
            }
#pragma unroll
            for (int p = 0; p < QP; ++p)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const v8 x = p == 0 ? q[nt][k] : bits<v8>(s_lo[((rw * NT + nt) * KS + k) * WAVE + l]);
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) sc[nt][kt] = Types<E>::mfma(kf[kt], x, sc[nt][kt]);
                }
        }
        if ((t + 1) * KT > s.at.past || there != 0xFFFFFFFFu) rows.hide(sc, there, t * KT - s.at.past);
        rows.add(sc, kd + TB);
        if (special) rows.template add_special<P>(sc, special, t, s, pg);
    }

    rows.drop();
    // join the teams' results through LDS: reference = the greatest, sums and rows scaled to it; the first team adds and stores
    float *js = reinterpret_cast<float *>(sm);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        rows.sum[nt] = row_sum(rows.sum[nt]);
        if (lg == 0) {
            s_ref[wv][nt * 16 + lr] = rows.ref[nt];
            s_sum[wv][nt * 16 + lr] = rows.sum[nt];
        }
    }
    __syncthreads();                                              // and every wave is done with the buffers
    float m[NT], total[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 16 + lr;
        m[nt] = s_ref[rw][r];
#pragma unroll
        for (int w = 1; w < KW; ++w) m[nt] = fmaxf(m[nt], s_ref[w * RW + rw][r]);
        total[nt] = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
            const float x = s_ref[w * RW + rw][r];
            total[nt] += x == NONE ? 0.f : s_sum[w * RW + rw][r] * __builtin_amdgcn_exp2f(x - m[nt]);
        }
        const float own = rows.ref[nt] == NONE ? 0.f : __builtin_amdgcn_exp2f(rows.ref[nt] - m[nt]);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            rows.acc[nt][d] *= own;
            if (kw > 0) *reinterpret_cast<f32x4_t *>(js + (((kw - 1) * RW + rw) * 32 + r) * DP + d * 16 + 4 * lg) = rows.acc[nt][d];
        }
    }
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            f32x4_t o = rows.acc[nt][d];
#pragma unroll
            for (int w = 1; w < KW; ++w) o += *reinterpret_cast<f32x4_t *>(js + (((w - 1) * RW + rw) * 32 + nt * 16 + lr) * DP + d * 16 + 4 * lg);
            R::template finish<P>(a, s, RW * 32, rw * 32 + nt * 16 + lr, d * 16 + 4 * lg, o, m[nt], total[nt]);
        }
}

// Joins the parts of the requests that were cut, in their order: a wave takes a query row, D / 8 lanes its
// columns and the others further parts. Block (request x kv head x group, rows).
template <class E, bool PAIR, class P, int D>
__global__ void __launch_bounds__(BT) k_tree_join(Args a, int group_rows) {
    constexpr int CL = D / 8, PL = WAVE / CL;
    const int l = threadIdx.x & 63, c = l % CL, pl = l / CL;
    int id = blockIdx.x;
    const int kvh = id % a.hkv;
    id /= a.hkv;
    const int group = id % a.groups, req = id / a.groups, qrow0 = group * group_rows;
    const uint32_t b0 = gld(a.first + group * (a.n + 1) + req), b1 = gld(a.first + group * (a.n + 1) + req + 1);
    const int k0 = static_cast<int>(b0 >> 16), k1 = static_cast<int>(b1 >> 16);
    if (k0 == k1) return;                                         // a block had all of it and has stored it
    const Where wh = where_is(a, req);
    const int left = min(group_rows, wh.rows * a.g - qrow0);
    for (int r = blockIdx.y * NW + (threadIdx.x >> 6); r < left; r += gridDim.y * NW) {
        float m = NONE, sum = 0.f;
        f32x4_t o[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll 4
        for (int k = k0 + pl; k < k1; k += PL) {
            const size_t at = part_of(a, kvh, group, k) * group_rows + r;
            const float ref = gld(a.pm + 2 * at), z = gld(a.pm + 2 * at + 1);
            const f32x4_t x0 = ld4(a.po + at * D + 8 * c), x1 = ld4(a.po + at * D + 8 * c + 4);
            const float top = fmaxf(m, ref);
            const float fo = m == NONE ? 0.f : __builtin_amdgcn_exp2f(m - top), fx = ref == NONE ? 0.f : __builtin_amdgcn_exp2f(ref - top);
            m = top;
            sum = sum * fo + z * fx;
            o[0] = o[0] * fo + x0 * fx;
            o[1] = o[1] * fo + x1 * fx;
        }
        float top = m;
#pragma unroll
        for (int x = CL; x < WAVE; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float f = m == NONE ? 0.f : __builtin_amdgcn_exp2f(m - top);
        sum *= f;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i >> 2][i & 3] *= f;
#pragma unroll
        for (int x = CL; x < WAVE; x <<= 1) {
            sum += __shfl_xor(sum, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i >> 2][i & 3] += __shfl_xor(o[i >> 2][i & 3], x);
        }
        if (pl == 0) {
            const int mrow = qrow0 + r, j = div_by(a.heads_per, mrow), head = kvh * a.g + mrow - j * a.g;
            const float inv = top == NONE ? 0.f : value_factor<P>(a, kvh) / sum;
            store_out<E, PAIR>(a, wh.c0 + j, head * D + 8 * c, a.hkv * a.g * D, o[0] * inv);
            store_out<E, PAIR>(a, wh.c0 + j, head * D + 8 * c + 4, a.hkv * a.g * D, o[1] * inv);
        }
    }
}

// How a call is cut: query tiles and, above 32 query rows, waves that share them (waves 1: none share), rows of a group and
// groups, and blocks wanted for a kv head and group (0: one a request).
struct Cut {
    int tiles, waves, rows, groups, workers, step, parts;
};
Cut cut_of(const navi_kv_pages &p, const navi_kv_heads &h, int max_keys, bool pair) {
    const int m = std::min(p.max_new, 64) * (h.n_head / h.n_kv_head);
    Cut c;
    c.tiles = m <= 16 ? 1 : 2;
    c.waves = m <= 32 ? 1 : m <= 64 ? 2 : 4;
    c.rows = 16 * c.tiles * c.waves;
    c.groups = (m + c.rows - 1) / c.rows;
    const int64_t heads = static_cast<int64_t>(h.n_kv_head) * c.groups;
    const int waves = c.waves == 1 ? alone_of(true) : waves_of(pair, c.waves);
    c.step = waves / c.waves;                           // tiles of a block's turn
    const int steps = (max_keys + KT * c.step - 1) / (KT * c.step);
    // A block a request where no request can be long enough to share (one row of 16 heads over 256 keys: 8.6 us, cut 10.6; over
    // 512: 11.9 and 10.5); where there are blocks for all CUs and no request is long; and for more requests than a block lays out,
    // whatever their lengths (of 1 to 1000 keys: 256 requests 70 us, 300 81; of 1 to 32768: 950 and 1000). Else enough blocks for
    // all waves of the CUs. The second rule is a choice, since the host knows the most keys and not the lengths: cutting costs a
    // batch of even lengths the layout and the join, and gains where they are uneven, the more the longer the longest. 32 requests,
    // us uncut / cut, all alike and of lengths spread down to one:
    //   one row, up to 1000 keys 25.6 / 30.2 and 19.6 / 14.4, 1400 38.2 / 44.5 and 24.9 / 19.3, 2000 53.6 / 59.0 and 34.3 / 22.6;
    //   24 rows (48 query rows), up to 600 keys 26.0 / 33.8 and 22.8 / 22.4, 1000 37.3 / 42.8 and 31.3 / 27.6, 1400 54.8 / 59.7 and
    //   42.4 / 30.9.
    // Below 1280 keys even batches are favoured, above uneven ones. Just past a block a CU an uncut call pays a second round: 33
    // requests of one row, up to 1000 keys, 42.7 / 37.2 and 19.7 / 16.7; 48 requests 49.6 / 47.2 and 20.0 / 20.0.
    if (p.n_requests > MAXB || steps == 1 || (c.waves == 1 && max_keys <= 384) || (max_keys <= 1280 && p.n_requests * heads >= 256)) {
        c.workers = c.parts = 0;
        return c;
    }
    const int64_t blocks = 2048 / waves;                           // two waves a SIMD
    c.workers = static_cast<int>(std::max<int64_t>(1, std::min((blocks + heads - 1) / heads, static_cast<int64_t>(steps) * p.n_requests)));
    c.parts = std::min(c.workers + p.n_requests, 2 * c.workers);
    return c;
}

// Rows of the parts: the workspace has head_dim floats for each, then two for each, then the first chunks.
size_t part_rows(const navi_kv_heads &h, const Cut &c) {
    return static_cast<size_t>(h.n_kv_head) * c.groups * c.parts * c.rows;
}

size_t workspace(const navi_kv_pages &p, const navi_kv_heads &h, int max_keys) {
    // q's type is not known here: enough for either
    size_t need = 0;
    for (const bool pair : {false, true}) {
        const Cut c = cut_of(p, h, max_keys, pair);
        if (c.workers > 0)
            need = std::max(need, part_rows(h, c) * (h.head_dim + 2) * sizeof(float) + static_cast<size_t>(c.groups) * (p.n_requests + 1) * sizeof(int32_t));
    }
    return need;
}

template <class E, bool PAIR, class P, int D, bool CUT>
void launch_cut(const Args &a, const Cut &c, hipStream_t s) {
    const dim3 rbt(static_cast<unsigned>(waves_of(PAIR, c.waves) * WAVE));
    const dim3 grid(static_cast<unsigned>(CUT ? c.workers + a.n : a.n) * a.groups * a.hkv);
    const dim3 abt(alone_of(CUT) * WAVE);
    if (c.tiles == 1) hipLaunchKernelGGL((k_tree<E, PAIR, P, D, 1, CUT>), grid, abt, 0, s, a);
    else if (c.waves == 1) hipLaunchKernelGGL((k_tree<E, PAIR, P, D, 2, CUT>), grid, abt, 0, s, a);
    else if (c.waves == 2) hipLaunchKernelGGL((k_tree_rows<E, PAIR, P, D, 2, CUT>), grid, rbt, 0, s, a);
    else hipLaunchKernelGGL((k_tree_rows<E, PAIR, P, D, 4, CUT>), grid, rbt, 0, s, a);
}

template <class E, bool PAIR, class P, int D>
void launch_as(const Args &a, const Cut &c, hipStream_t s) {
    if (c.workers == 0) return launch_cut<E, PAIR, P, D, false>(a, c, s);
    launch_cut<E, PAIR, P, D, true>(a, c, s);
    const unsigned units = static_cast<unsigned>(a.n) * a.groups * a.hkv;
    hipLaunchKernelGGL((k_tree_join<E, PAIR, P, D>), dim3(units, std::max(1u, std::min(static_cast<unsigned>(c.rows / NW), 1024u / units))), dim3(BT), 0, s,
                       a, c.rows);
}

template <int D>
void launch_dim(const Args &a, const Cut &c, int q_dtype, int kv_dtype, hipStream_t s) {
    const bool pair = q_dtype == NAVI_DT_F32, bf = q_dtype == NAVI_DT_BF16;
    if (kv_dtype == NAVI_DT_F8E4M3) {
        if (pair) launch_as<_Float16, true, f8_t, D>(a, c, s);
        else if (bf) launch_as<__bf16, false, f8_t, D>(a, c, s);
        else launch_as<_Float16, false, f8_t, D>(a, c, s);
    } else {
        if (pair) launch_as<_Float16, true, _Float16, D>(a, c, s);
        else if (bf) launch_as<__bf16, false, __bf16, D>(a, c, s);
        else launch_as<_Float16, false, _Float16, D>(a, c, s);
    }
}

void launch(const Call &x, hipStream_t s) {
    const navi_kv_pages &p = *x.pages;
    const navi_kv_heads &h = *x.heads;
    const bool pair = x.q_dtype == NAVI_DT_F32;
    const Cut c = cut_of(p, h, x.max_keys, pair);
    Args a{};
    a.q = x.q;
    a.k = x.k;
    a.v = x.v;
    if (h.kv_dtype == NAVI_DT_F8E4M3) {
        a.ks = h.k_scale;
        a.vs = h.v_scale;
    }
    a.out = x.out;
    a.po = static_cast<float *>(x.ws);
    if (a.po) {
        a.pm = a.po + part_rows(h, c) * h.head_dim;
        a.first = reinterpret_cast<uint32_t *>(a.pm + 2 * part_rows(h, c));
    }
    a.table = p.block_table;
    a.n_past = p.n_past;
    a.cu = p.cu_rows;
    a.slot = x.slots ? p.row_slot : nullptr;
    a.mask = p.row_mask;
    a.n = p.n_requests;
    a.hkv = h.n_kv_head;
    a.g = h.n_head / h.n_kv_head;
    a.blocks = p.max_blocks;
    a.n_pages = p.n_pages;
    a.n_rows = p.n_rows;
    a.max_new = p.max_new;
    a.ldq = x.ldq;
    a.ldkv = x.ldkv;
    a.ldo = x.ldo;
    a.workers = c.workers;
    a.step = c.step;
    a.parts = c.parts;
    a.groups = c.groups;
    a.tiled = x.tiled;
    a.page = kv::make_div(static_cast<uint32_t>(p.page_size));
    a.heads_per = kv::make_div(static_cast<uint32_t>(a.g));
    a.flip = x.scale < 0.f;
    a.scale = std::fabs(x.scale) * 1.44269504088896340736f;
    if (h.head_dim == 128) launch_dim<128>(a, c, x.q_dtype, h.kv_dtype, s);
    else launch_dim<64>(a, c, x.q_dtype, h.kv_dtype, s);
}

} // namespace tree
} // namespace navi_amd

using namespace navi_amd;

extern "C" {

size_t navi_tree_workspace(const navi_kv_pages *pages, const navi_kv_heads *heads, int32_t max_keys) {
    if (kv::check_pages("tree_workspace", pages, nullptr, 0) != NAVI_OK || !heads ||
        kv::check_heads("tree_workspace", heads, heads->n_kv_head * heads->head_dim, nullptr, 0) != NAVI_OK || pages->max_new > 64 || max_keys < 1)
        return 0;
    return tree::workspace(*pages, *heads, max_keys);
}

navi_status navi_tree_attention(const navi_kv_pages *pages, const navi_kv_heads *heads, const void *d_q, int32_t q_dtype, int32_t ldq,
                                const void *d_k, const void *d_v, int32_t ld_kv, float scale, int32_t max_keys, void *d_out,
                                int32_t ldo, void *d_ws, size_t ws_bytes, void *stream, char *err, size_t errlen) {
    navi_status st = kv::check_pages("tree_attention", pages, err, errlen);
    if (st == NAVI_OK) st = kv::check_heads("tree_attention", heads, ld_kv, err, errlen);
    if (st != NAVI_OK) return st;
    const long width = static_cast<long>(heads->n_head) * heads->head_dim;
    const bool known = heads->kv_dtype == NAVI_DT_F8E4M3 ? q_dtype == NAVI_DT_F32 || q_dtype == NAVI_DT_F16 || q_dtype == NAVI_DT_BF16
                                                         : q_dtype == heads->kv_dtype || (q_dtype == NAVI_DT_F32 && heads->kv_dtype == NAVI_DT_F16);
    if (!known) {
        set_err(err, errlen, "tree_attention: unsupported types (q %d, cache %d): the cache's type, or f32 over f16, or any over e4m3", q_dtype, heads->kv_dtype);
        return NAVI_ERR_UNSUPPORTED;
    }
    if (pages->max_new > 64) {
        set_err(err, errlen, "tree_attention: up to %d rows a request; at most 64", pages->max_new);
        return NAVI_ERR_INVALID;
    }
    if (!kv::rows_ok(d_q, pages->n_rows, q_dtype, ldq, width) || !kv::rows_ok(d_out, pages->n_rows, q_dtype, ldo, width) || !d_k || !d_v || !kv::aligned16(d_k) ||
        !kv::aligned16(d_v)) {
        set_err(err, errlen, "tree_attention: a null or misaligned pointer, or a stride too small (ldq %d, ldo %d)", ldq, ldo);
        return NAVI_ERR_INVALID;
    }
    if (max_keys < 1 || max_keys > INT32_MAX - 64) {
        set_err(err, errlen, "tree_attention: max_keys %d out of range", max_keys);
        return NAVI_ERR_INVALID;
    }
    // at most n_requests * n_head blocks of 512 threads, and a launch has less than 2^32
    if (static_cast<int64_t>(pages->n_requests) * heads->n_head * 512 > UINT32_MAX) {
        set_err(err, errlen, "tree_attention: %d requests of %d heads are too many for one call", pages->n_requests, heads->n_head);
        return NAVI_ERR_INVALID;
    }
    if (!std::isfinite(scale)) {
        set_err(err, errlen, "tree_attention: scale %g", static_cast<double>(scale));
        return NAVI_ERR_INVALID;
    }
    if (d_out && d_out == d_q && ldo != ldq) {
        set_err(err, errlen, "tree_attention: d_out over d_q of another stride (%d, %d)", ldo, ldq);
        return NAVI_ERR_INVALID;
    }
    const size_t need = tree::workspace(*pages, *heads, max_keys);
    if (need > 0 && (!d_ws || !kv::aligned16(d_ws) || ws_bytes < need)) {
        set_err(err, errlen, "tree_attention: the workspace is null, misaligned or smaller than %zu bytes (%zu)", need, ws_bytes);
        return NAVI_ERR_INVALID;
    }
    kv::OnDevice dev;
    if ((st = dev.enter(stream, "tree_attention", err, errlen)) != NAVI_OK) return st;
    if (pages->n_rows == 0) return NAVI_OK;
    tree::launch({pages, heads, d_q, d_k, d_v, d_out, d_ws, q_dtype, ldq, ld_kv, ldo, max_keys, scale, false, false},
                 static_cast<hipStream_t>(stream));
    NAVI_TRY_HIP(hipGetLastError(), err, errlen);
    return NAVI_OK;
}

} // extern "C"

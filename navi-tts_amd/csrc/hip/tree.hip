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
//    its registers, and a row's maximum, sum and mask are a lane's own values.
//  * V^T's operand is V read from LDS through the transposing load (ds_read_b64_tr_b16: in a
//    16-lane group lane 4r + c fetches columns 4c.. of key r and gets column `lane`, keys 0..3). V rows sit
//    in LDS with their 32-byte chunks XORed by the key, so that the 16 rows such a load touches
//    spread over all banks. K goes from memory to registers in operand form.
//  * A wave works alone on its own 32-key tiles (every fourth of the block's range), with its own V buffer
//    and no barrier until its range ends; then the block's four partial results are joined in LDS.
//  * Softmax against a reference value that moves only when a score passes it by more than SLACK: the
//    rescaling, and the maximum over lanes that it needs, are off the common path. exp2 with the scale folded in.
//  * Few requests: a request's keys are split over several blocks, whose partial results (unnormalised sums,
//    reference, sum) a second kernel joins in split order.
#include "dev_common.h"
#include "tile_layout.h"
#include "tree.h"

#include <algorithm>
#include <cmath>

namespace navi_amd {
namespace tree {

using kv::Div;
using kv::div_by;

constexpr int NW = 4, BT = NW * WAVE;  // waves of a block
constexpr int KT = 32;                 // keys of a wave's tile
// p = 2^(s - reference + LIFT): at most 2^(SLACK + LIFT) = 2^14, inside f16, and f16's full precision down to
// 2^-24 of the reference instead of 2^-14.
constexpr float SLACK = 4.f, LIFT = 10.f;
constexpr float NONE = -INFINITY;

struct Args {
    const void *q, *k, *v;
    void *out;
    float *po, *pm;                    // the parts of requests that are cut (part_of)
    const int32_t *table, *n_past, *cu;
    const uint64_t *mask;
    int n, hkv, g, blocks, n_pages, n_rows, max_new, ldq, ldkv, ldo, workers, groups;
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
    w.c0 = gld(a.cu + req);
    const int count = max(min(gld(a.cu + req + 1), a.n_rows) - w.c0, 0);
    w.rows = min(count, a.max_new);
    w.past = static_cast<int>(min<int64_t>(max(gld(a.n_past + req), 0), room));
    w.len = static_cast<int>(min<int64_t>(static_cast<int64_t>(w.past) + count, room));
    return w;
}

// Requests of uneven length over evenly long chunks: with `workers` wanted blocks a kv head and query group, a chunk is
// at most total / workers steps (of KT * NW keys), and a request is cut into as few even chunks of that as it takes:
// at most workers + requests of them, in the requests' order.
constexpr int MAXB = BT;               // most requests of a call that is cut
struct Chunks {
    int before[MAXB + 1];              // chunks before request i
    int steps[MAXB];
    Where at[MAXB];
    int red[NW];
    float sum[NW];
};
__device__ __forceinline__ int block_upto(int v, int *red) {
    const int wv = threadIdx.x >> 6, upto = wave_incl_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) red[wv] = upto;
    __syncthreads();
    int off = 0;
#pragma unroll
    for (int i = 0; i < NW - 1; ++i) off += i < wv ? red[i] : 0;
    return off + upto;
}
__device__ __forceinline__ void lay_out(const Args &a, int qrow0, Chunks &q) {
    const int t = threadIdx.x;
    Where w{0, 0, 0, 0};
    if (t < a.n) w = where_is(a, t);
    const int steps = w.rows * a.g > qrow0 ? (w.len + KT * NW - 1) / (KT * NW) : 0;
    // the steps in all, exact below 2^24; above (lengths out of all proportion) rounded up, so that the chunks stay as few
    const float part = wave_sum(static_cast<float>(steps));
    if ((t & 63) == 0) q.sum[t >> 6] = part;
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) total += q.sum[i];
    const int most = max(total < 16777216.f ? (static_cast<int>(total) + a.workers - 1) / a.workers
                                            : static_cast<int>(total * 1.001f / static_cast<float>(a.workers)) + 1, 1);
    const int chunks = block_upto((steps + most - 1) / most, q.red);
    if (t == 0) q.before[0] = 0;
    if (t < a.n) {
        q.before[t + 1] = chunks;
        q.steps[t] = steps;
        q.at[t] = w;
    }
    __syncthreads();
}
// Where chunk k's part is kept: NT * 16 rows of [D], and (reference, sum) pairs.
__device__ __forceinline__ size_t part_of(const Args &a, int kvh, int group, int k) {
    return (static_cast<size_t>(kvh) * a.groups + group) * (a.workers + a.n) + k;
}

// PAIR: q and out are f32, q and p travel as hi + lo pairs. NT: 16-row query tiles of a block. CUT: a block takes a
// chunk of a request's keys, else all of them.
template <class E, bool PAIR, int D, int NT, bool CUT>
__global__ void __launch_bounds__(BT, NT == 1 ? 3 : NT == 2 ? 2 : 1) k_tree(Args a) {
    typedef typename Types<E>::v8 v8;
    typedef typename Types<E>::v4 v4;
    constexpr int KS = D / 32, DT = D / 16;                      // MFMA steps of a score, column tiles of O
    constexpr int VB = KT * D * 2 > NT * 16 * KT * 4 ? KT * D * 2 : NT * 16 * KT * 4;   // a wave's buffer, bytes
    constexpr int CD = D / NT, CDP = CD + 4;                     // columns joined at a time, padded
    constexpr int JOIN = NW * NT * 16 * CDP * 4;
    __shared__ __align__(16) unsigned char sm[NW * VB > JOIN ? NW * VB : JOIN];
    __shared__ float s_ref[NW][NT * 16], s_sum[NW][NT * 16];
    constexpr int QP = PAIR ? 2 : 1;
    __shared__ u32x4_t s_q[QP * NT * KS * WAVE];      // the operands of q, a pair's hi before its lo

    const int wv = threadIdx.x >> 6, l = threadIdx.x & 63, lr = l & 15, lg = l >> 4;
    int id = blockIdx.x;
    const int kvh = id % a.hkv;
    id /= a.hkv;
    const int group = id % a.groups, unit = id / a.groups;
    const int qrow0 = group * NT * 16;

    int req = unit, t0 = 0, t_end;
    bool whole = true;                                            // the block has all of the request's keys
    Where wh;
    if constexpr (CUT) {
        __shared__ Chunks s_c;
        lay_out(a, qrow0, s_c);
        if (unit >= s_c.before[a.n]) return;
        int lo = 0, hi = a.n;                                     // before[lo] <= unit < before[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_c.before[mid] <= unit) lo = mid;
            else hi = mid;
        }
        req = lo;
        wh = s_c.at[req];
        const int n = s_c.before[req + 1] - s_c.before[req], k = unit - s_c.before[req], steps = s_c.steps[req];
        whole = n == 1;
        t0 = static_cast<int>(static_cast<int64_t>(steps) * k / n) * NW;
        t_end = min((wh.len + KT - 1) / KT, static_cast<int>(static_cast<int64_t>(steps) * (k + 1) / n) * NW);
    } else {
        wh = where_is(a, req);
        if (qrow0 >= wh.rows * a.g) return;                       // uniform: this request has fewer rows
        t_end = (wh.len + KT - 1) / KT;
    }
    const int c0 = wh.c0, rows = wh.rows, past = wh.past, len = wh.len;

    // this lane's query rows (one a tile): masks and factor of the scores; the operands into LDS
    uint64_t seen[NT];
    float fac[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int m = qrow0 + nt * 16 + lr, j = div_by(a.heads_per, m);
        const bool on = j < rows;
        seen[nt] = on ? gld(a.mask + c0 + j) : 0;
        fac[nt] = a.scale;
        const size_t at = static_cast<size_t>(c0 + (on ? j : 0)) * a.ldq + static_cast<size_t>(kvh * a.g + (on ? m - j * a.g : 0)) * D + 8 * lg;
        if constexpr (PAIR) {
            // q times a power of two that puts the row's largest value into [1, 2): pairs keep 22 bits of it
            // whatever its range; the scores get the inverse
            const float *q = static_cast<const float *>(a.q) + at;
            f32x4_t x[KS][2];
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    x[s][hf] = on ? ld4(q + 32 * s + 4 * hf) : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[s][hf][e]));
                }
            top = row_max(top);
            const int ex = top > 0.f && top < INFINITY ? ilogbf(top) : 0;
            fac[nt] = ldexpf(a.scale, ex);
            if (wv == 0) {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    v8 qhi, qlo;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float y = ldexpf(a.flip ? -x[s][e >> 2][e & 3] : x[s][e >> 2][e & 3], -ex);
                        qhi[e] = static_cast<E>(y);
                        qlo[e] = static_cast<E>(y - static_cast<float>(qhi[e]));
                    }
                    s_q[(nt * KS + s) * WAVE + l] = bits<u32x4_t>(qhi);
                    s_q[((NT + nt) * KS + s) * WAVE + l] = bits<u32x4_t>(qlo);
                }
            }
        } else {
            const E *q = static_cast<const E *>(a.q) + at;
            if (wv == 0) {
                const uint32_t sign = a.flip ? 0x80008000u : 0u;
#pragma unroll
                for (int s = 0; s < KS; ++s)
                    s_q[(nt * KS + s) * WAVE + l] = on ? *(const NAVI_GLOBAL u32x4_t *) (q + 32 * s) ^ sign : u32x4_t{0u, 0u, 0u, 0u};
            }
        }
        // a factor of 0 (all scores alike) as the least normal number: -inf, a place not seen, must stay -inf
        fac[nt] = fmaxf(fac[nt], 1.17549435e-38f);
    }

    f32x4_t acc[NT][DT];
    float ref[NT], sub[NT], sum[NT];                          // ref: the reference + SLACK; sub: reference - LIFT
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        ref[nt] = NONE;
        sub[nt] = sum[nt] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[nt][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    unsigned char *buf = sm + wv * VB;
    const E *kb = static_cast<const E *>(a.k) + kvh * D + 8 * lg, *vb = static_cast<const E *>(a.v) + kvh * D + 8 * lg;
    const int32_t *table = a.table + static_cast<size_t>(req) * a.blocks;
    // page and place in it of key `key`; slot: its row, or -1 past the end and outside the pool
    auto page_of = [&](int key) { return key < len ? gld(table + div_by(a.page, key)) : -1; };
    auto slot_of = [&](int key, int p) {
        return static_cast<unsigned>(p) < static_cast<unsigned>(a.n_pages)
                   ? p * static_cast<int>(a.page.d) + key - div_by(a.page, key) * static_cast<int>(a.page.d) : -1;
    };
    u32x4_t kr[2][KS], vr[2][KS];
    int slot[2], page[2];
    auto load_kv = [&]() {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const size_t at = static_cast<size_t>(max(slot[kt], 0)) * a.ldkv;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                kr[kt][s] = *(const NAVI_GLOBAL u32x4_t *) (kb + at + 32 * s);
                vr[kt][s] = *(const NAVI_GLOBAL u32x4_t *) (vb + at + 32 * s);
            }
        }
    };
    int t = t0 + wv;
    if (t < t_end) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) page[kt] = page_of(t * KT + kt * 16 + lr);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) slot[kt] = slot_of(t * KT + kt * 16 + lr, page[kt]);
        load_kv();
        if (t + NW < t_end)                                   // pages are looked up two tiles ahead
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) page[kt] = page_of((t + NW) * KT + kt * 16 + lr);
    }
    __syncthreads();                                              // the operands of q
    for (; t < t_end; t += NW) {
        // keys of this tile that exist (uniform), and whether any row may not see one
        const uint32_t there =
            static_cast<uint32_t>(__ballot(slot[0] >= 0) & 0xFFFFu) | static_cast<uint32_t>(__ballot(slot[1] >= 0) & 0xFFFFu) << 16;
        const bool masked = (t + 1) * KT > past || there != 0xFFFFFFFFu;
        // V rows into LDS: 32-byte chunk i of key r at chunk i ^ (r & 7)
        uint32_t special = 0;                                 // drafted keys with an infinity or NaN in V
        if (masked) {
            bool sp[2] = {false, false};
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    if (slot[kt] < 0) vr[kt][s] = u32x4_t{0u, 0u, 0u, 0u};
                    if (t * KT + kt * 16 + lr >= past) sp[kt] |= any_special<E>(vr[kt][s]);
                }
            uint64_t b0 = __ballot(sp[0]), b1 = __ballot(sp[1]);
            if (b0 | b1) {
                b0 |= b0 >> 32;
                b1 |= b1 >> 32;
                special = static_cast<uint32_t>((b0 | b0 >> 16) & 0xFFFFu) | static_cast<uint32_t>((b1 | b1 >> 16) & 0xFFFFu) << 16;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
                    if (special >> (kt * 16 + lr) & 1)
#pragma unroll
                        for (int s = 0; s < KS; ++s) vr[kt][s] = u32x4_t{0u, 0u, 0u, 0u};
            }
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int r = kt * 16 + lr, ch = 2 * s + (lg >> 1);
                *reinterpret_cast<u32x4_t *>(buf + r * (D * 2) + ((ch ^ (r & (DT - 1))) << 5) + ((lg & 1) << 4)) = vr[kt][s];
            }
        // scores
        f32x4_t sc[NT][2];
        asm volatile("" ::: "memory");                        // or the operands would be kept in registers after all
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        // the operands of a step are read while the step before is multiplied
        v8 qb[2][QP * NT];
        auto load_q = [&](int s) {
#pragma unroll
            for (int i = 0; i < QP * NT; ++i) qb[s & 1][i] = bits<v8>(s_q[(i * KS + s) * WAVE + l]);
        };
        load_q(0);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (s + 1 < KS) load_q(s + 1);
#pragma unroll
            for (int i = 0; i < QP * NT; ++i)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) sc[i % NT][kt] = Types<E>::mfma(bits<v8>(kr[kt][s]), qb[s & 1][i], sc[i % NT][kt]);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, QP * NT, 0);          // LDS reads
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            __builtin_amdgcn_sched_group_barrier(0x100, QP * NT, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 2 * QP * NT, 0);  // MFMAs
        }
        // the next tile's rows, in flight from here
        const int was0 = slot[0], was1 = slot[1];
        if (t + NW < t_end) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) slot[kt] = slot_of((t + NW) * KT + kt * 16 + lr, page[kt]);
            load_kv();
            if (t + 2 * NW < t_end)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) page[kt] = page_of((t + 2 * NW) * KT + kt * 16 + lr);
        }
        // p
        if (masked) {
            // bit k of `vis`: key k of the tile; the tile begins `ahead` positions after the first drafted one
            const int ahead = t * KT - past;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                uint32_t vis = ahead >= 64 ? 0u : ahead >= 0 ? static_cast<uint32_t>(seen[nt] >> ahead)
                             : ahead <= -KT ? ~0u : static_cast<uint32_t>(seen[nt] << -ahead) | ((1u << -ahead) - 1u);
                vis = (vis & there) >> (4 * lg);
#pragma unroll
                for (int i = 0; i < 8; ++i) sc[nt][i >> 2][i & 3] = vis >> ((i >> 2) * 16 + (i & 3)) & 1u ? sc[nt][i >> 2][i & 3] : NONE;
            }
        }
        // the reference follows where a score passes it by more than SLACK (one test for all query tiles, so
        // that what follows is one straight run of instructions)
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
        // O^T += V^T P^T
        v8 va[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const int r = kt * 16 + 4 * lg + (lr >> 2);
                const v4 x = bits<v4>(__builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4 *) (buf + r * (D * 2) + ((d ^ (r & (DT - 1))) << 5) + ((lr & 3) << 3))));
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
                if constexpr (PAIR) {
                    // hi truncated, two at once; lo is the exact rest, rounded
                    const auto hi = bits<half2_t>(__builtin_amdgcn_cvt_pkrtz(p0, p1));
                    ph[i] = hi[0];
                    ph[i + 1] = hi[1];
                    pl[i] = static_cast<E>(p0 - static_cast<float>(hi[0]));
                    pl[i + 1] = static_cast<E>(p1 - static_cast<float>(hi[1]));
                } else {
                    ph[i] = static_cast<E>(p0);
                    ph[i + 1] = static_cast<E>(p1);
                }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                acc[nt][d] = Types<E>::mfma(va[d], ph, acc[nt][d]);
                if constexpr (PAIR) acc[nt][d] = Types<E>::mfma(va[d], pl, acc[nt][d]);
            }
        }
        // Drafted keys with an infinity or NaN in V (rare): zeros in the products above, since 0 times
        // one would reach the rows that do not see them; here only the rows that do see them add theirs.
        if (special) {
            float *ps = reinterpret_cast<float *>(buf);       // [query row][key]
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 8; ++i) ps[(nt * 16 + lr) * KT + (i >> 2) * 16 + 4 * lg + (i & 3)] = sc[nt][i >> 2][i & 3];
            __builtin_amdgcn_wave_barrier();
            for (uint32_t rest = special; rest; rest &= rest - 1) {
                const int kin = __builtin_ctz(rest), ahead = t * KT + kin - past;
                const int sl = __shfl(kin < 16 ? was0 : was1, kin & 15);
                const E *vp = static_cast<const E *>(a.v) + static_cast<size_t>(max(sl, 0)) * a.ldkv + kvh * D + 4 * lg;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (!(ahead < 64 && (seen[nt] >> (ahead & 63) & 1))) continue;
                    const float p = ps[(nt * 16 + lr) * KT + kin];
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        const v4 x = bits<v4>(*(const NAVI_GLOBAL u32x2_t *) (vp + 16 * d));
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[nt][d][e] = fmaf(p, static_cast<float>(x[e]), acc[nt][d][e]);
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
    }

    // join the four waves: reference = the greatest, sums and rows scaled to it
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        sum[nt] = row_sum(sum[nt]);
        if (lg == 0) {
            s_ref[wv][nt * 16 + lr] = ref[nt];
            s_sum[wv][nt * 16 + lr] = sum[nt];
        }
    }
    __syncthreads();                                          // and every wave is done with its buffer
    float own[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 16 + lr;
        float m = s_ref[0][r];
#pragma unroll
        for (int w = 1; w < NW; ++w) m = fmaxf(m, s_ref[w][r]);
        own[nt] = ref[nt] == NONE ? 0.f : __builtin_amdgcn_exp2f(ref[nt] - m);
    }
    float *js = reinterpret_cast<float *>(sm);
    const size_t part = CUT ? part_of(a, kvh, group, unit) * (NT * 16) : 0;
#pragma unroll
    for (int cols = 0; cols < NT; ++cols) {                   // CD columns at a time
        if (cols) __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int d = 0; d < DT / NT; ++d)
                *reinterpret_cast<f32x4_t *>(js + (wv * NT * 16 + nt * 16 + lr) * CDP + d * 16 + 4 * lg) = acc[nt][cols * (DT / NT) + d] * own[nt];
        __syncthreads();
        for (int i = threadIdx.x; i < NT * 16 * (CD / 4); i += BT) {
            const int r = i / (CD / 4), c = i % (CD / 4) * 4, m = qrow0 + r, j = div_by(a.heads_per, m);
            if (j >= rows) continue;
            f32x4_t o = *reinterpret_cast<f32x4_t *>(js + r * CDP + c);
            float mx = s_ref[0][r];
#pragma unroll
            for (int w = 1; w < NW; ++w) {
                o += *reinterpret_cast<f32x4_t *>(js + (w * NT * 16 + r) * CDP + c);
                mx = fmaxf(mx, s_ref[w][r]);
            }
            float total = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) total += s_ref[w][r] == NONE ? 0.f : s_sum[w][r] * __builtin_amdgcn_exp2f(s_ref[w][r] - mx);
            const int head = kvh * a.g + m - j * a.g, col = cols * CD + c;
            if (CUT && !whole) {
                st4(a.po + (part + r) * D + col, o);
                if (col == 0) {
                    gst(a.pm + 2 * (part + r), mx);
                    gst(a.pm + 2 * (part + r) + 1, total);
                }
            } else {
                const float inv = mx == NONE ? 0.f : 1.f / total;
                store_out<E, PAIR>(a, c0 + j, head * D + col, a.hkv * a.g * D, o * inv);
            }
        }
    }
}

// Joins the parts of the requests that were cut, in their order: a wave takes a query row, D / 8 lanes its
// columns and the others further parts. Block (request x kv head x group, rows).
template <class E, bool PAIR, int D>
__global__ void __launch_bounds__(BT) k_tree_join(Args a, int nt16) {
    constexpr int CL = D / 8, PL = WAVE / CL;
    __shared__ Chunks seq;
    const int l = threadIdx.x & 63, c = l % CL, pl = l / CL;
    int id = blockIdx.x;
    const int kvh = id % a.hkv;
    id /= a.hkv;
    const int group = id % a.groups, req = id / a.groups, qrow0 = group * nt16;
    lay_out(a, qrow0, seq);
    const int k0 = seq.before[req], k1 = seq.before[req + 1];
    if (k1 - k0 < 2) return;                                      // a block had all of it and has stored it
    const Where wh = seq.at[req];
    const int left = min(nt16, wh.rows * a.g - qrow0);
    for (int r = blockIdx.y * NW + (threadIdx.x >> 6); r < left; r += gridDim.y * NW) {
        float m = NONE, sum = 0.f;
        f32x4_t o[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll 4
        for (int k = k0 + pl; k < k1; k += PL) {
            const size_t at = part_of(a, kvh, group, k) * nt16 + r;
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
            const float inv = top == NONE ? 0.f : 1.f / sum;
            store_out<E, PAIR>(a, wh.c0 + j, head * D + 8 * c, a.hkv * a.g * D, o[0] * inv);
            store_out<E, PAIR>(a, wh.c0 + j, head * D + 8 * c + 4, a.hkv * a.g * D, o[1] * inv);
        }
    }
}

// How a call is cut: query tiles of a block, groups of them, and blocks wanted for a kv head and group (0: one a request).
struct Cut {
    int nt, groups, workers;
};
Cut cut_of(const navi_kv_pages &p, const navi_kv_heads &h, int max_keys) {
    const int m = std::min(p.max_new, 64) * (h.n_head / h.n_kv_head);
    Cut c;
    c.nt = m <= 16 ? 1 : m <= 32 ? 2 : 4;
    c.groups = (m + 16 * c.nt - 1) / (16 * c.nt);
    const int64_t heads = static_cast<int64_t>(h.n_kv_head) * c.groups;
    const int steps = (max_keys + KT * NW - 1) / (KT * NW);
    // A block a request where no request can be long and there are blocks for all CUs (32 requests of 1024 keys: 30.0 us,
    // cut 33.2: the chunks and the join), or more requests than a block lays out. Else two blocks a CU, or the one that
    // fits with four query tiles.
    if (p.n_requests > MAXB || steps == 1 || (steps <= 16 && p.n_requests * heads >= 256)) {
        c.workers = 0;
        return c;
    }
    const int64_t blocks = c.nt == 4 ? 256 : 512;
    c.workers = static_cast<int>(std::max<int64_t>(1, std::min((blocks + heads - 1) / heads, static_cast<int64_t>(steps) * p.n_requests)));
    return c;
}

size_t workspace(const navi_kv_pages &p, const navi_kv_heads &h, int max_keys) {
    const Cut c = cut_of(p, h, max_keys);
    if (c.workers == 0) return 0;
    return static_cast<size_t>(h.n_kv_head) * c.groups * (c.workers + p.n_requests) * (c.nt * 16) * (h.head_dim + 2) * sizeof(float);
}

template <class E, bool PAIR, int D, int NT>
void launch_nt(const Args &a, const Cut &c, hipStream_t s) {
    if (c.workers == 0) {
        hipLaunchKernelGGL((k_tree<E, PAIR, D, NT, false>), dim3(static_cast<unsigned>(a.n) * a.groups * a.hkv), dim3(BT), 0, s, a);
        return;
    }
    hipLaunchKernelGGL((k_tree<E, PAIR, D, NT, true>), dim3(static_cast<unsigned>(c.workers + a.n) * a.groups * a.hkv), dim3(BT), 0, s, a);
    const unsigned units = static_cast<unsigned>(a.n) * a.groups * a.hkv;
    hipLaunchKernelGGL((k_tree_join<E, PAIR, D>), dim3(units, std::max(1u, std::min(NT * 16u / NW, 1024u / units))), dim3(BT), 0, s, a, NT * 16);
}

template <class E, bool PAIR, int D>
void launch_as(const Args &a, const Cut &c, hipStream_t s) {
    if (c.nt == 1) launch_nt<E, PAIR, D, 1>(a, c, s);
    else if (c.nt == 2) launch_nt<E, PAIR, D, 2>(a, c, s);
    else launch_nt<E, PAIR, D, 4>(a, c, s);
}

void launch(const Call &x, hipStream_t s) {
    const navi_kv_pages &p = *x.pages;
    const navi_kv_heads &h = *x.heads;
    const Cut c = cut_of(p, h, x.max_keys);
    Args a{};
    a.q = x.q;
    a.k = x.k;
    a.v = x.v;
    a.out = x.out;
    a.po = static_cast<float *>(x.ws);
    a.pm = a.po ? a.po + static_cast<size_t>(h.n_kv_head) * c.groups * (c.workers + p.n_requests) * (c.nt * 16) * h.head_dim : nullptr;
    a.table = p.block_table;
    a.n_past = p.n_past;
    a.cu = p.cu_rows;
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
    a.groups = c.groups;
    a.tiled = x.tiled;
    a.page = kv::make_div(static_cast<uint32_t>(p.page_size));
    a.heads_per = kv::make_div(static_cast<uint32_t>(a.g));
    a.flip = x.scale < 0.f;
    a.scale = std::fabs(x.scale) * 1.44269504088896340736f;
    const bool pair = x.q_dtype == NAVI_DT_F32, bf = h.kv_dtype == NAVI_DT_BF16;
    if (h.head_dim == 128) {
        if (pair) launch_as<_Float16, true, 128>(a, c, s);
        else if (bf) launch_as<__bf16, false, 128>(a, c, s);
        else launch_as<_Float16, false, 128>(a, c, s);
    } else {
        if (pair) launch_as<_Float16, true, 64>(a, c, s);
        else if (bf) launch_as<__bf16, false, 64>(a, c, s);
        else launch_as<_Float16, false, 64>(a, c, s);
    }
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
    if (q_dtype != heads->kv_dtype && !(q_dtype == NAVI_DT_F32 && heads->kv_dtype == NAVI_DT_F16)) {
        set_err(err, errlen, "tree_attention: unsupported types (q %d, cache %d): the cache's type, or f32 over f16", q_dtype, heads->kv_dtype);
        return NAVI_ERR_UNSUPPORTED;
    }
    if (pages->max_new > 64) {
        set_err(err, errlen, "tree_attention: up to %d rows a request; at most 64", pages->max_new);
        return NAVI_ERR_INVALID;
    }
    if (!kv::rows_ok(d_q, q_dtype, ldq, width) || !kv::rows_ok(d_out, q_dtype, ldo, width) || !d_k || !d_v || !kv::aligned16(d_k) ||
        !kv::aligned16(d_v)) {
        set_err(err, errlen, "tree_attention: a null or misaligned pointer, or a stride too small (ldq %d, ldo %d)", ldq, ldo);
        return NAVI_ERR_INVALID;
    }
    if (max_keys < 1 || max_keys > INT32_MAX - 64) {
        set_err(err, errlen, "tree_attention: max_keys %d out of range", max_keys);
        return NAVI_ERR_INVALID;
    }
    if (static_cast<int64_t>(pages->n_requests) * heads->n_head * 64 > INT32_MAX) {
        set_err(err, errlen, "tree_attention: %d requests of %d heads are too many for one call", pages->n_requests, heads->n_head);
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
    tree::launch({pages, heads, d_q, d_k, d_v, d_out, d_ws, ws_bytes, q_dtype, ldq, ld_kv, ldo, max_keys, scale, false}, static_cast<hipStream_t>(stream));
    NAVI_TRY_HIP(hipGetLastError(), err, errlen);
    return NAVI_OK;
}

} // extern "C"

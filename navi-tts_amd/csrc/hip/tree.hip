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
    float *po, *pm;                    // split: partial sums [split][row * heads + head][D], then (reference, sum) pairs
    const int32_t *table, *n_past, *cu;
    const uint64_t *mask;
    int n, hkv, g, blocks, n_pages, n_rows, max_new, ldq, ldkv, ldo, splits, tiles, groups;   // tiles: of a split
    int tiled;                         // f32 out: in the tile layout of rows.h, heads * D wide
    Div page, heads_per;               // heads_per: by g
    float scale;                       // scale * log2 e
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

// PAIR: q and out are f32, q and p travel as hi + lo pairs. NT: 16-row query tiles of a block.
template <class E, bool PAIR, int D, int NT>
__global__ void __launch_bounds__(BT) k_tree(Args a) {
    typedef typename Types<E>::v8 v8;
    typedef typename Types<E>::v4 v4;
    constexpr int KS = D / 32, DT = D / 16;                      // MFMA steps of a score, column tiles of O
    constexpr int VB = KT * D * 2 > NT * 16 * KT * 4 ? KT * D * 2 : NT * 16 * KT * 4;   // a wave's buffer, bytes
    constexpr int CD = D / NT, CDP = CD + 4;                     // columns joined at a time, padded
    constexpr int JOIN = NW * NT * 16 * CDP * 4;
    __shared__ __align__(16) unsigned char sm[NW * VB > JOIN ? NW * VB : JOIN];
    __shared__ float s_ref[NW][NT * 16], s_sum[NW][NT * 16];

    const int wv = threadIdx.x >> 6, l = threadIdx.x & 63, lr = l & 15, lg = l >> 4;
    int id = blockIdx.x;
    const int kvh = id % a.hkv;
    id /= a.hkv;
    const int group = id % a.groups;
    id /= a.groups;
    const int split = id % a.splits, req = id / a.splits;

    const int c0 = gld(a.cu + req), c1 = min(gld(a.cu + req + 1), a.n_rows);
    const int rows = min(c1 - c0, a.max_new);
    const int qrow0 = group * NT * 16;
    if (qrow0 >= rows * a.g) return;                              // uniform: this request has fewer rows
    const int64_t room = min(static_cast<int64_t>(a.blocks) * a.page.d, static_cast<int64_t>(INT32_MAX - 2 * KT));
    const int past = static_cast<int>(min<int64_t>(max(gld(a.n_past + req), 0), room));
    const int len = static_cast<int>(min<int64_t>(static_cast<int64_t>(past) + max(c1 - c0, 0), room));
    const int t_end_all = (len + KT - 1) / KT;
    const int t0 = split * a.tiles, t_end = split == a.splits - 1 ? t_end_all : min(t_end_all, t0 + a.tiles);
    if (t0 >= t_end && split > 0) return;                         // the join counts the splits as this does

    // this lane's query rows (one a tile): their operands, masks, and factor of the scores
    v8 qh[NT][KS], ql[PAIR ? NT : 1][PAIR ? KS : 1];
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
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float y = ldexpf(x[s][hf][e], -ex);
                        const E hi = static_cast<E>(y);
                        qh[nt][s][4 * hf + e] = hi;
                        ql[nt][s][4 * hf + e] = static_cast<E>(y - static_cast<float>(hi));
                    }
        } else {
            const E *q = static_cast<const E *>(a.q) + at;
#pragma unroll
            for (int s = 0; s < KS; ++s)
                qh[nt][s] = bits<v8>(on ? *(const NAVI_GLOBAL u32x4_t *) (q + 32 * s) : u32x4_t{0u, 0u, 0u, 0u});
        }
    }

    f32x4_t acc[NT][DT];
    float ref[NT], sub[NT], sum[NT];                              // ref: the reference + SLACK; sub: reference - LIFT
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
    // slot of key `key`, or -1 past the end and outside the pool
    auto slot_of = [&](int key) {
        const int b = div_by(a.page, key);
        const int p = key < len ? gld(table + b) : -1;
        return static_cast<unsigned>(p) < static_cast<unsigned>(a.n_pages) ? p * static_cast<int>(a.page.d) + key - b * static_cast<int>(a.page.d) : -1;
    };
    u32x4_t kr[2][KS], vr[2][KS];
    int slot[2];
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
        for (int kt = 0; kt < 2; ++kt) slot[kt] = slot_of(t * KT + kt * 16 + lr);
        load_kv();
    }
    for (; t < t_end; t += NW) {
        // keys of this tile that exist (uniform), and whether any row may not see one
        const uint32_t there = static_cast<uint32_t>(__ballot(slot[0] >= 0) & 0xFFFFu) | static_cast<uint32_t>(__ballot(slot[1] >= 0) & 0xFFFFu) << 16;
        const bool tree_tile = (t + 1) * KT > past, masked = tree_tile || there != 0xFFFFFFFFu;
        // V rows into LDS: 32-byte chunk i of key r at chunk i ^ (r & 7)
        uint32_t special = 0;                                     // drafted keys with an infinity or NaN in V
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
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                f32x4_t z{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    z = Types<E>::mfma(bits<v8>(kr[kt][s]), qh[nt][s], z);
                    if constexpr (PAIR) z = Types<E>::mfma(bits<v8>(kr[kt][s]), ql[nt][s], z);
                }
                sc[nt][kt] = z;
            }
        // the next tile's rows, in flight from here
        const int spec_slot0 = slot[0], spec_slot1 = slot[1];
        if (t + NW < t_end) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) slot[kt] = slot_of((t + NW) * KT + kt * 16 + lr);
            load_kv();
        }
        // p
        v8 ph[NT], pl[PAIR ? NT : 1];
        float pf[NT][8];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float top = NONE;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float x = sc[nt][i >> 2][i & 3] * fac[nt];
                if (masked) {
                    const int kin = (i >> 2) * 16 + 4 * lg + (i & 3), ahead = t * KT + kin - past;
                    const bool vis = (there >> kin & 1) && (ahead < 0 || (ahead < 64 && (seen[nt] >> (ahead & 63) & 1)));
                    x = vis ? x : NONE;
                }
                pf[nt][i] = x;
                top = fmaxf(top, x);
            }
            if (__ballot(top > ref[nt])) {
                const float mx = row_max(top);
                if (mx > ref[nt]) {
                    const float f = ref[nt] == NONE ? 0.f : __builtin_amdgcn_exp2f(ref[nt] - SLACK - mx);
                    sum[nt] *= f;
#pragma unroll
                    for (int d = 0; d < DT; ++d) acc[nt][d] *= f;
                    ref[nt] = mx + SLACK;
                    sub[nt] = mx - LIFT;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float p = __builtin_amdgcn_exp2f(pf[nt][i] - sub[nt]);
                sum[nt] += p;
                pf[nt][i] = p;
                const E hi = static_cast<E>(p);
                ph[nt][i] = hi;
                if constexpr (PAIR) pl[nt][i] = static_cast<E>(p - static_cast<float>(hi));
            }
        }
        // O^T += V^T P^T
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            v8 va;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const int r = kt * 16 + 4 * lg + (lr >> 2);
                const v4 x = bits<v4>(__builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4 *) (buf + r * (D * 2) + ((d ^ (r & (DT - 1))) << 5) + ((lr & 3) << 3))));
#pragma unroll
                for (int e = 0; e < 4; ++e) va[4 * kt + e] = x[e];
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                acc[nt][d] = Types<E>::mfma(va, ph[nt], acc[nt][d]);
                if constexpr (PAIR) acc[nt][d] = Types<E>::mfma(va, pl[nt], acc[nt][d]);
            }
        }
        // Drafted keys with an infinity or NaN in V (rare): zeros in the products above, since 0 times
        // one would reach the rows that do not see them; here only the rows that do see them add theirs.
        if (special) {
            float *ps = reinterpret_cast<float *>(buf);           // [query row][key]
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 8; ++i) ps[(nt * 16 + lr) * KT + (i >> 2) * 16 + 4 * lg + (i & 3)] = pf[nt][i];
            __builtin_amdgcn_wave_barrier();
            for (uint32_t rest = special; rest; rest &= rest - 1) {
                const int kin = __builtin_ctz(rest), ahead = t * KT + kin - past;
                const int sl = __shfl(kin < 16 ? spec_slot0 : spec_slot1, kin & 15);
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
    __syncthreads();                                              // and every wave is done with its buffer
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
#pragma unroll
    for (int part = 0; part < NT; ++part) {                       // CD columns at a time
        if (part) __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int d = 0; d < DT / NT; ++d)
                *reinterpret_cast<f32x4_t *>(js + (wv * NT * 16 + nt * 16 + lr) * CDP + d * 16 + 4 * lg) = acc[nt][part * (DT / NT) + d] * own[nt];
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
            const int head = kvh * a.g + m - j * a.g, col = part * CD + c;
            if (a.splits > 1) {
                const size_t at = (static_cast<size_t>(split) * a.n_rows + c0 + j) * (a.hkv * a.g) + head;
                st4(a.po + at * D + col, o);
                if (col == 0) {
                    gst(a.pm + 2 * at, mx);
                    gst(a.pm + 2 * at + 1, total);
                }
            } else {
                const float inv = mx == NONE ? 0.f : 1.f / total;
                store_out<E, PAIR>(a, c0 + j, head * D + col, a.hkv * a.g * D, o * inv);
            }
        }
    }
}

// Joins the splits of every row in split order: block (head and column tile, row of the request, request).
template <class E, bool PAIR, int D>
__global__ void __launch_bounds__(BT) k_tree_join(Args a) {
    const int req = blockIdx.z, j = blockIdx.y, heads = a.hkv * a.g;
    const int c0 = gld(a.cu + req), c1 = min(gld(a.cu + req + 1), a.n_rows);
    if (j >= c1 - c0) return;
    const int i = blockIdx.x * BT + threadIdx.x, head = i / (D / 4), col = i % (D / 4) * 4;
    if (head >= heads) return;
    const int64_t room = min(static_cast<int64_t>(a.blocks) * a.page.d, static_cast<int64_t>(INT32_MAX - 2 * KT));
    const int past = static_cast<int>(min<int64_t>(max(gld(a.n_past + req), 0), room));
    const int len = static_cast<int>(min<int64_t>(static_cast<int64_t>(past) + (c1 - c0), room));
    const int n = max(1, min(a.splits, ((len + KT - 1) / KT + a.tiles - 1) / a.tiles));
    const size_t step = static_cast<size_t>(a.n_rows) * heads, at = static_cast<size_t>(c0 + j) * heads + head;
    float m = NONE;
    for (int s = 0; s < n; ++s) m = fmaxf(m, gld(a.pm + 2 * (s * step + at)));
    f32x4_t o{0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
    for (int s = 0; s < n; ++s) {
        const float r = gld(a.pm + 2 * (s * step + at)), z = gld(a.pm + 2 * (s * step + at) + 1);
        const f32x4_t x = ld4(a.po + (s * step + at) * D + col);
        const float f = r == NONE ? 0.f : __builtin_amdgcn_exp2f(r - m);
        total += f * z;
        o += x * f;
    }
    store_out<E, PAIR>(a, c0 + j, head * D + col, heads * D, o * (m == NONE ? 0.f : 1.f / total));
}

// How a call is cut: query tiles of a block, groups of them, splits of the keys and 32-key tiles of a split.
struct Cut {
    int nt, groups, splits, tiles;
};
Cut cut_of(const navi_kv_pages &p, const navi_kv_heads &h, int max_keys) {
    const int m = std::min(p.max_new, 64) * (h.n_head / h.n_kv_head);
    Cut c;
    c.nt = m <= 16 ? 1 : m <= 32 ? 2 : 4;
    c.groups = (m + 16 * c.nt - 1) / (16 * c.nt);
    const int64_t units = static_cast<int64_t>(p.n_requests) * h.n_kv_head * c.groups;
    const int all = (max_keys + KT - 1) / KT;
    const int64_t want = std::max<int64_t>(1, 512 / units);
    c.tiles = std::max(NW, static_cast<int>((all + want - 1) / want + NW - 1) / NW * NW);
    c.splits = std::max(1, (all + c.tiles - 1) / c.tiles);
    return c;
}

size_t workspace(const navi_kv_pages &p, const navi_kv_heads &h, int max_keys) {
    const Cut c = cut_of(p, h, max_keys);
    if (c.splits == 1) return 0;
    return static_cast<size_t>(c.splits) * p.n_rows * h.n_head * (h.head_dim + 2) * sizeof(float);
}

template <class E, bool PAIR, int D>
void launch_as(const Args &a, const Cut &c, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.n) * c.splits * c.groups * a.hkv));
    if (c.nt == 1) hipLaunchKernelGGL((k_tree<E, PAIR, D, 1>), grid, dim3(BT), 0, s, a);
    else if (c.nt == 2) hipLaunchKernelGGL((k_tree<E, PAIR, D, 2>), grid, dim3(BT), 0, s, a);
    else hipLaunchKernelGGL((k_tree<E, PAIR, D, 4>), grid, dim3(BT), 0, s, a);
    if (c.splits > 1)
        hipLaunchKernelGGL((k_tree_join<E, PAIR, D>), dim3((a.hkv * a.g * (D / 4) + BT - 1) / BT, a.max_new, a.n), dim3(BT), 0, s, a);
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
    a.pm = a.po ? a.po + static_cast<size_t>(c.splits) * p.n_rows * h.n_head * h.head_dim : nullptr;
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
    a.splits = c.splits;
    a.tiles = c.tiles;
    a.groups = c.groups;
    a.tiled = x.tiled;
    a.page = kv::make_div(static_cast<uint32_t>(p.page_size));
    a.heads_per = kv::make_div(static_cast<uint32_t>(a.g));
    a.scale = x.scale * 1.44269504088896340736f;
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

// A pool of cache pages shared by several requests on gfx950 (the C ABI's navi_kv_*): a step's block
// tables and slots from the requests' lengths, its K and V rows into the pages, and the accepted
// drafts' rows moved into place. The attention that reads the pages is in tree.hip.
#include "dev_common.h"
#include "kv.h"

#include <algorithm>
#include <memory>
#include <new>

namespace navi_amd {
namespace kv {

navi_status check_pages(const char *who, const navi_kv_pages *p, char *err, size_t errlen) {
    if (!p || !p->block_table || !p->n_past || !p->cu_rows || (p->n_rows > 0 && (!p->row_slot || !p->row_pos || !p->row_mask))) {
        set_err(err, errlen, "%s: null argument", who);
        return NAVI_ERR_INVALID;
    }
    if (p->n_requests < 1 || p->n_requests > 65535 || p->page_size < 1 || p->n_pages < 1 || p->max_blocks < 1 || p->n_rows < 0 || p->max_new < 1 ||
        static_cast<int64_t>(p->n_pages) * p->page_size > INT32_MAX) {
        set_err(err, errlen, "%s: pages out of range (requests %d, page size %d, pages %d, blocks %d, rows %d, new rows %d)", who,
                p->n_requests, p->page_size, p->n_pages, p->max_blocks, p->n_rows, p->max_new);
        return NAVI_ERR_INVALID;
    }
    return NAVI_OK;
}

navi_status check_heads(const char *who, const navi_kv_heads *h, int ld_kv, char *err, size_t errlen) {
    if (!h) {
        set_err(err, errlen, "%s: null argument", who);
        return NAVI_ERR_INVALID;
    }
    if (h->n_head < 1 || h->n_kv_head < 1 || h->n_head > 1024 || h->n_head % h->n_kv_head != 0) {
        set_err(err, errlen, "%s: %d heads over %d kv heads", who, h->n_head, h->n_kv_head);
        return NAVI_ERR_INVALID;
    }
    if ((h->head_dim != 64 && h->head_dim != 128) || (h->kv_dtype != NAVI_DT_F16 && h->kv_dtype != NAVI_DT_BF16)) {
        set_err(err, errlen, "%s: unsupported head_dim %d or cache type %d (64 or 128; f16 or bf16)", who, h->head_dim, h->kv_dtype);
        return NAVI_ERR_UNSUPPORTED;
    }
    if (ld_kv < h->n_kv_head * h->head_dim || ld_kv % 8 != 0) {
        set_err(err, errlen, "%s: cache row stride %d for %d kv heads of %d", who, ld_kv, h->n_kv_head, h->head_dim);
        return NAVI_ERR_INVALID;
    }
    return NAVI_OK;
}

// ---- plan ------------------------------------------------------------------------------------

struct PlanArgs {
    const int32_t *n_past, *n_new, *parent, *table_in, *held_in, *free_in;
    int32_t *free_pages, *table, *held, *n_free, *status, *cu, *slot, *pos;
    uint64_t *mask;
    int4 *rec;                         // per request: what the fill reads (below)
    int n, n_pages, blocks, n_rows, max_new;
    Div page;
};
// rec = { held pages before, pages taken, stack index of the first page taken, flags }
constexpr int REC_ENDED = 1, REC_REFUSED = 2, REC_BAD = 4;

constexpr int PT = 1024, PW = PT / WAVE;   // the planning block: 16 waves

// Exclusive prefix sums of x and y over the block's threads, and their totals. red: PW pairs of LDS.
struct Two {
    int64_t x, y;
};
__device__ __forceinline__ Two block_before(Two v, Two *red, Two &total) {
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    Two s = v;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const int64_t x = __shfl_up(static_cast<long long>(s.x), o), y = __shfl_up(static_cast<long long>(s.y), o);
        if (l >= o) {
            s.x += x;
            s.y += y;
        }
    }
    __syncthreads();                                  // red's readers of the call before are done
    if (l == 63) red[w] = s;
    __syncthreads();
    Two before{0, 0};
    total = Two{0, 0};
#pragma unroll
    for (int i = 0; i < PW; ++i) {
        if (i < w) {
            before.x += red[i].x;
            before.y += red[i].y;
        }
        total.x += red[i].x;
        total.y += red[i].y;
    }
    return Two{before.x + s.x - v.x, before.y + s.y - v.y};
}

// The page of block b of a request: kept from its table, or taken from the stack (whose top part was
// filled before); -1: none.
__device__ __forceinline__ int page_at(const PlanArgs &a, int i, const int4 &r, int b) {
    if (b < r.x) return gld(a.table_in + static_cast<size_t>(i) * a.blocks + b);
    return b - r.x < r.y ? gld(a.free_pages + (r.z - (b - r.x))) : -1;
}

// Ancestors (itself included) of node `lane` as bits, by pointer jumping: after round k a node has
// the bits of its 2^k nearest, so six rounds cover 64 nodes. par < 0: nothing above. All lanes call it.
__device__ __forceinline__ uint64_t ancestors(int par) {
    const int l = threadIdx.x & 63;
    uint64_t m = uint64_t(1) << l;
#pragma unroll
    for (int k = 0; k < 6; ++k) {
        const int src = par < 0 ? l : par;
        const uint64_t um = __shfl(static_cast<unsigned long long>(m), src);
        const int up = __shfl(par, src);
        if (par >= 0) {
            m |= um;
            par = up;
        }
    }
    return m;
}

// Rows and table entries of request i from its record, part `part` of `parts` (a part: `width` threads
// from thread `t`, a multiple of a wave).
__device__ __forceinline__ void fill_request(const PlanArgs &a, int i, int part, int parts, int t, int width) {
    const int4 r = a.rec[i];
    const int c0 = gld(a.cu + i), count = gld(a.cu + i + 1) - c0;
    const int past = gld(a.n_past + i);
    const bool ended = r.w & REC_ENDED, bad = r.w & REC_BAD, none = r.w & (REC_BAD | REC_REFUSED);
    const int held = ended ? 0 : r.x + r.y;
    for (int b = part * width + t; b < a.blocks; b += parts * width) {
        // a request with lengths out of range keeps its table as it is
        const int p = bad ? gld(a.table_in + static_cast<size_t>(i) * a.blocks + b) : b < held ? page_at(a, i, r, b) : -1;
        gst(a.table + static_cast<size_t>(i) * a.blocks + b, p);
    }
    auto slot_of = [&](int j) {
        if (none) return -1;
        const int at = past + j, b = div_by(a.page, at), p = page_at(a, i, r, b);
        const bool in = static_cast<unsigned>(p) < static_cast<unsigned>(a.n_pages);
        return in ? p * static_cast<int>(a.page.d) + (at - b * static_cast<int>(a.page.d)) : -1;
    };
    if (a.parent && !bad) {                           // at most 64 rows: one wave's
        if (part == 0 && t < WAVE) {
            const int j = t;
            const uint64_t m = ancestors(j < count ? gld(a.parent + c0 + j) : -1);
            if (j < count) {
                gst(a.slot + c0 + j, slot_of(j));
                gst(a.pos + c0 + j, past + static_cast<int>(__popcll(m)) - 1);
                gst(a.mask + c0 + j, m);
            }
        }
        return;
    }
    for (int j = part * width + t; j < count; j += parts * width) {
        gst(a.slot + c0 + j, slot_of(j));
        gst(a.pos + c0 + j, bad ? 0 : past + j);
        gst(a.mask + c0 + j, bad ? uint64_t(0) : j >= 63 ? ~uint64_t(0) : (uint64_t(2) << j) - 1);
    }
}

// One block plans all requests: row offsets, the checks, the stack; FILL: the tables and rows too, a
// wave a request at a time. Thread t has requests t R .. t R + R - 1 (R = 1 up to PT requests, whose
// lengths then stay in registers); it is bound by the latencies of its rounds of loads, barriers and sums, so
// these are few: 256 requests with trees 13 us with the fill, 21 when every check read its request's record from memory.
template <bool FILL>
__global__ void __launch_bounds__(PT) k_plan(PlanArgs a) {
    __shared__ Two red[PW];
    __shared__ int s_top, s_list;
    __shared__ int4 list[PT];                         // of a round: row offset, rows, parents checked?; then the pages that go back
    __shared__ bool s_bad[PT];
    const int tid = threadIdx.x, wv = tid >> 6, l = tid & 63;
    const int R = (a.n + PT - 1) / PT, i0 = tid * R;
    const int64_t room = min(static_cast<int64_t>(a.blocks) * a.page.d, static_cast<int64_t>(INT32_MAX));
    const int free_in = gld(a.free_in);
    struct Lengths {
        int past, add, held;
    };
    auto lengths = [&](int i) {
        return i < a.n ? Lengths{gld(a.n_past + i), gld(a.n_new + i), gld(a.held_in + i)} : Lengths{0, 0, 0};
    };
    const Lengths first = lengths(i0);
    auto own = [&](int k) { return k == 0 ? first : lengths(i0 + k); };
    // rows: offsets, and which lengths are in range
    Two total, v{0, 0};
    for (int k = 0; k < R; ++k) v.x += max(own(k).add, 0);
    int64_t at = block_before(v, red, total).x;
    if (tid == 0) {
        gst(a.cu + a.n, static_cast<int>(min(total.x, static_cast<int64_t>(a.n_rows))));
        s_top = s_list = 0;
    }
    int flags0 = 0;                                   // of this thread's first request; the others' are in their records
    for (int k = 0; k < R; ++k) {
        const int i = i0 + k;
        const Lengths x = own(k);
        const int count = max(x.add, 0);
        const bool bad = x.past < 0 || x.held < 0 || x.held > a.blocks || x.add > a.max_new || at + count > a.n_rows ||
                         (x.add >= 0 && static_cast<int64_t>(x.past) + count > room);
        const int flags = (x.add < 0 ? REC_ENDED : 0) | (bad ? REC_BAD : 0);
        const int c0 = static_cast<int>(min(at, static_cast<int64_t>(a.n_rows)));
        if (i < a.n) {
            gst(a.cu + i, c0);
            gst(a.status + i, bad ? 2 : 0);
            if (k > 0) a.rec[i] = int4{x.held, 0, 0, flags};
        }
        if (k == 0) flags0 = flags;
        at += count;
        // parents come before their rows: a wave eight requests at a time, a lane a row
        if (a.parent) {
            list[tid] = int4{c0, i < a.n && flags == 0 ? count : 0, 0, 0};
            s_bad[tid] = false;
            __syncthreads();
            const int used = min(PT, (a.n - k + R - 1) / R);      // threads with a request in this round
            for (int t0 = wv * 8; t0 < used; t0 += PW * 8) {
                int p[8], n[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int4 q = t0 + u < used ? list[t0 + u] : int4{0, 0, 0, 0};
                    n[u] = q.y;
                    p[u] = l < q.y ? gld(a.parent + q.x + l) : -1;
                }
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (__ballot(p[u] < -1 || p[u] >= l) != 0 && n[u] > 0 && l == 0) s_bad[t0 + u] = true;
            }
            __syncthreads();
            if (i < a.n && s_bad[tid]) {
                gst(a.status + i, 3);
                if (k == 0) flags0 |= REC_BAD;
                else a.rec[i].w |= REC_BAD;
            }
        }
    }
    // pages that ended requests give back, and pages that the others need
    auto flags_of = [&](int k) { return k == 0 ? flags0 : a.rec[i0 + k].w; };
    auto back_and_want = [&](int k) {
        Two r{0, 0};
        if (i0 + k >= a.n) return r;
        const Lengths x = own(k);
        const int f = flags_of(k);
        if ((f & (REC_ENDED | REC_BAD)) == REC_ENDED) r.x = x.held;
        else if (!(f & (REC_ENDED | REC_BAD))) {
            const int len = x.past + max(x.add, 0);               // <= room
            r.y = max((len > 0 ? div_by(a.page, len - 1) + 1 : 0) - x.held, 0);
        }
        return r;
    };
    v = Two{0, 0};
    for (int k = 0; k < R; ++k) {
        const Two r = back_and_want(k);
        v.x += r.x;
        v.y += r.y;
    }
    Two off = block_before(v, red, total);
    const int below = min(max(free_in, 0), a.n_pages);            // the stack's top before, and with the pages given back
    const int top = static_cast<int>(min(below + total.x, static_cast<int64_t>(a.n_pages)));
    for (int k = 0; k < R; ++k) {
        const int i = i0 + k;
        const Two r = back_and_want(k);
        if (i < a.n) {
            const int held = own(k).held, f = flags_of(k);
            const bool refused = r.y > 0 && off.y + r.y > top;
            const int taken = refused ? 0 : static_cast<int>(r.y);
            if (refused) gst(a.status + i, 1);
            a.rec[i] = int4{held, taken, static_cast<int>(max<int64_t>(top - 1 - off.y, 0)), f | (refused ? REC_REFUSED : 0)};
            gst(a.held + i, (f & (REC_ENDED | REC_BAD)) == REC_ENDED ? 0 : held + taken);
            // the granted requests' pages lie without gaps below the top
            if (taken > 0) atomicMax(&s_top, static_cast<int>(off.y) + taken);
            if (r.x > 0) list[atomicAdd(&s_list, 1)] = int4{i, static_cast<int>(min(below + off.x, static_cast<int64_t>(a.n_pages))), held, 0};
        }
        off.x += r.x;
        off.y += r.y;
        if (total.x > 0) {                                        // onto the stack, a wave a request (in places that do not
            __syncthreads();                                      // depend on the list's order)
            for (int e = wv; e < s_list; e += PW) {
                const int4 q = list[e];
                for (int b = l; b < q.z && q.y + b < a.n_pages; b += WAVE)
                    gst(a.free_pages + q.y + b, gld(a.table_in + static_cast<size_t>(q.x) * a.blocks + b));
            }
            __syncthreads();
            if (tid == 0) s_list = 0;
            __syncthreads();
        }
    }
    __threadfence_block();
    __syncthreads();
    if (tid == 0) gst(a.n_free, top - s_top);
    if constexpr (FILL)
        for (int i = wv; i < a.n; i += PW) fill_request(a, i, 0, 1, l, WAVE);
}

constexpr int FT = 256;
__global__ void __launch_bounds__(FT) k_plan_fill(PlanArgs a) {
    fill_request(a, blockIdx.x, blockIdx.y, gridDim.y, threadIdx.x, FT);
}

// ---- append ----------------------------------------------------------------------------------

struct AppendArgs {
    const void *x;
    const float *qn, *kn, *rot;
    void *k, *v, *q;
    const int32_t *cu, *pos;
    int32_t *slot;
    float eps;
    int n, n_rows, n_rot, slots, hq, hk, ldx, ldkv, ldq;
    Div heads;                         // by hq + 2 hk
};

// Four consecutive elements as f32, and back with one rounding to nearest (ties to even).
template <class T>
__device__ __forceinline__ f32x4_t load4(const T *p) {
    if constexpr (sizeof(T) == 4) return ld4(reinterpret_cast<const float *>(p));
    else {
        typedef T T4 __attribute__((ext_vector_type(4)));
        const T4 t = *(const NAVI_GLOBAL T4 *) p;
        return f32x4_t{static_cast<float>(t[0]), static_cast<float>(t[1]), static_cast<float>(t[2]), static_cast<float>(t[3])};
    }
}
template <class T>
__device__ __forceinline__ void store4(T *p, f32x4_t v) {
    if constexpr (sizeof(T) == 4) st4(reinterpret_cast<float *>(p), v);
    else {
        typedef T T4 __attribute__((ext_vector_type(4)));
        *(NAVI_GLOBAL T4 *) p = T4{static_cast<T>(v[0]), static_cast<T>(v[1]), static_cast<T>(v[2]), static_cast<T>(v[3])};
    }
}

// One head of one row takes D / 8 lanes: lane c holds elements 4c .. 4c + 3 of each half, the pairs that
// the rotation mixes, so a head is read, normed, turned and written from registers. Its bytes bound it: 9009 bf16 rows
// of 16 + 2 x 8 heads of 128 (148 MB read and written) take 35.4 us, 4.2 TB/s, a large copy 4.6; one row 2.9 us.
template <class X, class Q, class E, int D>
__global__ void __launch_bounds__(256) k_append(AppendArgs a) {
    constexpr int LN = D / 8, HB = 256 / LN;
    const int c = threadIdx.x % LN, nh = a.hq + 2 * a.hk;
    const int task = blockIdx.x * HB + threadIdx.x / LN;
    const int r = div_by(a.heads, task), h = task - r * nh;
    if (r >= min(gld(a.cu + a.n), a.n_rows)) return;
    const X *x = static_cast<const X *>(a.x) + static_cast<size_t>(r) * a.ldx + h * D + 4 * c;
    f32x4_t x0 = load4(x), x1 = load4(x + D / 2);
    const int slot = gld(a.slot + r), pos = gld(a.pos + r);
    const bool in = !a.rot || static_cast<unsigned>(pos) < static_cast<unsigned>(a.n_rot);
    const bool isq = h < a.hq;
    // a row that is not stored has no slot (the row's other tasks do not use it either)
    if (!in && h == 0 && c == 0) gst(a.slot + r, -1);
    if (h < a.hq + a.hk) {
        const float *w = isq ? a.qn : a.kn;
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) ss = fmaf(x0[j], x0[j], fmaf(x1[j], x1[j], ss));
            ss += dpp_red<0xB1>(ss);
            ss += dpp_red<0x4E>(ss);
            ss += dpp_red<0x141>(ss);
            if (LN == 16) ss += dpp_red<0x140>(ss);
            const float scl = rsqrtf(ss / static_cast<float>(D) + a.eps);
            const f32x4_t w0 = ld4(w + 4 * c), w1 = ld4(w + D / 2 + 4 * c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x0[j] = x0[j] * scl * w0[j];
                x1[j] = x1[j] * scl * w1[j];
            }
        }
        if (a.rot && in) {
            const float *t = a.rot + static_cast<size_t>(pos) * D + 4 * c;
            const f32x4_t cs = ld4(t), sn = ld4(t + D / 2);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float y0 = x0[j] * cs[j] - x1[j] * sn[j], y1 = x1[j] * cs[j] + x0[j] * sn[j];
                x0[j] = y0;
                x1[j] = y1;
            }
        }
    }
    if (isq) {
        if (!in) x0 = x1 = f32x4_t{0.f, 0.f, 0.f, 0.f};
        Q *q = static_cast<Q *>(a.q) + static_cast<size_t>(r) * a.ldq + h * D + 4 * c;
        store4(q, x0);
        store4(q + D / 2, x1);
    } else if (in && static_cast<unsigned>(slot) < static_cast<unsigned>(a.slots)) {
        const bool isk = h < a.hq + a.hk;
        E *d = static_cast<E *>(isk ? a.k : a.v) + static_cast<size_t>(slot) * a.ldkv + (h - a.hq - (isk ? 0 : a.hk)) * D + 4 * c;
        store4(d, x0);
        store4(d + D / 2, x1);
    }
}

template <class X, class Q, class E>
void launch_append(const AppendArgs &a, int D, hipStream_t s) {
    const int64_t tasks = static_cast<int64_t>(a.n_rows) * (a.hq + 2 * a.hk), per = 256 / (D / 8);
    const dim3 grid(static_cast<unsigned>((tasks + per - 1) / per));
    if (D == 128) hipLaunchKernelGGL((k_append<X, Q, E, 128>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_append<X, Q, E, 64>), grid, dim3(256), 0, s, a);
}

template <class E>
void launch_append_types(const AppendArgs &a, bool xf, bool qf, int D, hipStream_t s) {
    if (xf && qf) launch_append<float, float, E>(a, D, s);
    else if (xf) launch_append<float, E, E>(a, D, s);
    else if (qf) launch_append<E, float, E>(a, D, s);
    else launch_append<E, E, E>(a, D, s);
}

// ---- commit ----------------------------------------------------------------------------------

constexpr int CL = 64;                 // arrays (a layer's K or V) a launch
struct CommitArgs {
    void *base[CL];
    const int32_t *table, *n_past, *cu, *path, *accept, *planned, *slot;   // planned: the plan's status, or null
    int32_t *past_out, *status;
    int max_path, max_new, blocks, n_pages, n_rows, ld, write;   // write: this launch stores the results
    Div page;
};

// Block (columns, request, array): each thread moves 16 bytes of a row for the whole path, in order. A
// path ascends, so its j-th source lies at or above position j: a row is read before, or when, it
// is written, and batches of eight that read before they write keep that. 32 requests' paths of 8 rows in 28 layers (44 MB)
// take 10.6 us, 4.1 TB/s; one request's 3.9 us, four rounds of memory latency (lengths; path; tables and slots; rows).
constexpr int CT = 128;
__global__ void __launch_bounds__(CT) k_commit(CommitArgs a) {
    __shared__ int src[WAVE], dst[WAVE];
    __shared__ int s_n;
    const int i = blockIdx.y, l = threadIdx.x;
    const int past = gld(a.n_past + i), c0 = gld(a.cu + i), count = gld(a.cu + i + 1) - c0, n = gld(a.accept + i);
    const int refused = a.planned ? gld(a.planned + i) : 0;
    if (l < WAVE) {
        bool bad = n < 0 || n > a.max_path || past < 0;
        int p = -1;
        if (!bad && l < n) p = gld(a.path + static_cast<size_t>(i) * a.max_path + l);
        const int prev = __shfl_up(p, 1);
        auto slot_of = [&](int node) {
            const int64_t at = static_cast<int64_t>(past) + node;
            if (at >= static_cast<int64_t>(a.blocks) * a.page.d || at > INT32_MAX) return -1;
            const int b = div_by(a.page, static_cast<int>(at)), g = gld(a.table + static_cast<size_t>(i) * a.blocks + b);
            return static_cast<unsigned>(g) < static_cast<unsigned>(a.n_pages)
                       ? g * static_cast<int>(a.page.d) + static_cast<int>(at) - b * static_cast<int>(a.page.d) : -1;
        };
        // rows that a plan refused were never appended: the request's last row has no page, or its status says so
        const int last = past >= 0 && count > 0 ? slot_of(count - 1) : -1;
        if (!bad && l < n) {
            bad = p < 0 || p >= count || (l > 0 && p <= prev) || count > a.max_new || last < 0 || refused != 0;
            if (!bad && a.planned) bad = c0 < 0 || p >= a.n_rows - c0 || gld(a.slot + c0 + p) < 0;
            if (!bad) {
                src[l] = slot_of(p);
                dst[l] = slot_of(l);
                bad = src[l] < 0 || dst[l] < 0;
            }
        }
        const bool any = __ballot(bad) != 0;
        if (l == 0) {
            s_n = any ? 0 : n;
            if (a.write && blockIdx.x == 0 && blockIdx.z == 0) {
                gst(a.past_out + i, any ? past : past + n);
                gst(a.status + i, any ? 2 : 0);
            }
        }
    }
    __syncthreads();
    const int m = s_n, col = (blockIdx.x * CT + l) * 8;
    if (col >= a.ld) return;
    uint16_t *base = static_cast<uint16_t *>(a.base[blockIdx.z]) + col;
    for (int j0 = 0; j0 < m; j0 += 8) {
        u32x4_t t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j0 + j < m && src[j0 + j] != dst[j0 + j])
                t[j] = *(const NAVI_GLOBAL u32x4_t *) (base + static_cast<size_t>(src[j0 + j]) * a.ld);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j0 + j < m && src[j0 + j] != dst[j0 + j])
                *(NAVI_GLOBAL u32x4_t *) (base + static_cast<size_t>(dst[j0 + j]) * a.ld) = t[j];
    }
}

} // namespace kv
} // namespace navi_amd

using namespace navi_amd;
using namespace navi_amd::kv;

extern "C" {

navi_status navi_kv_plan(const navi_kv_pages *pages, const int32_t *d_n_new, const int32_t *d_parent, const int32_t *d_table_in,
                         const int32_t *d_held_in, const int32_t *d_free_in, int32_t *d_free_pages, int32_t *d_held,
                         int32_t *d_free, int32_t *d_status, int32_t *d_scratch, void *stream, char *err, size_t errlen) {
    navi_status st = check_pages("kv_plan", pages, err, errlen);
    if (st != NAVI_OK) return st;
    if (!d_n_new || !d_table_in || !d_held_in || !d_free_in || !d_free_pages || !d_held || !d_free || !d_status || !d_scratch) {
        set_err(err, errlen, "kv_plan: null argument");
        return NAVI_ERR_INVALID;
    }
    if (d_parent && pages->max_new > 64) {
        set_err(err, errlen, "kv_plan: trees of up to %d rows a request; at most 64", pages->max_new);
        return NAVI_ERR_INVALID;
    }
    if (!aligned16(d_scratch)) {
        set_err(err, errlen, "kv_plan: d_scratch is not 16-byte aligned");
        return NAVI_ERR_INVALID;
    }
    OnDevice dev;
    if ((st = dev.enter(stream, "kv_plan", err, errlen)) != NAVI_OK) return st;
    const PlanArgs a{pages->n_past, d_n_new, d_parent, d_table_in, d_held_in, d_free_in, d_free_pages, pages->block_table, d_held, d_free,
                     d_status, pages->cu_rows, pages->row_slot, pages->row_pos, pages->row_mask, reinterpret_cast<int4 *>(d_scratch),
                     pages->n_requests, pages->n_pages, pages->max_blocks, pages->n_rows, pages->max_new,
                     make_div(static_cast<uint32_t>(pages->page_size))};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t words = static_cast<int64_t>(pages->n_requests) * pages->max_blocks + pages->n_rows;
    if (words <= 4096) {
        hipLaunchKernelGGL(k_plan<true>, dim3(1), dim3(PT), 0, s, a);
    } else {
        hipLaunchKernelGGL(k_plan<false>, dim3(1), dim3(PT), 0, s, a);
        const int longest = std::max(pages->max_blocks, d_parent ? 1 : std::min(pages->max_new, pages->n_rows));
        hipLaunchKernelGGL(k_plan_fill, dim3(pages->n_requests, std::min((longest + 4 * FT - 1) / (4 * FT), 256)), dim3(FT), 0, s, a);
    }
    NAVI_TRY_HIP(hipGetLastError(), err, errlen);
    return NAVI_OK;
}

navi_status navi_kv_append(const navi_kv_pages *pages, const navi_kv_heads *heads, const void *d_x, int32_t x_dtype, int32_t ldx,
                           const float *d_q_norm, const float *d_k_norm, float eps, const float *d_rot, int32_t n_rot, void *d_k,
                           void *d_v, int32_t ld_kv, void *d_q, int32_t q_dtype, int32_t ldq, void *stream, char *err,
                           size_t errlen) {
    navi_status st = check_pages("kv_append", pages, err, errlen);
    if (st == NAVI_OK) st = check_heads("kv_append", heads, ld_kv, err, errlen);
    if (st != NAVI_OK) return st;
    const int D = heads->head_dim, nh = heads->n_head + 2 * heads->n_kv_head;
    if ((x_dtype != NAVI_DT_F32 && x_dtype != heads->kv_dtype) || (q_dtype != NAVI_DT_F32 && q_dtype != heads->kv_dtype)) {
        set_err(err, errlen, "kv_append: unsupported types (x %d, q %d, cache %d)", x_dtype, q_dtype, heads->kv_dtype);
        return NAVI_ERR_UNSUPPORTED;
    }
    if (!rows_ok(d_x, pages->n_rows, x_dtype, ldx, static_cast<long>(nh) * D) || !rows_ok(d_q, pages->n_rows, q_dtype, ldq, static_cast<long>(heads->n_head) * D) ||
        !d_k || !d_v || !aligned16(d_k) || !aligned16(d_v) || !aligned16(d_q_norm) || !aligned16(d_k_norm) || !aligned16(d_rot) ||
        (d_rot && n_rot < 1)) {
        set_err(err, errlen, "kv_append: a null or misaligned pointer, or a stride too small (ldx %d, ldq %d, n_rot %d)", ldx, ldq, n_rot);
        return NAVI_ERR_INVALID;
    }
    // D / 8 threads a head, and a launch has less than 2^32
    if (static_cast<int64_t>(pages->n_rows) * nh * (D / 8) + 256 > UINT32_MAX) {
        set_err(err, errlen, "kv_append: %d rows of %d heads are too many for one call", pages->n_rows, nh);
        return NAVI_ERR_INVALID;
    }
    if (d_q && d_q == d_x && (x_dtype != q_dtype || ldx != ldq)) {
        set_err(err, errlen, "kv_append: d_q over d_x of another type or stride (x %d, %d; q %d, %d)", x_dtype, ldx, q_dtype, ldq);
        return NAVI_ERR_INVALID;
    }
    OnDevice dev;
    if ((st = dev.enter(stream, "kv_append", err, errlen)) != NAVI_OK) return st;
    if (pages->n_rows == 0) return NAVI_OK;
    const AppendArgs a{d_x, d_q_norm, d_k_norm, d_rot, d_k, d_v, d_q, pages->cu_rows, pages->row_pos, pages->row_slot, eps, pages->n_requests,
                       pages->n_rows, n_rot, pages->n_pages * pages->page_size, heads->n_head, heads->n_kv_head, ldx, ld_kv, ldq,
                       make_div(static_cast<uint32_t>(nh))};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (heads->kv_dtype == NAVI_DT_F16) launch_append_types<_Float16>(a, x_dtype == NAVI_DT_F32, q_dtype == NAVI_DT_F32, D, s);
    else launch_append_types<__bf16>(a, x_dtype == NAVI_DT_F32, q_dtype == NAVI_DT_F32, D, s);
    NAVI_TRY_HIP(hipGetLastError(), err, errlen);
    return NAVI_OK;
}

navi_status navi_kv_commit(const navi_kv_pages *pages, const navi_kv_view *kv, const int32_t *d_path, int32_t max_path,
                           const int32_t *d_accept, int32_t *d_n_past_out, int32_t *d_status, void *stream, char *err,
                           size_t errlen) {
    navi_status st = check_pages("kv_commit", pages, err, errlen);
    if (st != NAVI_OK) return st;
    if (!kv || !kv->k || !kv->v || !d_path || !d_accept || !d_n_past_out || !d_status) {
        set_err(err, errlen, "kv_commit: null argument");
        return NAVI_ERR_INVALID;
    }
    if (max_path < 1 || max_path > 64 || kv->n_layer < 1 || kv->kv_dim < 8 || kv->kv_dim % 8 != 0 ||
        static_cast<int64_t>(kv->max_pos) < static_cast<int64_t>(pages->n_pages) * pages->page_size) {
        set_err(err, errlen, "kv_commit: out of range (max_path %d, layers %d, row %d, %d cache rows for %d pages of %d)", max_path, kv->n_layer,
                kv->kv_dim, kv->max_pos, pages->n_pages, pages->page_size);
        return NAVI_ERR_INVALID;
    }
    for (int l = 0; l < kv->n_layer; ++l)
        if (!kv->k[l] || !kv->v[l] || !aligned16(kv->k[l]) || !aligned16(kv->v[l])) {
            set_err(err, errlen, "kv_commit: layer %d's cache is null or not 16-byte aligned", l);
            return NAVI_ERR_INVALID;
        }
    for (const int32_t *in : {pages->n_past, static_cast<const int32_t *>(pages->cu_rows), static_cast<const int32_t *>(pages->block_table),
                              static_cast<const int32_t *>(pages->row_slot), pages->status, d_path, d_accept})
        if (d_n_past_out == in || d_status == in || d_status == d_n_past_out) {
            set_err(err, errlen, "kv_commit: d_n_past_out and d_status are one array, or one of the inputs, which other blocks still read");
            return NAVI_ERR_INVALID;
        }
    // the arrays by address, each once; none may begin inside the one before
    const std::unique_ptr<uintptr_t[]> at(new (std::nothrow) uintptr_t[2 * static_cast<size_t>(kv->n_layer)]);
    if (!at) {
        set_err(err, errlen, "kv_commit: out of host memory");
        return NAVI_ERR_INVALID;
    }
    for (int l = 0; l < kv->n_layer; ++l) {
        at[2 * l] = reinterpret_cast<uintptr_t>(kv->k[l]);
        at[2 * l + 1] = reinterpret_cast<uintptr_t>(kv->v[l]);
    }
    std::sort(at.get(), at.get() + 2 * static_cast<size_t>(kv->n_layer));
    const int arrays = static_cast<int>(std::unique(at.get(), at.get() + 2 * static_cast<size_t>(kv->n_layer)) - at.get());
    const uint64_t bytes = static_cast<uint64_t>(pages->n_pages) * pages->page_size * 2 * kv->kv_dim;
    for (int i = 0; i + 1 < arrays; ++i)
        if (at[i + 1] - at[i] < bytes) {
            set_err(err, errlen, "kv_commit: the cache's arrays overlap (%d rows of %d elements)", pages->n_pages * pages->page_size, kv->kv_dim);
            return NAVI_ERR_INVALID;
        }
    OnDevice dev;
    if ((st = dev.enter(stream, "kv_commit", err, errlen)) != NAVI_OK) return st;
    for (int l0 = 0; l0 < arrays; l0 += CL) {
        const int n = std::min(CL, arrays - l0);
        CommitArgs a{};
        for (int l = 0; l < n; ++l) a.base[l] = reinterpret_cast<void *>(at[l0 + l]);
        a.table = pages->block_table;
        a.n_past = pages->n_past;
        a.cu = pages->cu_rows;
        a.path = d_path;
        a.accept = d_accept;
        a.planned = pages->status;
        a.slot = pages->row_slot;
        a.max_new = pages->max_new;
        a.n_rows = pages->n_rows;
        a.past_out = d_n_past_out;
        a.status = d_status;
        a.max_path = max_path;
        a.blocks = pages->max_blocks;
        a.n_pages = pages->n_pages;
        a.ld = kv->kv_dim;
        a.write = l0 == 0;
        a.page = make_div(static_cast<uint32_t>(pages->page_size));
        hipLaunchKernelGGL(k_commit, dim3((kv->kv_dim / 8 + CT - 1) / CT, pages->n_requests, n), dim3(CT), 0,
                           static_cast<hipStream_t>(stream), a);
    }
    NAVI_TRY_HIP(hipGetLastError(), err, errlen);
    return NAVI_OK;
}

} // extern "C"

// What the operators on a paged K/V cache (kv.hip, tree.hip) share: the checks of their arguments, the
// scope in which they run on the library's device, and the arithmetic of pages.
#pragma once

#include "host_util.h"

#include <hip/hip_runtime.h>

#include <cstdint>

namespace navi_amd {
namespace kv {

// n / d for 0 <= n < 2^31 as a multiplication (Granlund and Montgomery's round-up method): with
// l = ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1, n / d = (mulhi(m, n) + n) >> l; the sum stays
// below 2^32 since mulhi(m, n) <= n.
struct Div {
    uint32_t m, l, d;
};
inline Div make_div(uint32_t d) {
    uint32_t l = 0;
    while (l < 31 && (1u << l) < d) ++l;
    return {static_cast<uint32_t>((((uint64_t(1) << l) - d) << 32) / d + 1), l, d};
}
__device__ __forceinline__ int div_by(const Div &v, int n) {
    return static_cast<int>((__umulhi(v.m, static_cast<uint32_t>(n)) + static_cast<uint32_t>(n)) >> v.l);
}

// The library's device as the thread's current one for as long as it lives, then the one before it.
struct OnDevice {
    int before = -1;
    navi_status enter(void *stream, const char *who, char *err, size_t errlen) {
        int cur = -1;
        if (hipGetDevice(&cur) != hipSuccess) cur = -1;
        const navi_status st = ensure_device(err, errlen);
        if (cur >= 0 && cur != device_state().device) before = cur;
        if (st != NAVI_OK) return st;
        // the handles 0, 1 and 2 name the current device's default streams
        if (reinterpret_cast<uintptr_t>(stream) > 2 && stream != static_cast<void *>(device_state().stream)) {
            hipDevice_t dev = -1;
            NAVI_TRY_HIP(hipStreamGetDevice(static_cast<hipStream_t>(stream), &dev), err, errlen);
            if (dev != device_state().device) {
                set_err(err, errlen, "%s: the stream is of device %d, the library runs on device %d", who, static_cast<int>(dev),
                        device_state().device);
                return NAVI_ERR_INVALID;
            }
        }
        return NAVI_OK;
    }
    ~OnDevice() {
        if (before >= 0) (void) hipSetDevice(before);
    }
};

// The fields every operator reads (the plan writes the arrays, the others read them).
navi_status check_pages(const char *who, const navi_kv_pages *p, char *err, size_t errlen);
navi_status check_heads(const char *who, const navi_kv_heads *h, int ld_kv, char *err, size_t errlen);
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// `rows` rows (of none: p may be null) of `type` elements with stride ld >= width start on 16 bytes.
inline bool rows_ok(const void *p, int rows, int type, int ld, long width) {
    return (p || rows == 0) && aligned16(p) && ld >= width && ld % (type == NAVI_DT_F32 ? 4 : 8) == 0;
}

} // namespace kv
} // namespace navi_amd

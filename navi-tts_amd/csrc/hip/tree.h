// The attention of drafted rows over a paged cache (tree.hip) as a host launcher: navi_tree_attention and
// the talker's verification (prefill.hip) run it.
#pragma once

#include "kv.h"

namespace navi_amd {
namespace tree {

struct Call {
    const navi_kv_pages *pages;
    const navi_kv_heads *heads;
    const void *q, *k, *v;
    void *out, *ws;
    int q_dtype, ldq, ldkv, ldo, max_keys;
    float scale;
    bool tiled;                        // f32 out in the tile layout of rows.h (ldo unused)
    bool slots;                        // rows without a slot (a request that the plan refused) see nothing; their output is zeros, or left as it was
};
size_t workspace(const navi_kv_pages &pages, const navi_kv_heads &heads, int max_keys);
void launch(const Call &c, hipStream_t s);   // arguments already checked

} // namespace tree
} // namespace navi_amd

// Arguments of the paged-cache kernels (pages_kernels.h, included by pages.hip only).
#pragma once

#include "kernels.h"
#include "pages_host.h"

namespace fl {

// The pool: K [layer][page][kv head][slot][D], V [layer][page][kv head][slot / 32][D][32]
// (f32, binary16, or int8 codes with a binary16 scale per 32 channels, [layer][page]
// [kv head][slot][D / 32] for each).  A (page, kv head) of either begins at the same
// element: ((layer * pages + page) * nkv + head) * P * D.
struct PagePool {
    void *k, *v;
    uint16_t *ks, *vs;  // Q8
    int layers, pages, P, nkv;
    int per;               // blocks (32 slots) of a page
    uint32_t per_inv;      // floor(x / per) = x * per_inv >> 32 for blocks x of a sequence
};

struct PageAttnArgs {
    PagePool pool;
    int layer, group;
    float scale;           // log2(e) / sqrt(D)
    const float *q;        // query i, head h at i * q_stride + h * D
    long long q_stride;
    const PageItem *items;
    const PageQuery *order;
    const int *page_ids;
    float *part, *ml;      // partial results [unit][head][D], [unit][head][2] = (max, sum)
    float *out;            // [n][heads * D]
    // where the last workgroup to have a part of a query's result joins them (otherwise
    // arrived is nullptr, and k_pages_join does):
    int *arrived;          // [join][kv head], zeros between calls
    const PageJoin *joins;
    const int *units, *join_of;  // join of a query
    int njoins, nempty;    // the last nempty of them have no parts
};

// Waves per SIMD, so workgroups of 4 waves per CU, that the attention kernel's registers
// allow (without a bound the compiler takes accumulation registers as well, and half of
// them).  forms: 1 (up to 16 rows) or 2 (up to 32; f32 of D = 128 with two waves and
// its queries in LDS 66 us against 55 for 8 queries of 32768 tokens, 8 bits 31 against 33).
constexpr int page_waves(int fmt, int D, int forms) {
    return forms == 1 ? (D == 64 ? 4 : fmt == FL_KV_F16 ? 3 : 2) : fmt == FL_KV_Q8 ? (D == 64 ? 3 : 2) : D == 64 ? 2 : 1;
}

struct PageJoinArgs {
    const PageJoin *joins;
    const int *units;
    const float *part, *ml;
    float *out;
    int heads;
};

// Short lists go with the launch (a copy to the device costs the host 5 us and the
// stream 3); longer ones are in device memory.
constexpr int kInlineRuns = 128, kInlineCopies = 96;
struct PageRuns {
    const PageRun *list;   // nullptr: `some`
    PageRun some[kInlineRuns];
};
struct PageCopies {
    const PageCopy *list;  // nullptr: `some`
    PageCopy some[kInlineCopies];
};

struct PageWriteArgs {
    PagePool pool;
    const float *k, *v;    // token i, kv head h at (layer * n + i) * stride + h * D
    long long stride;
    int layer0, n;
};

struct PageReadArgs {
    PagePool pool;
    float *k, *v;          // [n][nkv * D]
    int layer;
};

}  // namespace fl

// Host side of the paged KV cache: which sequence holds which page, and the
// plan of an attention call.  Plain C++ without a device.
#pragma once

#include <cstdint>
#include <string>
#include <vector>

#include "../../include/flare_hip.h"

namespace fl {

constexpr int kPageBlock = 32;  // slots of a block: the unit of copies and of the attention's tiles

// Copy the first `blocks` 32-slot blocks of page src to page dst, in every layer.
struct PageCopy {
    int src, dst, blocks;
};

// Consecutive tokens in one 32-slot block: tokens token .. token + count - 1 of a call in
// slots slot .. of block page * (page_size / 32) + i.
struct PageRun {
    int block, token;
    short slot, count;
};

// Pages, their reference counts and the sequences' page lists.  Every call
// checks its arguments before it changes anything: a call that fails leaves the
// state as it was.
struct PageTable {
    int pages = 0, page_size = 0, seqs = 0, max_len = 0, max_pages = 0;
    int free_pages = 0;
    std::vector<int> table;  // [seqs][max_pages], -1 where a sequence holds none
    std::vector<int> len;    // tokens of each sequence
    std::vector<int> ref;    // sequences that hold a page
    std::vector<PageCopy> copies;  // of the last call
    std::vector<PageRun> runs;     // where the last extend's tokens go
    int tokens = 0;                // how many
    bool runs_valid = false;       // no other call since
    uint64_t version = 1;          // changes with the tables and lengths
    std::string error;

    int init(const fl_pages_config &c);
    int fork(const int32_t *src, const int32_t *dst, const int32_t *lens, int n);
    int copy(const int32_t *src, const int32_t *dst, int n);
    int release(const int32_t *s, int n);
    int truncate(const int32_t *s, const int32_t *lens, int n);
    int extend(const int32_t *s, const int32_t *counts, int n);
    int compact();

    // appends the runs of tokens [from, to) of a sequence, as tokens `token` .. of a call
    void add_runs(int s, int from, int to, int token, std::vector<PageRun> &out) const;
    int held(int s) const { return (len[s] + page_size - 1) / page_size; }
    int *row(int s) { return table.data() + (size_t)s * max_pages; }
    const int *row(int s) const { return table.data() + (size_t)s * max_pages; }

private:
    std::vector<uint64_t> free_bits;
    int hint = 0;            // no free page below 64 * hint
    std::vector<uint64_t> stamp;  // the last call that listed a sequence
    uint64_t stamp_now = 0;
    int take();
    void drop(int page);
    int fail(int code, const char *fmt, ...) __attribute__((format(printf, 3, 4)));
    int check_seqs(const int32_t *s, int n, bool once);
    int blocks_of(int s, int i) const;
};

// One workgroup's part of an attention call, per kv head: queries order[q0 ..
// q0 + nq) over tokens [slot0, slot1) of the sequences that share the pages
// page_ids[page0 ..) there (the page of slot0 first).
struct PageItem {
    int q0, nq, slot0, slot1, page0;
    int unit;  // partial result of the first query; -1: the item is all that its queries see
    int smin;  // fewest tokens that one of the queries sees
    int form;  // by its rows (query x head of a kv head), see PageForms
};

// A query in an item's order: its number, and how many tokens it sees.
struct PageQuery {
    int query, seen;
};

// A query whose result is joined from the partial results units[first .. first
// + count); of none: zeros.
struct PageJoin {
    int query, first, count, pad;
};

// The forms of items that a cache's kernels have, and what the cuts of long items go by.
// A launch without an item of a form above 0 has workgroups of 4 waves, `fill` of them at
// once on the chip; another has workgroups that take `wide_step` blocks at a time, `wide_slots` at
// once on the chip, each for `fixed` and wide_cost a 32-token block, in units of a block
// of the first form.
struct PageForms {
    int n, rows[3];
    int fill;
    float wide_cost[3], fixed;
    int wide_step, wide_slots;
};

struct PagePlan {
    std::vector<PageItem> items;  // longest first
    bool wide = false;            // an item of a form above 0
    std::vector<PageQuery> order;
    std::vector<int> page_ids, units;
    std::vector<PageJoin> joins;  // those without partial results last
    std::vector<int> join_of;     // of each query (-1: none)
    int num_units = 0, empty = 0; // joins without partial results
    int most_parts = 0, most_queries = 0;  // of a join; of an item with partial results
};

// seen[i] tokens of sequence s[i] for query i (checked against the table).
// group: query heads per kv head.  0, or a code and table.error.
int page_plan(PageTable &t, const int32_t *s, const int32_t *seen, int n, int group, int kv_heads, int head_dim,
              const PageForms &forms, PagePlan &p);

}  // namespace fl

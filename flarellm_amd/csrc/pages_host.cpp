// Page bookkeeping and attention plans of the paged KV cache (pages_host.h).
#include "pages_host.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <functional>
#include <numeric>

namespace fl {

namespace {
int ceil_div(int a, int b) { return (int)(((long long)a + b - 1) / b); }
constexpr size_t kMaxOrder = 1 << 26;  // a query once per run that it sees: 0.5 GB, and counts of parts stay in 32 bits
}  // namespace

int PageTable::fail(int code, const char *fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    error = buf;
    return code;
}

int PageTable::init(const fl_pages_config &c) {
    pages = c.num_pages;
    page_size = c.page_size;
    seqs = c.max_seqs;
    max_len = c.max_seq_len;
    max_pages = ceil_div(max_len, page_size);
    free_pages = pages;
    table.assign((size_t)seqs * max_pages, -1);
    len.assign(seqs, 0);
    ref.assign(pages, 0);
    stamp.assign(seqs, 0);
    free_bits.assign((pages + 63) / 64, ~0ull);
    if (pages % 64) free_bits.back() = (1ull << (pages % 64)) - 1;
    return 0;
}

// The free page of lowest index (the caller has counted that there is one).
int PageTable::take() {
    while (!free_bits[hint]) hint++;
    const int g = 64 * hint + __builtin_ctzll(free_bits[hint]);
    free_bits[hint] &= free_bits[hint] - 1;
    free_pages--;
    ref[g] = 1;
    return g;
}

void PageTable::drop(int g) {
    if (--ref[g]) return;
    free_bits[g / 64] |= 1ull << (g % 64);
    hint = std::min(hint, g / 64);
    free_pages++;
}

int PageTable::check_seqs(const int32_t *s, int n, bool once) {
    if (n < 0 || (n > 0 && !s)) return fail(FL_E_INVALID, "bad sequence list");
    stamp_now++;
    for (int i = 0; i < n; i++) {
        if (s[i] < 0 || s[i] >= seqs) return fail(FL_E_INVALID, "sequence %d of %d", s[i], seqs);
        if (once && stamp[s[i]] == stamp_now) return fail(FL_E_INVALID, "sequence %d is listed twice", s[i]);
        stamp[s[i]] = stamp_now;
    }
    return 0;
}

// 32-slot blocks in use of the i-th page of sequence s.
int PageTable::blocks_of(int s, int i) const {
    return ceil_div(std::min(page_size, len[s] - i * page_size), kPageBlock);
}

void PageTable::add_runs(int s, int from, int to, int token, std::vector<PageRun> &out) const {
    const int *r = row(s);
    while (from < to) {
        const int slot = from % kPageBlock, n = std::min(kPageBlock - slot, to - from);
        out.push_back({(r[from / page_size] * page_size + from % page_size) / kPageBlock, token, (short)slot, (short)n});
        from += n;
        token += n;
    }
}

int PageTable::fork(const int32_t *src, const int32_t *dst, const int32_t *lens, int n) {
    if (int rc = check_seqs(src, n, false)) return rc;
    if (int rc = check_seqs(dst, n, true)) return rc;
    for (int i = 0; i < n; i++) {
        if (len[dst[i]]) return fail(FL_E_STATE, "sequence %d is not empty", dst[i]);
        if (stamp[src[i]] == stamp_now) return fail(FL_E_INVALID, "sequence %d is both source and target", src[i]);
        if (lens && (lens[i] < 0 || lens[i] > len[src[i]]))
            return fail(FL_E_INVALID, "%d of the %d tokens of sequence %d", lens[i], len[src[i]], src[i]);
    }
    copies.clear();
    for (int i = 0; i < n; i++) {
        len[dst[i]] = lens ? lens[i] : len[src[i]];
        const int m = held(dst[i]), *from = row(src[i]);
        std::copy(from, from + m, row(dst[i]));
        for (int j = 0; j < m; j++) ref[from[j]]++;
    }
    runs_valid = false;
    version++;
    return 0;
}

int PageTable::copy(const int32_t *src, const int32_t *dst, int n) {
    if (int rc = check_seqs(src, n, false)) return rc;
    if (int rc = check_seqs(dst, n, true)) return rc;
    long long need = 0;
    for (int i = 0; i < n; i++) {
        if (len[dst[i]]) return fail(FL_E_STATE, "sequence %d is not empty", dst[i]);
        if (stamp[src[i]] == stamp_now) return fail(FL_E_INVALID, "sequence %d is both source and target", src[i]);
        need += held(src[i]);
    }
    if (need > free_pages) return fail(FL_E_OOM, "%lld pages needed, %d free", need, free_pages);
    copies.clear();
    copies.reserve(need);
    for (int i = 0; i < n; i++) {
        const int m = held(src[i]);
        len[dst[i]] = len[src[i]];
        for (int j = 0; j < m; j++) {
            const int g = row(dst[i])[j] = take();
            copies.push_back({row(src[i])[j], g, blocks_of(src[i], j)});
        }
    }
    runs_valid = false;
    version++;
    return 0;
}

int PageTable::release(const int32_t *s, int n) {
    if (int rc = check_seqs(s, n, false)) return rc;
    copies.clear();
    for (int i = 0; i < n; i++) {
        int *r = row(s[i]);
        for (int j = 0, m = held(s[i]); j < m; j++) {
            drop(r[j]);
            r[j] = -1;
        }
        len[s[i]] = 0;
    }
    runs_valid = false;
    version++;
    return 0;
}

int PageTable::truncate(const int32_t *s, const int32_t *lens, int n) {
    if (int rc = check_seqs(s, n, true)) return rc;
    if (n > 0 && !lens) return fail(FL_E_INVALID, "no lengths");
    for (int i = 0; i < n; i++)
        if (lens[i] < 0 || lens[i] > len[s[i]])
            return fail(FL_E_INVALID, "%d of the %d tokens of sequence %d", lens[i], len[s[i]], s[i]);
    copies.clear();
    for (int i = 0; i < n; i++) {
        int *r = row(s[i]);
        const int m = held(s[i]);
        len[s[i]] = lens[i];
        for (int j = held(s[i]); j < m; j++) {
            drop(r[j]);
            r[j] = -1;
        }
    }
    runs_valid = false;
    version++;
    return 0;
}

int PageTable::extend(const int32_t *s, const int32_t *counts, int n) {
    if (int rc = check_seqs(s, n, true)) return rc;
    if (n > 0 && !counts) return fail(FL_E_INVALID, "no counts");
    long long tokens = 0, need = 0;
    for (int i = 0; i < n; i++) {
        if (counts[i] < 0) return fail(FL_E_INVALID, "%d new tokens", counts[i]);
        if (counts[i] > max_len - len[s[i]])
            return fail(FL_E_INVALID, "sequence %d of %d tokens cannot take %d more: at most %d", s[i], len[s[i]],
                        counts[i], max_len);
        tokens += counts[i];
    }
    // A last page that others hold too is left to them.  Where several of the
    // call's sequences share one, all but the last of those that hold it take a copy.
    std::vector<int> left;  // pages that the call has left, once per sequence
    for (int i = 0; i < n; i++) {
        need += ceil_div(len[s[i]] + counts[i], page_size) - held(s[i]);
        if (!counts[i] || len[s[i]] % page_size == 0) continue;
        left.push_back(row(s[i])[held(s[i]) - 1]);
    }
    std::sort(left.begin(), left.end());
    for (size_t i = 0; i < left.size();) {
        size_t j = i;
        while (j < left.size() && left[j] == left[i]) j++;
        need += std::min<long long>(j - i, ref[left[i]] - 1);
        i = j;
    }
    if (need > free_pages) return fail(FL_E_OOM, "%lld pages needed, %d free", need, free_pages);
    size_t most = 0;
    for (int i = 0; i < n; i++) most += counts[i] / kPageBlock + 2;
    std::vector<PageRun> out;
    out.reserve(most);
    copies.clear();
    copies.reserve(left.size());
    runs.swap(out);
    this->tokens = 0;
    for (int i = 0; i < n; i++) {
        int *r = row(s[i]);
        const int at = len[s[i]];
        const int last = held(s[i]) - 1;
        if (counts[i] && at % page_size && ref[r[last]] > 1) {
            const int g = take();
            copies.push_back({r[last], g, blocks_of(s[i], last)});
            ref[r[last]]--;
            r[last] = g;
        }
        len[s[i]] += counts[i];
        for (int j = last + 1; j < held(s[i]); j++) r[j] = take();
        add_runs(s[i], at, len[s[i]], this->tokens, runs);
        this->tokens += counts[i];
    }
    runs_valid = true;
    version++;
    return 0;
}

int PageTable::compact() {
    const int used = pages - free_pages;
    // pages at or above `used` in use, and free ones below: equally many
    std::vector<int> to(pages, -1), fill(pages, 0);
    std::vector<PageCopy> moves;
    for (int g = used, d = 0; g < pages; g++) {
        if (!ref[g]) continue;
        while (ref[d]) d++;
        to[g] = d;
        moves.push_back({g, d++, 0});
    }
    for (int s = 0; s < seqs; s++)
        for (int j = 0, m = held(s); j < m; j++) fill[row(s)[j]] = std::max(fill[row(s)[j]], blocks_of(s, j));
    copies.clear();
    runs_valid = false;
    if (moves.empty()) return 0;
    for (PageCopy &c : moves) {
        c.blocks = fill[c.src];
        std::swap(ref[c.src], ref[c.dst]);
        free_bits[c.src / 64] |= 1ull << (c.src % 64);
        free_bits[c.dst / 64] &= ~(1ull << (c.dst % 64));
    }
    copies.swap(moves);
    hint = used / 64 < (int)free_bits.size() ? used / 64 : 0;
    for (int s = 0; s < seqs; s++)
        for (int j = 0, m = held(s); j < m; j++)
            if (to[row(s)[j]] >= 0) row(s)[j] = to[row(s)[j]];
    version++;
    return 0;
}

// ---------------------------------------------------------------------------
// Attention plan.  The sequences of the call are sorted by their page lists, so
// those that share leading pages are neighbours.  A run is a range of pages that
// the same sequences hold, as long as it can be: it ends where two of them
// differ, not where one of them ends (its queries are masked there).  So each page
// is in one run per set of sequences that hold it, and is read once for all of
// them.  A run's queries, longest first, are cut into tiles by the rows (query x head of a
// kv head) that a form takes, and its tokens into parts.
// ---------------------------------------------------------------------------
int page_plan(PageTable &t, const int32_t *s, const int32_t *seen, int n, int group, int kv_heads,
              int head_dim, const PageForms &forms, PagePlan &p) {
    auto fail = [&](int code, const std::string &m) {
        t.error = m;
        return code;
    };
    if (n < 0 || (n > 0 && (!s || !seen))) return fail(FL_E_INVALID, "bad query list");
    for (int i = 0; i < n; i++) {
        if (s[i] < 0 || s[i] >= t.seqs)
            return fail(FL_E_INVALID, "query " + std::to_string(i) + ": sequence " + std::to_string(s[i]));
        if (seen[i] < 0 || seen[i] > t.len[s[i]])
            return fail(FL_E_INVALID, "query " + std::to_string(i) + " sees " + std::to_string(seen[i]) + " of " +
                                          std::to_string(t.len[s[i]]) + " tokens");
    }
    p.items.clear();
    p.order.clear();
    p.page_ids.clear();
    p.units.clear();
    p.joins.clear();
    p.num_units = p.most_queries = 0;
    const int P = t.page_size;

    // the call's sequences, each with its queries (longest first) and pages in view
    struct Seq {
        const int *pages;
        int held;         // pages that its longest query sees
        int first, count; // queries
    };
    std::vector<int> by(n);
    std::iota(by.begin(), by.end(), 0);
    std::stable_sort(by.begin(), by.end(), [&](int a, int b) { return s[a] != s[b] ? s[a] < s[b] : seen[a] > seen[b]; });
    std::vector<Seq> seqs;
    for (int i = 0; i < n; i++) {
        if (i && s[by[i]] == s[by[i - 1]]) {
            seqs.back().count++;
        } else {
            seqs.push_back({t.row(s[by[i]]), ceil_div(seen[by[i]], P), i, 1});
        }
    }
    struct Run {
        int lo, hi, p0, p1;  // sequences, pages
    };
    struct Tile {
        int q0, nq, slot0, slot1, page0, form;
    };
    std::vector<Run> todo;
    std::vector<Tile> tiles;
    const int most = std::max(1, forms.rows[forms.n - 1] / group);  // queries of the largest tile
    auto add_tile = [&](int q0, int nq, int from, int end, int page0) {
        int form = 0;
        while (forms.rows[form] < nq * group) form++;
        tiles.push_back({q0, nq, from, std::min(p.order[q0].seen, end), page0, form});
    };
    // A sequence with enough queries for the largest tile: full tiles of its own, over all
    // that they see (they gain nothing from others' queries, and need no joining).
    for (Seq &x : seqs) {
        const int full = x.count / most;
        if (!full || !seen[by[x.first]]) continue;
        const int page0 = (int)p.page_ids.size();
        p.page_ids.insert(p.page_ids.end(), x.pages, x.pages + x.held);
        for (int i = 0; i < full && seen[by[x.first]]; i++) {
            const int q0 = (int)p.order.size();
            for (int j = 0; j < most && seen[by[x.first]]; j++, x.first++, x.count--)
                p.order.push_back({by[x.first], seen[by[x.first]]});
            add_tile(q0, (int)p.order.size() - q0, 0, t.max_len, page0);
            if (!x.count) break;
        }
        x.held = x.count ? ceil_div(seen[by[x.first]], P) : 0;
    }
    // the others: a list that ends is behind those that go on
    std::sort(seqs.begin(), seqs.end(), [](const Seq &a, const Seq &b) {
        const int m = std::min(a.held, b.held);
        const int k = (int)(std::mismatch(a.pages, a.pages + m, b.pages).first - a.pages);
        if (k < m) return a.pages[k] < b.pages[k];
        return a.held != b.held ? a.held > b.held : a.first < b.first;
    });
    todo.push_back({0, (int)seqs.size(), 0, 0});
    while (!todo.empty()) {
        Run r = todo.back();
        todo.pop_back();
        int lo = r.lo, hi = r.hi, e = r.p0;
        for (;;) {
            while (hi > lo && seqs[hi - 1].held <= e) hi--;  // those that have ended
            if (lo == hi) break;
            const Seq &a = seqs[lo], &b = seqs[hi - 1];
            const int m = std::min(a.held, b.held);
            const int k = (int)(std::mismatch(a.pages + e, a.pages + m, b.pages + e).first - a.pages);
            if (k == e) break;  // they differ here
            e = k;
        }
        // [lo, hi): go on behind the run, by their next page
        for (int i = lo; i < hi;) {
            int j = i;
            while (j < hi && seqs[j].pages[e] == seqs[i].pages[e]) j++;
            todo.push_back({i, j, e, 0});
            i = j;
        }
        if (e == r.p0) continue;
        const int from = r.p0 * P, first = (int)p.order.size();
        for (int i = r.lo; i < r.hi; i++)
            for (int j = 0; j < seqs[i].count; j++) {
                const int q = by[seqs[i].first + j];
                if (seen[q] <= from) break;
                p.order.push_back({q, seen[q]});
            }
        if (p.order.size() > kMaxOrder) return fail(FL_E_INVALID, "too many queries of too many shared lists at once");
        const int end = e * P, total = (int)p.order.size() - first;
        std::stable_sort(p.order.begin() + first, p.order.end(), [&](const PageQuery &a, const PageQuery &b) {
            return std::min(a.seen, end) > std::min(b.seen, end);
        });
        const int page0 = (int)p.page_ids.size();
        for (int i = r.p0; i < e; i++) p.page_ids.push_back(seqs[r.lo].pages[i]);
        for (int i = 0; i < total; i += most) add_tile(first + i, std::min(most, total - i), from, end, page0);
    }

    // Long tiles are cut, in whole steps of the workgroup's waves.
    p.wide = false;
    long long blocks = 0;
    int longest[2] = {1, 1};  // of the forms that the memory bounds, of the largest
    for (const Tile &x : tiles) {
        const int nb = ceil_div(x.slot1 - x.slot0, kPageBlock);
        p.wide = p.wide || x.form > 0;
        blocks += nb;
        longest[x.form > 1] = std::max(longest[x.form > 1], nb);
    }
    const float *cost = forms.wide_cost;
    const int step = p.wide ? forms.wide_step : 4, least = 8;  // blocks of a step, of a part
    auto whole = [&](long long x) { return (int)((std::max<long long>(x, least) + step - 1) / step * step); };
    // blocks of a part, of nb in parts of up to `part`
    auto cut = [&](int nb, int part) { return (ceil_div(nb, ceil_div(nb, part)) + step - 1) / step * step; };
    int part[2] = {longest[0], longest[1]};
    if (!p.wide) {
        // The memory bounds all of them, and a few workgroups a CU keep it busy.
        // As many as it takes at once where that does for all, or else twice as many: 32768
        // tokens alone 28.6 us in 512 workgroups and 35.9 in 1024, 16 sequences of 40 to 7800
        // tokens 46.8 and 43.6.
        for (int f = 1; f <= 2; f++) {
            part[0] = whole((blocks * kv_heads + f * forms.fill - 1) / (f * forms.fill));
            long long n = 0;
            for (const Tile &x : tiles) n += ceil_div(ceil_div(x.slot1 - x.slot0, kPageBlock), part[0]);
            if (n * kv_heads <= forms.fill) break;
        }
    } else {
        // Of a few lengths of the parts, those whose workgroups, handed out longest first, are done earliest.
        const int machines = std::max(1, forms.wide_slots / kv_heads);
        // joining: a launch and its traffic, in blocks (0.7 us for 16 KB a CU)
        const double even = (double)blocks / machines, join = 6, unit = 8.0 * kv_heads * group * head_dim / 3.5e6;
        static const double kOf[] = {0, 1, 0.9, 0.8, 0.67, 0.5, 0.34, 0.25, 0.12, 0.06};
        constexpr int kSome = sizeof kOf / sizeof *kOf;
        double best = 0;
        std::vector<std::pair<float, int>> jobs;  // (time, how many)
        std::vector<float> heap;
        auto of = [&](int i) { return whole((long long)(even * kOf[i])); };
        auto again = [&](int i) { return i > 1 && of(i) == of(i - 1); };
        for (int i = 0; i < kSome; i++)
            for (int j = 0; j < kSome; j++) {
                if (again(i) || again(j)) continue;
                const int len[2] = {i ? of(i) : longest[0], j ? of(j) : longest[1]};
                if ((i && len[0] >= longest[0]) || (j && len[1] >= longest[1])) continue;
                jobs.clear();
                double units = 0, sum = 0;
                for (const Tile &x : tiles) {
                    const int nb = ceil_div(x.slot1 - x.slot0, kPageBlock), each = cut(nb, len[x.form > 1]), cuts = ceil_div(nb, each);
                    jobs.push_back({std::min(each, nb) * cost[x.form] + forms.fixed, cuts});
                    sum += (double)jobs.back().first * cuts;
                    if (cuts > 1) units += (double)cuts * x.nq;
                }
                const double behind = units > 0 ? join + units * unit : 0;
                if ((i || j) && sum / machines + behind >= best) continue;
                std::sort(jobs.begin(), jobs.end(), std::greater<>());
                heap.assign(machines, 0.0f);  // a min-heap of when each machine is free
                for (auto &w : jobs)
                    for (int k = 0; k < w.second; k++) {
                        std::pop_heap(heap.begin(), heap.end(), std::greater<>());
                        heap.back() += w.first;
                        std::push_heap(heap.begin(), heap.end(), std::greater<>());
                    }
                const double time = *std::max_element(heap.begin(), heap.end()) + behind;
                if ((i || j) && time >= best) continue;
                best = time;
                part[0] = len[0];
                part[1] = len[1];
            }
    }
    std::vector<int> count(n, 0);
    for (const Tile &x : tiles) {
        const int nb = ceil_div(x.slot1 - x.slot0, kPageBlock), each = cut(nb, part[x.form > 1]);
        for (int b = 0; b < nb; b += each) {
            PageItem it{};
            it.q0 = x.q0;
            it.slot0 = x.slot0 + b * kPageBlock;
            it.slot1 = std::min(x.slot1, it.slot0 + each * kPageBlock);
            it.page0 = x.page0 + it.slot0 / P - x.slot0 / P;
            it.form = x.form;
            while (it.nq < x.nq && p.order[x.q0 + it.nq].seen > it.slot0) it.nq++;
            it.smin = p.order[x.q0 + it.nq - 1].seen;
            for (int i = 0; i < it.nq; i++) count[p.order[x.q0 + i].query]++;
            p.items.push_back(it);
        }
    }
    std::stable_sort(p.items.begin(), p.items.end(), [&](const PageItem &a, const PageItem &b) {
        return (a.slot1 - a.slot0) * cost[a.form] > (b.slot1 - b.slot0) * cost[b.form];
    });
    std::vector<int> first(n + 1, 0);
    std::vector<char> joined(n, 0);
    for (PageItem &it : p.items) {
        bool alone = true;
        for (int i = 0; i < it.nq; i++) alone = alone && count[p.order[it.q0 + i].query] == 1;
        it.unit = alone ? -1 : p.num_units;
        if (alone) continue;
        p.most_queries = std::max(p.most_queries, it.nq);
        for (int i = 0; i < it.nq; i++) joined[p.order[it.q0 + i].query] = 1;
        p.num_units += it.nq;
    }
    for (int i = 0; i < n; i++) first[i + 1] = first[i] + (joined[i] ? count[i] : 0);
    p.units.resize(first[n]);
    p.join_of.assign(n, -1);
    p.empty = p.most_parts = 0;
    for (int i = 0; i < n; i++) {
        if (!joined[i]) continue;
        p.join_of[i] = (int)p.joins.size();
        p.joins.push_back({i, first[i], count[i], 0});
        p.most_parts = std::max(p.most_parts, count[i]);
    }
    for (int i = 0; i < n; i++) {
        if (count[i]) continue;
        p.joins.push_back({i, 0, 0, 0});
        p.empty++;
    }
    std::vector<int> next(first.begin(), first.end() - 1);
    for (const PageItem &it : p.items) {
        if (it.unit < 0) continue;
        for (int i = 0; i < it.nq; i++) p.units[next[p.order[it.q0 + i].query]++] = it.unit + i;
    }
    return 0;
}

}  // namespace fl

// CPU unit test of shared pages (no GPU, no HIP): forks, reorders and their
// refusals, then random sequences of every call against a model that keeps
// each row's tokens in a vector of its own.
#include "page_table.h"

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <set>
#include <vector>

static int g_fail = 0;

#define EXPECT(cond)                                                       \
    do {                                                                   \
        if (!(cond)) {                                                     \
            std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond);    \
            ++g_fail;                                                      \
        }                                                                  \
    } while (0)

static bool is(const sa::Verdict& v, sa_status st, const char* needle = nullptr) {
    return v.status == st && (!needle || std::strstr(v.msg, needle));
}

static void fixed_cases() {
    sa::PageTable pt;
    pt.init(/*max_seqs*/ 4, /*max_pages*/ 4, /*num_pages*/ 7);
    std::vector<sa::PageCopy> cp;
    EXPECT(pt.reserve(0, 200).ok() && pt.set_len(0, 150).ok());     // pages 0, 1, 2, 3

    EXPECT(is(pt.fork(1, 0, 151, &cp), SA_ERANGE, "committed"));
    EXPECT(is(pt.fork(0, 0, 10, &cp), SA_EINVAL));
    EXPECT(is(pt.fork(1, 4, 0, &cp), SA_ERANGE));
    EXPECT(is(pt.fork(-1, 0, 0, &cp), SA_ERANGE));
    EXPECT(is(pt.fork(1, 0, -1, &cp), SA_EINVAL));
    EXPECT(cp.empty() && pt.npages(1) == 0 && pt.refs(0) == 1);

    // 150 tokens: two whole pages shared, 22 tokens of the third copied
    EXPECT(pt.fork(1, 0, 150, &cp).ok() && cp.size() == 1);
    EXPECT(cp[0].src == 2 && cp[0].dst == 4 && cp[0].tokens == 22);
    EXPECT(pt.len(1) == 150 && pt.npages(1) == 3 && pt.refs(0) == 2 && pt.refs(2) == 1 && pt.refs(4) == 1);
    EXPECT(pt.owner(0) == sa::PageTable::kShared && pt.owner(2) == 0 && pt.owner(4) == 1 && pt.owner(6) == -1);
    const int32_t r01[] = {0, 1};
    EXPECT(pt.shared_tokens(r01, 0, 2, 0) == 128 && pt.shared_tokens(nullptr, 0, 2, 0) == 128);
    EXPECT(pt.shared_tokens(nullptr, 0, 1, 0) == 0 && pt.shared_tokens(nullptr, 0, 3, 0) == 0);
    // a whole number of pages copies nothing
    cp.clear();
    EXPECT(pt.fork(2, 1, 128, &cp).ok() && cp.empty() && pt.refs(0) == 3 && pt.npages(2) == 2);
    // the shortest row bounds what is shared; a pending token counts
    EXPECT(pt.set_len(2, 127).ok() && pt.shared_tokens(nullptr, 0, 3, 0) == 64);
    EXPECT(pt.shared_tokens(nullptr, 0, 3, 1) == 128);

    // nobody writes into a shared page
    const int32_t r2[] = {2};
    EXPECT(is(pt.check_append(r2, 1, 1, 0), SA_EINVAL, "shares"));
    EXPECT(pt.set_len(2, 128).ok() && pt.reserve(2, 129).ok() && pt.check_append(r2, 1, 1, 0).ok());
    // a page that another row lists stays refused to set_pages, also while it is shared
    EXPECT(is(pt.set_pages(3, std::vector<int32_t>{0}.data(), 1, nullptr), SA_EINVAL, "another"));
    // a row may list its own pages again, shared ones too; dropping them keeps the others' copies
    EXPECT(pt.set_pages(1, std::vector<int32_t>{0, 4}.data(), 2, nullptr).ok() && pt.refs(0) == 3 && pt.refs(1) == 2);
    EXPECT(pt.set_pages(1, nullptr, 0, nullptr).ok() && pt.refs(0) == 2 && pt.refs(4) == 0);
    EXPECT(pt.set_pages(2, nullptr, 0, nullptr).ok() && pt.owner(0) == 0 && pt.check_append(nullptr, 1, 1, 0).ok());

    // no page for the copy: refused, nothing changed
    pt.reset();
    EXPECT(pt.reserve(0, 256).ok() && pt.reserve(1, 192).ok() && pt.free_count() == 0);
    EXPECT(pt.set_len(0, 70).ok() && pt.set_len(1, 10).ok());
    EXPECT(is(pt.fork(2, 0, 70, &cp), SA_EFULL) && cp.empty() && pt.refs(0) == 1 && pt.npages(2) == 0);
    // dst's own page serves when the pool has none left
    EXPECT(pt.fork(1, 0, 70, &cp).ok() && cp.size() == 1 && pt.npages(1) == 2 && pt.free_count() == 2);

    // reorder refusals
    const int32_t r9[] = {0, 9};
    const int32_t r00[] = {0, 0};
    EXPECT(is(pt.reorder(r00, r01, 2, &cp), SA_EINVAL, "twice"));
    EXPECT(is(pt.reorder(r01, r9, 2, &cp), SA_ERANGE));
    EXPECT(is(pt.reorder(r9, r01, 2, &cp), SA_ERANGE));
    EXPECT(is(pt.reorder(nullptr, r01, 2, &cp), SA_EINVAL));
    EXPECT(is(pt.reorder(r01, r01, -1, &cp), SA_EINVAL));
    EXPECT(pt.reorder(nullptr, nullptr, 0, &cp).ok());

    // a swap moves both partial pages and copies nothing
    pt.reset();
    cp.clear();
    EXPECT(pt.reserve(0, 100).ok() && pt.reserve(1, 10).ok() && pt.set_len(0, 100).ok() && pt.set_len(1, 10).ok());
    const int32_t r10[] = {1, 0};
    EXPECT(pt.reorder(r01, r10, 2, &cp).ok() && cp.empty());
    EXPECT(pt.len(0) == 10 && pt.len(1) == 100 && pt.row(1)[0] == 0 && pt.row(1)[1] == 1 && pt.row(0)[0] == 2);
    EXPECT(pt.npages(0) == 2);   // its capacity stays
}

// ---------------------------------------------------------------------------
static uint64_t g_state = 12345;
static int rnd(int n) {
    g_state = g_state * 6364136223846793005ull + 1442695040888963407ull;
    return (int)((g_state >> 33) % (uint64_t)n);
}

static void random_calls(int seqs, int max_pages, int pages, int steps) {
    sa::PageTable pt;
    pt.init(seqs, max_pages, pages);
    std::vector<std::vector<int>> store(pages, std::vector<int>(64, -1));   // what each page holds
    std::vector<std::vector<int>> want(seqs);                               // each row's tokens
    int next = 0, done = 0, refused = 0;
    auto apply = [&](const std::vector<sa::PageCopy>& cp) {
        std::set<int> dsts;
        for (const auto& c : cp) {
            EXPECT(c.src != c.dst && c.tokens > 0 && c.tokens < 64 && pt.refs(c.dst) == 1);
            EXPECT(dsts.insert(c.dst).second);
        }
        for (const auto& c : cp) EXPECT(!dsts.count(c.src));   // the copies may run in any order
        for (const auto& c : cp) std::copy(store[c.src].begin(), store[c.src].begin() + c.tokens, store[c.dst].begin());
    };
    for (int step = 0; step < steps && !g_fail; ++step) {
        std::vector<sa::PageCopy> cp;
        const int what = rnd(10), s = rnd(seqs);
        if (what < 4) {   // append and commit
            const int n = 1 + rnd(what == 0 ? 100 : 3);
            if (pt.reserve(s, pt.len(s) + n).ok() && pt.check_append(&s, 1, n, 0).ok()) {
                for (int i = 0; i < n; ++i) {
                    const int t = pt.len(s) + i;
                    const int page = pt.row(s)[t / 64];
                    EXPECT(pt.refs(page) == 1);
                    store[page][t % 64] = next;
                    want[s].push_back(next++);
                }
                EXPECT(pt.commit(&s, 1, n).ok());
            } else ++refused;
        } else if (what < 6) {
            const int src = rnd(seqs), n = rnd(2) ? pt.len(src) : rnd(pt.len(src) + 1);
            if (pt.fork(s, src, n, &cp).ok()) {
                apply(cp);
                want[s].assign(want[src].begin(), want[src].begin() + n);
                ++done;
            } else ++refused;
        } else if (what < 8) {
            std::vector<int32_t> rows, par;
            for (int r = 0; r < seqs; ++r)
                if (rnd(3)) {
                    rows.push_back(r);
                    par.push_back(rnd(4) ? rnd(seqs) : r);
                }
            std::vector<int> before(seqs);
            for (int r = 0; r < seqs; ++r) before[r] = pt.npages(r);
            if (pt.reorder(rows.data(), par.data(), (int)rows.size(), &cp).ok()) {
                apply(cp);
                const auto old = want;
                for (size_t i = 0; i < rows.size(); ++i) {
                    want[rows[i]] = old[par[i]];
                    EXPECT(pt.npages(rows[i]) >= before[rows[i]]);
                }
                ++done;
            } else {
                EXPECT(cp.empty());
                ++refused;
            }
        } else if (what == 8) {
            const int n = rnd(pt.capacity(s) + 1);
            if (n <= pt.len(s)) {
                EXPECT(pt.set_len(s, n).ok());
                want[s].resize(n);
            }
        } else if (pt.npages(s) && rnd(2)) {   // keep some of the leading pages
            const int keep = rnd(pt.npages(s) + 1);
            const std::vector<int32_t> list(pt.row(s), pt.row(s) + keep);
            EXPECT(pt.set_pages(s, list.data(), keep, nullptr).ok());
            want[s].resize(std::min<int>((int)want[s].size(), keep * 64));
        }
        // every row reads back its own tokens; the counts and the free list agree with the table
        std::vector<int> refs(pages, 0);
        int used = 0;
        for (int r = 0; r < seqs; ++r) {
            EXPECT(pt.len(r) == (int)want[r].size() && pt.len(r) <= pt.capacity(r));
            for (int j = 0; j < max_pages; ++j) {
                const int page = pt.row(r)[j];
                EXPECT((page >= 0) == (j < pt.npages(r)));
                if (page >= 0) ++refs[page];
            }
            for (int t = 0; t < pt.len(r); ++t) EXPECT(store[pt.row(r)[t / 64]][t % 64] == want[r][t]);
        }
        for (int p = 0; p < pages; ++p) {
            EXPECT(refs[p] == pt.refs(p));
            used += refs[p] > 0;
        }
        EXPECT(pt.free_count() == pages - used);
    }
    EXPECT(done > 0 && refused > 0);
}

int main() {
    fixed_cases();
    random_calls(6, 4, 14, 20000);
    random_calls(3, 6, 9, 20000);
    random_calls(12, 3, 20, 20000);
    if (g_fail) {
        std::printf("%d check(s) failed\n", g_fail);
        return 1;
    }
    std::printf("page sharing: all checks passed\n");
    return 0;
}

// Host bookkeeping of the paged KV cache (see page_table.h).
#include "page_table.h"

#include <algorithm>

namespace sa {

namespace {
constexpr Verdict kOk{SA_OK, ""};
Verdict refuse(sa_status st, const char* msg) { return Verdict{st, msg}; }
}  // namespace

void PageTable::init(int max_seqs, int max_pages_per_seq, int num_pages) {
    max_seqs_ = max_seqs;
    max_pages_ = max_pages_per_seq;
    num_pages_ = num_pages;
    reset();
}

void PageTable::reset() {
    table_.assign((size_t)max_seqs_ * max_pages_, -1);
    lens_.assign(max_seqs_, 0);
    npages_.assign(max_seqs_, 0);
    refs_.assign(num_pages_, 0);
    free_.resize(num_pages_);
    for (int i = 0; i < num_pages_; ++i) free_[i] = num_pages_ - 1 - i;
}

Verdict PageTable::reserve(int seq, int n_tokens) {
    if (!valid_seq(seq)) return refuse(SA_ERANGE, "sequence index out of range");
    if (n_tokens < 0) return refuse(SA_EINVAL, "n_tokens must be >= 0");
    const long long need = ((long long)n_tokens + kPage - 1) / kPage;
    if (need > max_pages_) return refuse(SA_EFULL, "KV cache full, cannot append more tokens");
    int have = npages_[seq];
    if (need <= have) return kOk;
    if ((long long)free_.size() < need - have) return refuse(SA_EFULL, "KV cache full, cannot append more tokens");
    int32_t* r = table_.data() + (size_t)seq * max_pages_;
    for (; have < need; ++have) {
        const int32_t p = free_.back();
        free_.pop_back();
        r[have] = p;
        refs_[p] = 1;
    }
    npages_[seq] = have;
    return kOk;
}

Verdict PageTable::set_pages(int seq, const int32_t* pages, int n, bool* len_cut) {
    if (len_cut) *len_cut = false;
    if (!valid_seq(seq)) return refuse(SA_ERANGE, "sequence index out of range");
    if (n < 0 || n > max_pages_ || (n > 0 && !pages)) return refuse(SA_EINVAL, "bad page list");
    std::vector<char> listed(num_pages_, 0), mine(num_pages_, 0);
    int32_t* r = row_mut(seq);
    for (int j = 0; j < npages_[seq]; ++j) mine[r[j]] = 1;
    for (int j = 0; j < n; ++j) {
        const int32_t p = pages[j];
        if (p < 0 || p >= num_pages_) return refuse(SA_ERANGE, "page id out of range");
        if (listed[p]) return refuse(SA_EINVAL, "page listed twice");
        listed[p] = 1;
        if (refs_[p] != 0 && !mine[p]) return refuse(SA_EINVAL, "page owned by another sequence");
    }
    // The sequence's pages that are not kept go back to the free list, unless
    // another sequence shares them.
    for (int j = 0; j < npages_[seq]; ++j) {
        const int32_t p = r[j];
        if (!listed[p] && --refs_[p] == 0) free_.push_back(p);
    }
    // Listed pages that were free leave the free list.
    free_.erase(std::remove_if(free_.begin(), free_.end(), [&](int32_t p) { return listed[p] != 0; }),
                free_.end());
    for (int j = 0; j < max_pages_; ++j) r[j] = j < n ? pages[j] : -1;
    for (int j = 0; j < n; ++j)
        if (!mine[pages[j]]) refs_[pages[j]] = 1;
    npages_[seq] = n;
    if (lens_[seq] > n * kPage) {
        lens_[seq] = n * kPage;
        if (len_cut) *len_cut = true;
    }
    return kOk;
}

Verdict PageTable::set_len(int seq, int len) {
    if (!valid_seq(seq)) return refuse(SA_ERANGE, "sequence index out of range");
    if (len < 0 || len > capacity(seq)) return refuse(SA_EFULL, "length exceeds reserved pages");
    lens_[seq] = len;
    return kOk;
}

Verdict PageTable::set_lens(const int32_t* seqs, const int32_t* lens, int n) {
    Verdict v = check_rows(seqs, n, true);
    if (!v.ok()) return v;
    for (int i = 0; i < n; ++i)
        if (lens[i] < 0 || lens[i] > capacity(seqs[i])) return refuse(SA_EFULL, "length exceeds reserved pages");
    for (int i = 0; i < n; ++i) lens_[seqs[i]] = lens[i];
    return kOk;
}

Verdict PageTable::check_rows(const int32_t* ids, int n, bool unique) const {
    if (n < 0) return refuse(SA_EINVAL, "negative sequence count");
    if (!ids) {
        if (n > max_seqs_) return refuse(SA_ERANGE, "sequence index out of range");
        return kOk;
    }
    std::vector<char> seen(unique ? max_seqs_ : 0, 0);
    for (int i = 0; i < n; ++i) {
        if (!valid_seq(ids[i])) return refuse(SA_ERANGE, "sequence index out of range");
        if (unique) {
            if (seen[ids[i]]) return refuse(SA_EINVAL, "sequence listed twice");
            seen[ids[i]] = 1;
        }
    }
    return kOk;
}

Verdict PageTable::check_append(const int32_t* ids, int n, int S, int rope_max_pos) const {
    Verdict v = check_rows(ids, n, true);
    if (!v.ok()) return v;
    for (int i = 0; i < n; ++i) {
        v = check_append_row(ids ? ids[i] : i, S, rope_max_pos);
        if (!v.ok()) return v;
    }
    return kOk;
}

Verdict PageTable::check_append(const int32_t* ids, int n, const int32_t* counts, int rope_max_pos) const {
    Verdict v = check_rows(ids, n, true);
    if (!v.ok()) return v;
    for (int i = 0; i < n; ++i) {
        if (counts[i] < 0) return refuse(SA_EINVAL, "counts must be >= 0");
        if (counts[i] == 0) continue;
        v = check_append_row(ids ? ids[i] : i, counts[i], rope_max_pos);
        if (!v.ok()) return v;
    }
    return kOk;
}

Verdict PageTable::check_append_row(int s, int S, int rope_max_pos) const {
    const long long end = (long long)lens_[s] + S;
    if (end > capacity(s)) return refuse(SA_EFULL, "KV cache full, cannot append more tokens");
    if (rope_max_pos > 0 && end > rope_max_pos) return refuse(SA_ERANGE, "position beyond RoPE table");
    for (long long j = lens_[s] / kPage; j * kPage < end; ++j)
        if (refs_[row(s)[j]] > 1) return refuse(SA_EINVAL, "append into a page that another sequence shares");
    return kOk;
}

Verdict PageTable::check_decode(const int32_t* ids, int n, int n_pending, int* max_len, long long* total) const {
    Verdict v = check_rows(ids, n, false);
    if (!v.ok()) return v;
    if (n_pending < 0) return refuse(SA_EINVAL, "n_pending must be >= 0");
    int mx = 0;
    long long sum = 0;
    for (int i = 0; i < n; ++i) {
        const int s = ids ? ids[i] : i;
        const long long L = (long long)lens_[s] + n_pending;
        if (L > capacity(s)) return refuse(SA_ERANGE, "Requested seq_len exceeds cached length");
        mx = std::max(mx, (int)L);
        sum += L;
    }
    if (max_len) *max_len = mx;
    if (total) *total = sum;
    return kOk;
}

Verdict PageTable::commit(const int32_t* ids, int n_rows, int n) {
    if (n < 0) return refuse(SA_EINVAL, "n must be >= 0");
    Verdict v = check_rows(ids, n_rows, true);
    if (!v.ok()) return v;
    for (int i = 0; i < n_rows; ++i) {
        const int s = ids ? ids[i] : i;
        if ((long long)lens_[s] + n > capacity(s)) return refuse(SA_EFULL, "KV cache full, cannot append more tokens");
    }
    for (int i = 0; i < n_rows; ++i) lens_[ids ? ids[i] : i] += n;
    return kOk;
}

int PageTable::owner(int page) const {
    if (refs_[page] != 1) return refs_[page] == 0 ? -1 : kShared;
    for (int s = 0; s < max_seqs_; ++s)
        if (std::find(row(s), row(s) + npages_[s], page) != row(s) + npages_[s]) return s;
    return -1;
}

Verdict PageTable::fork(int dst, int src, int n_tokens, std::vector<PageCopy>* copies) {
    if (!valid_seq(dst) || !valid_seq(src)) return refuse(SA_ERANGE, "sequence index out of range");
    if (dst == src) return refuse(SA_EINVAL, "a sequence cannot be forked onto itself");
    if (n_tokens < 0) return refuse(SA_EINVAL, "n_tokens must be >= 0");
    if (n_tokens > lens_[src]) return refuse(SA_ERANGE, "fork beyond the committed length");
    copies->reserve(copies->size() + 1);
    const int full = n_tokens / kPage, rem = n_tokens % kPage;
    int32_t* d = row_mut(dst);
    const int32_t* s = row(src);
    if (rem) {
        // A page that src does not list and that is free, or is once dst has
        // given its own back.
        bool room = !free_.empty();
        for (int j = 0; !room && j < npages_[dst]; ++j) room = refs_[d[j]] == 1;
        if (!room) return refuse(SA_EFULL, "KV cache full, no page for the copy");
    }
    for (int j = 0; j < full; ++j) ++refs_[s[j]];
    for (int j = 0; j < npages_[dst]; ++j)
        if (--refs_[d[j]] == 0) free_.push_back(d[j]);
    std::copy(s, s + full, d);
    int have = full;
    if (rem) {
        const int32_t p = free_.back();
        free_.pop_back();
        refs_[p] = 1;
        copies->push_back(PageCopy{s[full], p, rem});
        d[have++] = p;
    }
    std::fill(d + have, d + max_pages_, -1);
    npages_[dst] = have;
    lens_[dst] = n_tokens;
    return kOk;
}

Verdict PageTable::reorder(const int32_t* rows, const int32_t* parents, int n, std::vector<PageCopy>* copies) {
    if (n < 0) return refuse(SA_EINVAL, "negative sequence count");
    if (n > 0 && (!rows || !parents)) return refuse(SA_EINVAL, "null rows or parents");
    Verdict v = check_rows(rows, n, true);
    if (!v.ok()) return v;
    v = check_rows(parents, n, false);
    if (!v.ok()) return v;

    // What each replaced row will list: the parent's whole pages, then the
    // pages of its own, of which the first holds the parent's partial page
    // (moved from the parent, or -1: fresh, with a copy).
    struct Plan {
        int row, full, rem, have, moved;
        std::vector<int32_t> shared;
        int32_t src;
        int len;
    };
    std::vector<char> replaced(max_seqs_, 0), given(max_seqs_, 0);
    for (int i = 0; i < n; ++i)
        if (rows[i] != parents[i]) replaced[rows[i]] = 1;
    std::vector<int32_t> refs = refs_;
    std::vector<char> source(num_pages_, 0);   // read by a copy: not handed out in this call
    std::vector<Plan> plans;
    long long fresh = 0;
    for (int i = 0; i < n; ++i) {
        const int r = rows[i], p = parents[i];
        if (r == p) continue;
        Plan q{r, lens_[p] / kPage, lens_[p] % kPage, 0, -1, {}, -1, lens_[p]};
        q.shared.assign(row(p), row(p) + q.full);
        q.have = std::max(npages_[r], q.full + (q.rem ? 1 : 0));
        if (q.rem) {
            const int32_t page = row(p)[q.full];
            if (replaced[p] && !given[p] && refs_[page] == 1) {
                given[p] = 1;
                q.moved = page;
            } else {
                q.src = page;
                source[page] = 1;
            }
        }
        fresh += q.have - q.full - (q.moved >= 0 ? 1 : 0);
        plans.push_back(std::move(q));
    }
    for (const Plan& q : plans) {
        for (int32_t page : q.shared) ++refs[page];
        if (q.moved >= 0) ++refs[q.moved];
        for (int j = 0; j < npages_[q.row]; ++j) --refs[row(q.row)[j]];
    }
    std::vector<int32_t> freed, kept;
    for (const Plan& q : plans) {
        for (int j = 0; j < npages_[q.row]; ++j) {
            const int32_t page = row(q.row)[j];
            if (refs[page] == 0) {
                refs[page] = -1;   // listed once below
                (source[page] ? kept : freed).push_back(page);
            }
        }
    }
    if (fresh > (long long)(free_.size() + freed.size()))
        return refuse(SA_EFULL, "KV cache full, no pages for the reordered sequences");

    // Nothing can be refused, and nothing allocates, from here on.
    copies->reserve(copies->size() + plans.size());
    for (int32_t page : freed) refs[page] = 0;
    for (int32_t page : kept) refs[page] = 0;
    refs_ = std::move(refs);
    free_.insert(free_.end(), freed.begin(), freed.end());
    for (const Plan& q : plans) {
        int32_t* d = row_mut(q.row);
        std::copy(q.shared.begin(), q.shared.end(), d);
        for (int j = q.full; j < q.have; ++j) {
            if (j == q.full && q.moved >= 0) {
                d[j] = q.moved;
                continue;
            }
            d[j] = free_.back();
            free_.pop_back();
            refs_[d[j]] = 1;
            if (j == q.full && q.rem) copies->push_back(PageCopy{q.src, d[j], q.rem});
        }
        std::fill(d + q.have, d + max_pages_, -1);
        npages_[q.row] = q.have;
        lens_[q.row] = q.len;
    }
    free_.insert(free_.end(), kept.begin(), kept.end());
    return kOk;
}

int PageTable::shared_tokens(const int32_t* ids, int first, int n, int n_pending) const {
    if (n < 2) return 0;
    const int32_t* a = row(ids ? ids[0] : first);
    long long pages = max_pages_;
    for (int i = 0; i < n; ++i) {
        const int s = ids ? ids[i] : first + i;
        pages = std::min<long long>(pages, ((long long)lens_[s] + n_pending) / kPage);
        pages = std::min<long long>(pages, npages_[s]);
        pages = std::mismatch(a, a + pages, row(s)).first - a;
    }
    return (int)pages * kPage;
}

}  // namespace sa

// Host-side bookkeeping of the paged KV cache: which pages each sequence
// owns, the committed lengths, the free list, and every check an append or a
// decode needs before a kernel is launched.  No HIP here: the device copy of
// the table and the lengths is written by the cache glue (kvcache.hip) from
// what this class decides, and the class is unit-tested on the CPU.
//
// The reference's dense cache has one length for the whole batch and throws
// on overflow (reference tensor_cpp/include/tensor_cpp/kv_cache.h:94-130); here
// each sequence has its own pages and length, and every overflow, bad index
// or page conflict is refused before any device work is enqueued.
//
// Pages may be shared: after a fork or a reorder several sequences list the
// same leading pages, each counted once per sequence.  A shared page is never
// written: an append whose tokens would fall into one is refused.
#pragma once

#include <stdint.h>

#include <vector>

#include "sa_amd.h"

namespace sa {

struct Verdict {
    sa_status status;
    const char* msg;   // static text; "" when status == SA_OK
    bool ok() const { return status == SA_OK; }
};

// The first tokens rows of page src are to be copied to page dst (every layer,
// K and V).
struct PageCopy {
    int32_t src, dst, tokens;
};

class PageTable {
public:
    void init(int max_seqs, int max_pages_per_seq, int num_pages);
    // Every sequence back to length 0, every page back to the free list
    // (page 0 is handed out first).
    void reset();

    // Room for n_tokens tokens in total in seq, taking pages from the free list.
    Verdict reserve(int seq, int n_tokens);
    // Replace seq's pages with pages[0, n).  Every page must be in the pool,
    // listed once, and either free or already one of seq's.  A length beyond
    // the new capacity is cut to it (*len_cut tells the caller to publish it).
    Verdict set_pages(int seq, const int32_t* pages, int n, bool* len_cut);
    Verdict set_len(int seq, int len);
    // Lengths lens[0, n) of rows seqs[0, n), each listed once; refused as a whole.
    Verdict set_lens(const int32_t* seqs, const int32_t* lens, int n);
    // Rows ids[0, n) (NULL: 0 .. n-1) are cache rows; with unique, no row twice.
    Verdict check_rows(const int32_t* ids, int n, bool unique) const;
    // An append of S tokens to each row: every row has pages of its own (none
    // that another row shares) for tokens len .. len + S - 1 and, when
    // rope_max_pos > 0, len + S <= rope_max_pos.
    Verdict check_append(const int32_t* ids, int n, int S, int rope_max_pos) const;
    // The same of counts[i] >= 0 tokens to row i.
    Verdict check_append(const int32_t* ids, int n, const int32_t* counts, int rope_max_pos) const;
    // A decode over len + n_pending tokens of each row: every row has pages for
    // them.  Returns the longest such length and their sum.
    Verdict check_decode(const int32_t* ids, int n, int n_pending, int* max_len, long long* total) const;
    // len += n for each row, refused as a whole if any row would overflow.
    Verdict commit(const int32_t* ids, int n_rows, int n);
    // Row dst gives its pages back and becomes the first n_tokens committed
    // tokens of src: it shares src's whole pages and, where n_tokens ends
    // inside a page, gets a page of its own (a copy is appended to *copies).
    Verdict fork(int dst, int src, int n_tokens, std::vector<PageCopy>* copies);
    // At once for all i: row rows[i] (each listed once) becomes what row
    // parents[i] was, with parents[i]'s length.  Whole pages are shared; the
    // page that the length ends inside goes to one of the parent's children
    // if the parent is itself replaced, the others get a page of their own and
    // a copy.  A row keeps its capacity (spare pages behind its tokens) unless
    // the parent's tokens need more.  A row that is its own parent is left as
    // it is.  Refused as a whole if the pool has too few pages.
    Verdict reorder(const int32_t* rows, const int32_t* parents, int n, std::vector<PageCopy>* copies);
    // Tokens in the whole pages that rows ids[0, n) (NULL: first, first + 1,
    // ...) list alike from the start on, up to the shortest row's
    // len + n_pending.  0 for fewer than two rows.
    int shared_tokens(const int32_t* ids, int first, int n, int n_pending) const;

    int max_seqs() const { return max_seqs_; }
    int max_pages() const { return max_pages_; }
    int num_pages() const { return num_pages_; }
    int len(int seq) const { return lens_[seq]; }
    int capacity(int seq) const { return npages_[seq] * kPage; }
    int npages(int seq) const { return npages_[seq]; }
    int free_count() const { return (int)free_.size(); }
    int refs(int page) const { return refs_[page]; }   // rows that list the page
    // The one row that lists the page; -1: none, kShared: several.
    int owner(int page) const;
    static constexpr int kShared = -2;
    const int32_t* row(int seq) const { return table_.data() + (size_t)seq * max_pages_; }
    bool valid_seq(int seq) const { return seq >= 0 && seq < max_seqs_; }

    static constexpr int kPage = SA_PAGE_TOKENS;

private:
    int max_seqs_ = 0, max_pages_ = 0, num_pages_ = 0;
    std::vector<int32_t> table_;   // [max_seqs][max_pages], -1 = no page
    std::vector<int> lens_;        // committed length per sequence
    std::vector<int> npages_;      // pages assigned per sequence
    std::vector<int32_t> free_;    // stack of free pages
    std::vector<int32_t> refs_;    // [num_pages]: rows that list the page, 0 = free

    Verdict check_append_row(int seq, int S, int rope_max_pos) const;
    int32_t* row_mut(int seq) { return table_.data() + (size_t)seq * max_pages_; }
};

}  // namespace sa

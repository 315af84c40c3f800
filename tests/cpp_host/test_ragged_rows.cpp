// CPU unit test of the page table's ragged checks (no GPU, no HIP): appends of a
// count per row and lengths of many rows at once, refused as a whole.
#include "page_table.h"

#include <cstdio>
#include <cstring>
#include <vector>

static int g_fail = 0;

#define EXPECT(cond)                                                       \
    do {                                                                   \
        if (!(cond)) {                                                     \
            std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond);    \
            ++g_fail;                                                      \
        }                                                                  \
    } while (0)

static bool is(const sa::Verdict& v, sa_status st, const char* needle) {
    return v.status == st && std::strstr(v.msg, needle) != nullptr;
}

int main() {
    sa::PageTable pt;
    pt.init(/*max_seqs*/ 4, /*max_pages*/ 4, /*num_pages*/ 12);
    EXPECT(pt.reserve(0, 100).ok() && pt.reserve(1, 64).ok() && pt.reserve(2, 256).ok());   // 128, 64, 256, 0 tokens
    const int32_t rows[] = {0, 1, 2}, lens[] = {100, 64, 7};
    EXPECT(pt.set_lens(rows, lens, 3).ok());
    EXPECT(pt.len(0) == 100 && pt.len(1) == 64 && pt.len(2) == 7 && pt.len(3) == 0);

    const int32_t fits[] = {28, 0, 249, 0}, over[] = {28, 1, 0, 0}, back[] = {1, -1, 0, 0}, none[] = {0, 0, 0, 0};
    EXPECT(pt.check_append(nullptr, 4, fits, 0).ok());
    EXPECT(pt.check_append(nullptr, 4, none, 1).ok());      // rows without tokens are not looked at
    EXPECT(is(pt.check_append(nullptr, 4, over, 0), SA_EFULL, "full"));
    EXPECT(is(pt.check_append(nullptr, 4, back, 0), SA_EINVAL, "counts"));
    EXPECT(is(pt.check_append(nullptr, 4, fits, 128 + 127), SA_ERANGE, "RoPE"));
    EXPECT(pt.check_append(nullptr, 4, fits, 256).ok());
    EXPECT(is(pt.check_append(nullptr, 5, none, 0), SA_ERANGE, "range"));
    const int32_t twice[] = {2, 2}, one[] = {1, 1};
    EXPECT(is(pt.check_append(twice, 2, one, 0), SA_EINVAL, "twice"));

    // a shared page refuses the row whose tokens would fall into it, not the others
    std::vector<sa::PageCopy> copies;
    EXPECT(pt.fork(3, 0, 64, &copies).ok());
    const int32_t to[] = {3, 0}, at[] = {10, 100};
    EXPECT(pt.set_lens(to, at, 2).ok());
    const int32_t into[] = {0, 0, 0, 1}, beside[] = {5, 0, 5, 0};
    EXPECT(is(pt.check_append(nullptr, 4, into, 0), SA_EINVAL, "shares"));
    EXPECT(pt.check_append(nullptr, 4, beside, 0).ok());

    // refused as a whole
    const int32_t bad_rows[] = {0, 9}, same[] = {1, 1}, high[] = {1, 65}, low[] = {1, -1};
    EXPECT(is(pt.set_lens(bad_rows, one, 2), SA_ERANGE, "range"));
    EXPECT(is(pt.set_lens(same, one, 2), SA_EINVAL, "twice"));
    EXPECT(is(pt.set_lens(rows, high, 2), SA_EFULL, "length"));
    EXPECT(is(pt.set_lens(rows, low, 2), SA_EFULL, "length"));
    EXPECT(pt.len(0) == 100 && pt.len(1) == 64);
    EXPECT(pt.set_lens(nullptr, nullptr, 0).ok());

    if (g_fail) return 1;
    std::printf("all checks passed\n");
    return 0;
}

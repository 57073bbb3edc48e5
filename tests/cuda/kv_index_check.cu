// Host-side check of the paged cache's index arithmetic (attn.cuh): the functions that the
// kernels call, run on the CPU over random starts, tables and lengths, wrong ones among them.
// Prints "ok" or the first case that leaves its bounds.
#include "attn.cuh"

#include <cstdio>
#include <random>
#include <vector>

using namespace amoe::attn;

namespace amoe {
void set_thread_error(const std::string &) {}
}  // namespace amoe

int main() {
    std::mt19937 r(7);
    auto in = [&](int lo, int hi) { return (int)(lo + r() % (unsigned)(hi - lo + 1)); };
    for (int c = 0; c < 20000; ++c) {
        const int seqs = in(1, 9);
        std::vector<int32_t> cu(seqs + 1);
        const bool wild = c % 3 == 0;
        int at = 0;
        for (int i = 0; i <= seqs; ++i) {
            cu[i] = wild ? (int)r() : at;
            at += in(0, 5);
        }
        const int t = wild ? in(0, 100) : in(0, cu[seqs] + 3);
        const int s = find_seq(cu.data(), seqs, t);
        if (s < 0 || s >= seqs) return printf("find_seq %d of %d\n", s, seqs), 1;
        if (!wild && t < cu[seqs] && !(cu[s] <= t && t < cu[s + 1])) return printf("row %d not in %d\n", t, s), 1;

        CacheDev k{};
        k.pages = in(1, 12);
        k.table_stride = in(1, 6);
        k.shift = in(0, 7);
        k.heads = in(1, 4);
        std::vector<int32_t> table((size_t)seqs * k.table_stride);
        for (auto &p : table) p = in(0, 4) ? in(0, (int)k.pages - 1) : (int)r();
        k.table = table.data();
        const int64_t pos = in(0, 3) ? in(0, (k.table_stride << k.shift) + 5) : (int64_t)INT32_MAX + in(0, 1 << 20);
        const int page = lookup_page(k, s, pos);
        if ((pos >> k.shift) >= k.table_stride) {
            if (page != -AMOE_KV_PAST_TABLE) return printf("position %lld past the table\n", (long long)pos), 1;
            continue;
        }
        const int want = table[(size_t)s * k.table_stride + (pos >> k.shift)];
        if (want < 0 || want >= k.pages) {
            if (page != -AMOE_KV_BAD_PAGE) return printf("page %d accepted\n", want), 1;
            continue;
        }
        if (page != want) return printf("page %d, want %d\n", page, want), 1;
        const int64_t row = cache_row(k, page, k.heads - 1, pos);
        if (row < 0 || row >= (k.pages * k.heads) << k.shift) return printf("row %lld\n", (long long)row), 1;
    }
    CacheDev k{};  // offsets of a long cache pass 32 bits
    k.heads = 8, k.shift = 7;
    if (cache_row(k, 5000000, 7, 12345) != ((5000000LL * 8 + 7) << 7 | (12345 & 127))) return printf("64-bit row\n"), 1;
    return printf("ok\n"), 0;
}

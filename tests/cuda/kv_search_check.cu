// Host-side check of the search for packed rows' sequences (attn.cuh: find_seqs), the one that the kernels run, over
// more sequences than a warp looks at in one step: right for starts that ascend, in range for any others.
// And the last fill of a ring's stage, which the prefill waits for before it ends.
// Prints "ok" or the first case that fails.
#include "attn.cuh"

#include <cstdio>
#include <random>
#include <vector>

using namespace amoe::attn;

namespace amoe {
void set_thread_error(const std::string &) {}
}  // namespace amoe

int main() {
    std::mt19937 r(11);
    auto in = [&](int lo, int hi) { return (int)(lo + r() % (unsigned)(hi - lo + 1)); };
    for (int c = 0; c < 20000; ++c) {
        const int seqs = c % 2 ? in(30, 200) : 32 * in(1, 5) + in(-1, 1);
        const bool wild = c % 4 == 0;
        const int most = in(0, 3) ? in(0, 4) : 200;
        std::vector<int32_t> cu(seqs + 1);
        for (int i = 0, at = 0; i <= seqs; ++i) {
            cu[i] = wild ? (int)r() : at;
            at += in(0, 1) ? in(0, most) : 0;
        }
        const int t = in(0, wild ? 1000 : cu[seqs] + 5);
        int four[4];
        find_seqs(cu.data(), seqs, t, four);
        for (int k = 0; k < 4; ++k) {
            const int s = four[k];
            if (s < 0 || s >= seqs) return printf("sequence %d of %d\n", s, seqs), 1;
            if (!wild && s != find_seq(cu.data(), seqs, t + k)) return printf("row %d alone differs\n", t + k), 1;
            if (!wild && t + k < cu[seqs] && !(cu[s] <= t + k && t + k < cu[s + 1]))
                return printf("row %d of %d sequences not in %d\n", t + k, seqs, s), 1;
        }
    }
    for (int stages = 1; stages < 5; ++stages)
        for (int fills = 0; fills < 20; ++fills)
            for (int s = 0; s < stages; ++s) {
                int want = -1;
                for (int i = 0; i < fills; ++i)
                    if (i % stages == s) want = i;
                if (last_fill(fills, s, stages) != want) return printf("last fill of stage %d of %d\n", s, stages), 1;
            }
    return printf("ok\n"), 0;
}

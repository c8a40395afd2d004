// kv4_pieces against CTAs that go through random lists of units, and with
// workspace entries that are arbitrary.
#include "kv4_pieces.h"

#include <cstdio>
#include <cstdint>
#include <random>
#include <vector>

int main() {
    std::mt19937_64 rng(1);
    auto draw = [&](int lo, int hi) { return lo + (int)(rng() % (uint64_t)(hi - lo + 1)); };
    const int kCost = 3;   // of a unit, before its pages
    for (int round = 0; round < 2000; ++round) {
        const int ctas = draw(1, 160), units = draw(1, 300), longest = draw(1, 200);
        std::vector<int> pages(units), at(units);
        long long all = 0;
        for (int u = 0; u < units; ++u) {
            pages[u] = draw(0, longest);
            at[u] = (int)all + kCost;
            if (pages[u]) all += pages[u] + kCost;
        }
        const int even = (int)((all + ctas - 1) / ctas), chunk = even > kCost + 2 ? even : kCost + 2;
        for (int u = 0; u < units; ++u) {
            int first = -1, count = 0;   // the CTAs whose share has one of the unit's pages
            for (int c = 0; c < ctas && pages[u]; ++c) {
                const long long lo = (long long)c * chunk, hi = lo + chunk;
                if (lo < at[u] + pages[u] && hi > at[u]) {
                    if (first < 0) first = c;
                    ++count;
                }
            }
            const kvp::Kv4Pieces p = kvp::kv4_pieces(chunk, at[u], pages[u], ctas);
            if (p.count != count || (count && p.first != first)) {
                std::printf("unit %d: CTAs %d + %d, expected %d + %d\n", u, p.first, p.count, first, count);
                return 1;
            }
        }
    }
    const int ends[] = {0, 1, -1, INT32_MAX, INT32_MIN, INT32_MAX - 1};
    for (int i = 0; i < 5000000; ++i) {
        auto any = [&] { return rng() % 4 ? (int)(uint32_t)rng() : ends[rng() % 6]; };
        const int ctas = draw(1, 160), pages = draw(0, 1 << 23);
        const kvp::Kv4Pieces p = kvp::kv4_pieces(rng() % 2 ? any() : draw(-4, 40), rng() % 2 ? any() : draw(-4, 4000),
                                                 pages, ctas);
        if (p.count < 0 || p.first < 0 || (long long)p.first + p.count > ctas) {
            std::printf("CTAs %d + %d of %d\n", p.first, p.count, ctas);
            return 1;
        }
    }
    std::printf("kv4 pieces ok\n");
}

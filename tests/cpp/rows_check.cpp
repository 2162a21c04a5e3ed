// Whether rows lie over one another (csrc/rows.hpp), against all pairs of rows of small tensors.
// Prints how often each answer was given, and "rows_check: OK".
#include <cstdio>
#include <random>

#include "../../cu-roaring-bitmap_amd/csrc/rows.hpp"

using namespace crimpl;

static bool meet(const Rows& a, const Rows& b, bool same)
{
    for (uint64_t t = 0; t < a.tokens; ++t)
        for (uint64_t h = 0; h < a.heads; ++h)
            for (uint64_t u = 0; u < b.tokens; ++u)
                for (uint64_t g = 0; g < b.heads; ++g) {
                    if (same && t == u && h == g) continue;
                    const int64_t x = static_cast<int64_t>(a.at + t * a.token + h * a.head);
                    const int64_t y = static_cast<int64_t>(b.at + u * b.token + g * b.head);
                    if (x < y + static_cast<int64_t>(b.row) && y < x + static_cast<int64_t>(a.row)) return true;
                }
    return false;
}

int main()
{
    std::mt19937 rng(1);
    auto pick = [&](uint32_t lo, uint32_t hi) { return lo + rng() % (hi - lo + 1); };
    int errors = 0, answers[2][2] = {};
    for (int i = 0; i < 300000; ++i) {
        const uint64_t tokens = pick(1, 5), heads = pick(1, 5), row = pick(1, 6);
        auto stride = [&] { return pick(0, 9) ? row * pick(0, 7) + (pick(0, 3) ? 0 : pick(0, 5)) : pick(0, 60); };
        const uint64_t token = stride(), head = stride();
        const Rows a(reinterpret_cast<void*>(1000), tokens, token, heads, head, row);
        const bool want = meet(a, a, true), got = rows_overlap(a);
        errors += want != got;
        ++answers[0][got];
        const Rows b(reinterpret_cast<void*>(static_cast<uintptr_t>(pick(0, 2) ? 1000 + row * pick(0, 12) : pick(850, 1150))), tokens, token,
                     heads, head, row);
        const bool over = rows_overwrite(b, a);
        errors += over != (a.at == b.at ? false : meet(b, a, false));
        ++answers[1][over];
        // other strides: refused unless apart
        const Rows c(reinterpret_cast<void*>(static_cast<uintptr_t>(pick(900, 1100))), tokens, stride(), heads, stride(), row);
        if (meet(c, a, c.at == a.at && c.token == a.token && c.head == a.head) && !rows_overwrite(c, a))
            errors += !(c.at == a.at && c.token == a.token && c.head == a.head);
    }
    // strides that only rows of one token, or of one head, could have
    errors += rows_overlap(Rows(nullptr, 1, ~0ull, 4, 8, 8)) || rows_overlap(Rows(nullptr, 3, 8, 1, 0, 8));
    errors += rows_overlap(Rows(nullptr, 1u << 31, ~0ull >> 1, 65535, 8, 8));
    printf("over one another: %d of %d; written over others: %d of %d\n", answers[0][1], answers[0][0] + answers[0][1], answers[1][1],
           answers[1][0] + answers[1][1]);
    if (errors || !answers[0][0] || !answers[0][1] || !answers[1][0] || !answers[1][1]) {
        printf("rows_check: %d errors\n", errors);
        return 1;
    }
    printf("rows_check: OK\n");
    return 0;
}

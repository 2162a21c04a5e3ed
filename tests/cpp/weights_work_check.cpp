// How cr_paged_weights splits its work (csrc/weights_work.hpp), run on the CPU for shapes of every size.
//   - every launch has work and fewer than 2^32 threads, whatever the caller says of its lengths;
//   - the requests with many rows fit the list that is made of them;
//   - the sums that a launch leaves take at most 512 MB.
// Prints how often each way was taken, and "weights_work_check: OK".
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <string>
#include <vector>

#include "../../cu-roaring-bitmap_amd/csrc/weights_work.hpp"

using namespace crimpl;

static int g_errors = 0;
static std::map<std::string, int> g_ways;

#define EXPECT(ok, ...)                              \
    do {                                             \
        if (!(ok) && ++g_errors < 20) {              \
            printf("%s:%d: %s: ", __FILE__, __LINE__, #ok); \
            printf(__VA_ARGS__);                     \
            printf("\n");                            \
        }                                            \
    } while (0)

static std::string text(const WeightsShape& a)
{
    char s[256];
    snprintf(s, sizeof s, "%u tokens, %u/%u heads of %u, %u requests, room %llu, max_new %u, max_kv %u, some %d", a.n_tokens,
             a.heads, a.kv_heads, a.dim, a.n_requests, static_cast<unsigned long long>(a.room), a.max_new, a.max_kv, a.some);
    return s;
}

constexpr uint64_t LAUNCH = 1ull << 23;  // workgroups of 512 threads or fewer

static void check(const WeightsShape& a, std::mt19937_64& rng)
{
    const WeightsWork w = weights_work(a);
    const std::string what = text(a);
    const uint32_t group = a.heads / a.kv_heads;
    EXPECT(!(w.many && w.mixed), "%s", what.c_str());
    if (!w.many) {
        EXPECT(w.rows_grid && w.rows_grid < LAUNCH && w.rows_grid == static_cast<uint64_t>(w.spans) * a.n_requests, "%s", what.c_str());
        EXPECT(w.head_waves && WR_WAVES % w.head_waves == 0 && w.halves && w.halves * row_cols(a.dim) <= 64, "%s", what.c_str());
        EXPECT(w.sums == 0 || w.mixed, "%s", what.c_str());
    }
    if (w.many || w.mixed) {
        EXPECT(w.tiles_grid && w.tiles_grid < LAUNCH, "%s", what.c_str());
        EXPECT(w.part_rows >= 64 && w.part_rows % 64 == 0, "%s: %u", what.c_str(), w.part_rows);
        EXPECT(w.join_per_request && w.join_side && static_cast<uint64_t>(w.join_per_request) * w.join_side < LAUNCH * 2, "%s", what.c_str());
    }
    EXPECT(w.sums <= WT_SUMS, "%s: %llu", what.c_str(), static_cast<unsigned long long>(w.sums));
    if (w.many || w.mixed) EXPECT(w.side && w.side <= w.parts, "%s", what.c_str());
    if (w.many) {
        EXPECT(w.batch && w.batch <= a.n_requests, "%s", what.c_str());
        EXPECT(w.tiles_grid == static_cast<uint64_t>(w.side) * w.batch * w.tiles * a.kv_heads, "%s", what.c_str());
        EXPECT(w.sums == static_cast<uint64_t>(w.side) * w.batch * a.kv_heads * a.room, "%s", what.c_str());
    }
    if (w.mixed) {
        EXPECT(w.tiles_grid == static_cast<uint64_t>(w.side) * w.tiles * a.kv_heads, "%s", what.c_str());
        EXPECT(w.sums == static_cast<uint64_t>(w.side) * a.kv_heads * a.room, "%s", what.c_str());
        // the parts of requests that share the tokens in any way, of which none has more than the caller says
        for (int way = 0; way < 4; ++way) {
            uint64_t left = a.n_tokens, parts = 0;
            const uint64_t each = way == 0 ? w.few / group + 1 : way == 1 ? left : way == 2 ? w.part_rows / group + 1 : 0;
            for (uint32_t r = 0; r < a.n_requests && left; ++r) {
                uint64_t n = std::min<uint64_t>(left, each ? each : 1 + rng() % (left / 3 + 1));
                if (a.max_new) n = std::min<uint64_t>(n, a.max_new);
                left -= n;
                const uint64_t rows = n * group;
                if (rows > w.few) parts += (rows + w.part_rows - 1) / w.part_rows;
            }
            EXPECT(parts <= w.parts, "%s: %llu parts, %u listed", what.c_str(), static_cast<unsigned long long>(parts), w.parts);
        }
    }
    ++g_ways[w.many ? "many rows" : w.mixed ? "mixed" : "few rows"];
    if (w.many && w.batch < a.n_requests) ++g_ways["many rows, some requests at a time"];
    if (w.many && w.side < w.parts) ++g_ways["many rows, some parts at a time"];
    if (w.mixed && w.side < w.parts) ++g_ways["mixed, some parts at a time"];
}

int main()
{
    std::mt19937_64 rng(1);
    auto spread = [&](uint64_t lo, uint64_t hi) {  // evenly over the logarithm
        const double x = std::uniform_real_distribution<double>(0, 1)(rng);
        return static_cast<uint64_t>(static_cast<double>(lo) * __builtin_pow(static_cast<double>(hi) / static_cast<double>(lo), x));
    };
    const uint32_t dims[] = {64, 96, 128, 192, 256};
    // answered with hints as without
    check({524288, 32, 8, 128, 1, 524288, 0, 0, false, 256}, rng);
    check({524288, 32, 8, 128, 1, 524288, 524288, 524288, false, 256}, rng);
    check({512 * 2048, 32, 8, 128, 512, 131072, 2048, 131072, false, 256}, rng);
    check({4096, 32, 8, 128, 4096, 131072, 1, 0, false, 256}, rng);
    check({4096, 32, 8, 128, 4096, 131072, 1, 131072, false, 256}, rng);
    // a prompt's last tokens, or some of each request's, in a q that holds all: one part of rows
    for (bool some : {false, true}) {
        const WeightsShape last{131072, 32, 8, 128, 1, 131072, 64, 0, some, 256};
        const WeightsShape each{131072, 32, 8, 128, 8, 32768, 100, 32768, some, 256};
        check(last, rng);
        check(each, rng);
        EXPECT(weights_work(last).sums <= last.kv_heads * last.room, "%s: %llu", text(last).c_str(),
               static_cast<unsigned long long>(weights_work(last).sums));
        EXPECT(weights_work(each).sums <= 8 * 2 * each.kv_heads * each.room, "%s: %llu", text(each).c_str(),
               static_cast<unsigned long long>(weights_work(each).sums));
    }
    // long prompts, alone and among single tokens in wide tables
    check({131072, 32, 8, 128, 1, 131072, 131072, 131072, false, 256}, rng);
    check({1 << 21, 32, 8, 128, 1, 1 << 21, 0, 0, false, 256}, rng);
    check({4096 + 1023, 64, 8, 128, 1024, 131072, 4096, 0, false, 256}, rng);
    for (int i = 0; i < 200000; ++i) {
        WeightsShape a{};
        a.kv_heads = i % 7 ? 1u << rng() % 7 : static_cast<uint32_t>(spread(1, 65535));
        a.heads = a.kv_heads * static_cast<uint32_t>(1 + rng() % std::min<uint32_t>(8, 65535 / a.kv_heads));
        a.dim = dims[rng() % 5];
        a.n_requests = static_cast<uint32_t>(spread(1, i % 3 ? 3000 : (1 << 22) - 1));
        a.room = spread(1, i % 5 ? 1 << 20 : (1u << 31) - 1);
        a.n_tokens = static_cast<uint32_t>(std::min<uint64_t>(spread(1, 1 << 24), ((1ull << 31) - 1) / a.heads));
        if (rng() % 2) a.max_new = static_cast<uint32_t>(std::max<uint64_t>((a.n_tokens + a.n_requests - 1) / a.n_requests, spread(1, a.n_tokens)));
        if (rng() % 2) a.max_kv = static_cast<uint32_t>(spread(1, a.room));
        a.some = rng() % 4 == 0;
        a.cus = 256;
        check(a, rng);
    }
    for (const auto& [way, times] : g_ways) printf("%s: %d\n", way.c_str(), times);
    for (const char* way : {"many rows", "mixed", "few rows", "many rows, some requests at a time", "many rows, some parts at a time",
                            "mixed, some parts at a time"}) EXPECT(g_ways.count(way), "\"%s\" was not taken", way);
    if (g_errors) {
        printf("weights_work_check: %d errors\n", g_errors);
        return 1;
    }
    printf("weights_work_check: OK\n");
    return 0;
}

// The numbering of paged attention's work (csrc/attention_work.hpp) run on the CPU:
// 64 lanes of a wave as contexts that take turns at each exchange between lanes.
// For every workgroup number that the host sizes a launch for:
//   - entries of the ranges' table are written inside it, whatever the arrays hold;
//   - the workgroups answer each tile of rows once, over ranges that make up all keys;
//   - the join finds those ranges for every token and head.
// Prints how often each way to number was taken, and "attention_work_check: OK".
#include <setjmp.h>
#include <ucontext.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <string>
#include <vector>

// ---- a wave ----------------------------------------------------------------------
constexpr uint32_t LANES = 64;
static uint32_t g_lane, g_running;
static uint64_t g_slot[2][LANES];
static uint32_t g_phase[LANES];
static jmp_buf g_jump[LANES];
static ucontext_t g_start[LANES], g_main;
static bool g_begun[LANES];
static std::vector<char> g_stack[LANES];
static void (*g_body)();

static void resume(uint32_t lane)
{
    g_lane = lane;
    if (g_begun[lane]) _longjmp(g_jump[lane], 1);
    g_begun[lane] = true;
    setcontext(&g_start[lane]);
}

// The next lane's turn; this one goes on when all have come as far.
static void turn()
{
    const uint32_t me = g_lane;
    if (_setjmp(g_jump[me]) == 0) resume((me + 1) % LANES);
}

static void lane_main()
{
    g_body();
    // every lane leaves after the same exchange, in order
    if (--g_running == 0) setcontext(&g_main);
    resume((g_lane + 1) % LANES);
}

static void run_wave(void (*body)())
{
    g_body = body;
    g_running = LANES;
    for (uint32_t i = 0; i < LANES; ++i) {
        g_begun[i] = false;
        g_phase[i] = 0;
        g_stack[i].resize(1 << 16);
        getcontext(&g_start[i]);
        g_start[i].uc_stack.ss_sp = g_stack[i].data();
        g_start[i].uc_stack.ss_size = g_stack[i].size();
        g_start[i].uc_link = nullptr;
        makecontext(&g_start[i], lane_main, 0);
    }
    volatile bool back = false;
    getcontext(&g_main);
    if (back) return;
    back = true;
    resume(0);
}

// Every lane's value, in the lane that asks.
static const uint64_t* exchange(uint64_t mine)
{
    const uint32_t p = g_phase[g_lane]++ & 1u;
    g_slot[p][g_lane] = mine;
    turn();
    return g_slot[p];
}

struct Index {
    operator uint32_t() const { return g_lane; }
};
static struct {
    Index x;
} threadIdx;
struct uint2 {
    uint32_t x, y;
};
static uint2 make_uint2(uint32_t x, uint32_t y) { return {x, y}; }
static uint32_t __lane_id() { return g_lane; }
static uint64_t __ballot(bool b)
{
    const uint64_t* v = exchange(b);
    uint64_t m = 0;
    for (uint32_t i = 0; i < LANES; ++i) m |= (v[i] & 1ull) << i;
    return m;
}
template <class T>
static T __shfl_xor(T v, int o, int)
{
    return static_cast<T>(exchange(static_cast<uint64_t>(v))[g_lane ^ static_cast<uint32_t>(o)]);
}
static int read_lane(int v, int lane) { return static_cast<int>(exchange(static_cast<uint32_t>(v))[lane & 63]); }
static int __popcll(uint64_t x) { return __builtin_popcountll(x); }
static int __ffsll(unsigned long long x) { return __builtin_ffsll(static_cast<long long>(x)); }
static int __clz(int x) { return x ? __builtin_clz(static_cast<unsigned>(x)) : 32; }
static void atomicAdd(uint32_t* p, uint32_t v) { *p += v; }
using std::max;
using std::min;
#define __device__
#define __forceinline__ inline
#define __shared__ static
#define __builtin_amdgcn_readlane read_lane
namespace crimpl {
static void wave_lds_fence() { exchange(0); }
static uint32_t wave_incl_scan(uint32_t v)
{
    const uint64_t* x = exchange(v);
    uint32_t sum = 0;
    for (uint32_t i = 0; i <= g_lane; ++i) sum += static_cast<uint32_t>(x[i]);
    return sum;
}
}  // namespace crimpl
#include "../../cu-roaring-bitmap_amd/csrc/attention_work.hpp"

using namespace crimpl;

// ---- the check ---------------------------------------------------------------------
static AttnArgs g_a;
static uint32_t g_id, g_most, g_kind, g_token, g_head;
static Work g_work[LANES];
static Joined g_joined[LANES];

static void work_body()
{
    g_work[g_lane] = g_kind == 0   ? find_work<false, true>(g_a, g_id, g_most)    // at_rows
                     : g_kind == 1 ? find_work<true, false>(g_a, g_id, g_most)    // at_tiles, up to 128 dimensions
                                   : find_work<false, false>(g_a, g_id, g_most);  // and above
}
static void join_body() { g_joined[g_lane] = find_joined(g_a, g_token, g_head, g_most); }

static int g_errors;
#define EXPECT(cond, ...)                               \
    do {                                                \
        if (!(cond) && ++g_errors <= 20) {              \
            printf("FAILED %s: ", #cond);               \
            printf(__VA_ARGS__);                        \
            printf("\n");                               \
            fflush(stdout);                             \
        }                                               \
    } while (0)

struct Case {
    std::vector<int32_t> starts, kv_len;
    uint32_t n_tokens, heads, kv_heads, dim, page_lg, cols, max_new, max_kv;
    bool sound;  // offsets ascend and lengths are not negative
};
static std::map<std::string, int> g_ways;

static void check(const Case& c)
{
    g_a = AttnArgs{};
    g_a.n_tokens = c.n_tokens;
    g_a.heads = c.heads;
    g_a.kv_heads = c.kv_heads;
    g_a.dim = c.dim;
    g_a.n_requests = static_cast<uint32_t>(c.kv_len.size());
    g_a.page_lg = c.page_lg;
    g_a.cols = c.cols;
    g_a.starts = c.starts.data();
    g_a.kv_len = c.kv_len.data();
    uint32_t rows_a_wave = 0;
    if (!size_launch(g_a, static_cast<uint64_t>(c.cols) << c.page_lg, c.max_new, c.max_kv, 256, &rows_a_wave)) return;
    g_most = rows_a_wave ? 16 * rows_a_wave : 128;
    g_kind = rows_a_wave ? 0 : c.dim <= 128 ? 1 : 2;
    const uint32_t group = c.heads / c.kv_heads, n = g_a.n_requests + 2;
    const uint64_t room = static_cast<uint64_t>(c.cols) << c.page_lg;
    // entries of no meaning, inside the table and as far behind it as a number can reach
    const uint2 none = {0xABCD1234u, 0x87654321u};
    std::vector<uint2> table(g_a.n_tiles + g_a.n_ranges + 64, none);
    g_a.ranges = table.data();
    struct Piece {
        uint32_t k0, k1, id;
        bool whole;
    };
    std::map<std::pair<int32_t, uint32_t>, std::vector<Piece>> tiles;  // (first token, first row) of a segment
    bool any_cut = false;
    for (g_id = 0; g_id < g_a.n_ranges; ++g_id) {
        run_wave(work_body);
        const Work w = g_work[0];
        for (uint32_t i = 1; i < LANES; ++i)
            EXPECT(g_work[i].none == w.none && (w.none || (g_work[i].row0 == w.row0 && g_work[i].k0 == w.k0 &&
                                                           g_work[i].token0 == w.token0)),
                   "lane %u differs, id %u", i, g_id);
        if (w.none) continue;
        EXPECT(w.range == g_id && w.row0 < w.rows && w.rows == w.tokens * group && w.keys <= room, "id %u", g_id);
        EXPECT(w.token0 >= 0 && static_cast<uint64_t>(w.token0) + w.tokens <= c.n_tokens, "id %u", g_id);
        EXPECT(w.k1 <= w.keys && (!w.whole || (w.k0 == 0 && w.k1 == w.keys)), "id %u", g_id);
        tiles[{w.token0, w.row0}].push_back({w.k0, w.k1, g_id, w.whole});
        any_cut |= !w.whole;
    }
    for (size_t i = g_a.n_tiles; i < table.size(); ++i)
        EXPECT(table[i].x == none.x && table[i].y == none.y,
               "entry %zu of %u written: %u requests, %u tokens, %u heads over %u, share %u", i, g_a.n_tiles,
               g_a.n_requests, c.n_tokens, c.heads, c.kv_heads, g_a.share);
    g_ways[std::string(g_kind == 0 ? "rows" : g_kind == 1 ? "tiles" : "tiles of long rows") + (n > 64 ? ", many" : ", few") +
           (n > FIND_SORTED ? " more" : "") +
           (!g_a.share ? ", uncut" : g_a.if_uneven ? any_cut ? ", uneven, cut" : ", uneven, left" : ", cut")] += 1;
    if (!c.sound) return;
    for (uint32_t i = 0; i < n; ++i) {
        const int32_t from = segment_start(g_a, i), to = segment_start(g_a, i + 1);
        int32_t said;
        const uint32_t keys = segment_keys(g_a, i, said);
        const uint32_t rows = static_cast<uint32_t>(to - from) * group;
        for (uint32_t row0 = 0; row0 < rows; row0 += g_most) {
            auto at = tiles.find({from, row0});
            EXPECT(at != tiles.end(), "segment %u, row %u: nobody's", i, row0);
            if (at == tiles.end()) continue;
            const auto& p = at->second;
            uint32_t upto = 0;
            for (size_t x = 0; x < p.size(); ++x) {
                EXPECT(p[x].id == p[0].id + x && p[x].whole == (p.size() == 1), "segment %u, row %u", i, row0);
                EXPECT(p[x].k0 == upto || p[x].k0 >= p[x].k1, "segment %u, row %u: keys from %u, not %u", i, row0,
                       p[x].k0, upto);
                upto = max(upto, p[x].k0 < p[x].k1 ? p[x].k1 : 0u);
            }
            EXPECT(upto == keys, "segment %u, row %u: %u of %u keys", i, row0, upto, keys);
            if (g_a.share) {  // as the join sees the tile's first and last row
                for (uint32_t row : {row0, min(row0 + g_most, rows) - 1}) {
                    g_token = static_cast<uint32_t>(from) + row / group;
                    for (uint32_t kh = 0; kh < c.kv_heads; kh += max(1u, c.kv_heads - 1)) {
                        g_head = kh * group + row % group;
                        run_wave(join_body);
                        const Joined j = g_joined[0];
                        EXPECT(j.row == row - row0 && j.first == p[0].id && j.count == (p.size() == 1 ? 0 : p.size()),
                               "segment %u, row %u: joins %u from %u, not %zu from %u", i, row, j.count, j.first,
                               p.size(), p[0].id);
                    }
                }
            }
            tiles.erase(at);
        }
    }
    EXPECT(tiles.empty(), "%zu tiles that are nobody's rows", tiles.size());
}

// `requests` of `new_each` tokens and `kv` keys; uneven: every fourth has them all, the others a few.
static Case even(uint32_t requests, uint32_t new_each, uint32_t kv, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                 bool uneven = false)
{
    Case c{{0}, {}, 0, heads, kv_heads, dim, 4, (kv + 15) / 16, new_each, kv, true};
    for (uint32_t r = 0; r < requests; ++r) {
        c.n_tokens += new_each;
        c.starts.push_back(static_cast<int32_t>(c.n_tokens));
        c.kv_len.push_back(static_cast<int32_t>(!uneven || r % 16 == 3 ? kv : max(new_each, kv / 32)));
    }
    return c;
}

int main()
{
    std::mt19937 rng(1);
    auto pick = [&](uint32_t lo, uint32_t hi) { return lo + static_cast<uint32_t>(rng() % (hi - lo + 1)); };
    // tiles that fill more than half of the card, of more requests than a wave has lanes
    for (bool uneven : {false, true}) {
        check(even(100, 16, 4096, 16, 4, 128, uneven));
        check(even(64, 64, 8192, 16, 8, 128, uneven));
        check(even(64, 16, 8192, 32, 8, 128, uneven));
        check(even(63, 33, 4500, 16, 8, 64, uneven));
        check(even(62, 33, 4500, 16, 8, 64, uneven));
        check(even(300, 40, 5000, 1, 1, 96, uneven));
        check(even(70, 40, 5000, 2, 1, 128, uneven));
    }
    for (int i = 0; i < 160; ++i) {
        const uint32_t requests = i % 4 == 0 ? pick(0, 5) : i % 4 == 1 ? pick(60, 66) : i % 4 == 2 ? pick(100, 135) : pick(1, 300);
        const uint32_t kv_heads = 1u << pick(0, 4), group = pick(1, 5);
        const uint32_t dims[] = {64, 96, 128, 192, 256}, most_new = i % 3 == 0 ? 1 : pick(2, i % 3 == 1 ? 12 : 150);
        const uint32_t most_kv = pick(0, 1) ? pick(1, 3000) : pick(4096, 20000);
        Case c{{0}, {}, 0, kv_heads * group, kv_heads, dims[pick(0, 4)], pick(0, 7), 0, 0, 0, i % 5 != 4};
        for (uint32_t r = 0; r < requests; ++r) {
            c.n_tokens += pick(0, 7) ? pick(1, most_new) : 0;
            c.starts.push_back(static_cast<int32_t>(c.n_tokens));
            c.kv_len.push_back(static_cast<int32_t>(pick(0, 9) ? pick(1, most_kv) : pick(0, 1) ? most_kv : 0));
        }
        c.n_tokens += pick(0, 3) ? 0 : pick(0, 40);  // some behind all requests
        c.cols = (most_kv >> c.page_lg) + 1;
        if (pick(0, 1)) c.max_new = most_new, c.max_kv = most_kv;
        if (!c.sound) {
            for (auto& x : c.starts) x = pick(0, 1) ? static_cast<int32_t>(rng()) : static_cast<int32_t>(pick(0, c.n_tokens + 9));
            for (auto& x : c.kv_len) x = pick(0, 1) ? static_cast<int32_t>(rng()) : static_cast<int32_t>(most_kv);
            if (i % 2) std::sort(c.starts.rbegin(), c.starts.rend());
        }
        check(c);
    }
    for (const auto& [way, times] : g_ways) printf("%s: %d\n", way.c_str(), times);
    for (const char* way : {"rows, few, cut", "rows, many, cut", "rows, few, uncut", "rows, many, uncut", "rows, many more, uncut",
                            "tiles, few, cut", "tiles, many, uneven, left", "tiles, many, uneven, cut",
                            "tiles, few, uneven, left", "tiles, many more, uneven, left", "tiles, many, uncut"})
        EXPECT(g_ways.count(way), "\"%s\" was not taken", way);
    if (g_errors) {
        printf("attention_work_check: %d errors\n", g_errors);
        return 1;
    }
    printf("attention_work_check: OK\n");
    return 0;
}

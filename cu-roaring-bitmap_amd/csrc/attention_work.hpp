// How the work of cr_paged_attention is numbered: the launch that the host sizes and
// the tile of rows and range of keys that a workgroup's number stands for, found on
// the device from its own lengths.  Included by attention.hip, behind
// internal.hpp, and by a check that runs it on the CPU.
#pragma once
#include <algorithm>
#include <cstdint>

namespace crimpl {

namespace {

struct AttnArgs {
    const uint16_t* q;
    uint64_t q_token, q_head;
    uint16_t* out;
    uint64_t out_token, out_head;
    float* lse;
    uint32_t n_tokens, heads, kv_heads, dim, n_requests;
    const uint16_t* k;
    const uint16_t* v;
    uint64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
    uint32_t n_pages, page_lg;
    const int32_t* starts;
    const int32_t* kv_len;
    const int32_t* table;
    uint32_t cols;
    uint64_t table_stride;
    const int32_t* sel;
    uint64_t sel_stride;
    const int32_t* sel_len;
    const int32_t* limits;
    float scale;
    uint32_t causal;
    // The launch.  With `share` 0, a workgroup takes a tile of rows and all of its
    // keys.  Otherwise the tiles' keys are cut into about `share` ranges of even
    // length, a workgroup each for every key head; their results, in fp32, are
    // joined by another kernel.
    uint32_t n_tiles, n_ranges;
    uint32_t share, step, least_len;  // ranges are of a multiple of `step` keys, at least least_len
    uint32_t if_uneven;               // cut only if the longest tile has 2.5 times the keys of such a range
    uint2* ranges;    // [n_tiles] a tile's first range and how many it has
    float* part_o;    // [ranges][key heads][rows of a tile][dim]
    float* part_lse;  // [ranges][key heads][rows of a tile], base 2
};

// Keys that a wave of the kernel of few rows takes at a time, and its waves.
constexpr int DC_NT = 256;
constexpr uint32_t DC_WAVES = DC_NT / 64;
constexpr uint32_t DC_KEYS = 32;

// Sizes the launch for a call whose tensors stand in `a`: n_tiles, share, if_uneven,
// step, least_len and n_ranges, the workgroups of each key head.  room: positions of a
// table's row; max_new, max_kv: the caller's, 0 where it does not know; rows_a_wave:
// blocks of 16 rows (at_rows), or 0 for tiles of 128 (at_tiles).  False: too many rows.
inline bool size_launch(AttnArgs& a, uint64_t room, uint32_t max_new, uint32_t max_kv, uint32_t cus,
                        uint32_t* rows_a_wave)
{
    // Rows of a request that share a key head, as far as the caller says.
    const uint32_t group = a.heads / a.kv_heads;
    const uint64_t requests = std::max(1u, a.n_requests);
    const uint64_t typical = max_new ? max_new : (a.n_tokens + requests - 1) / requests;
    const uint64_t rows = typical * group;
    // blocks of 16 rows (two of long rows do not fit the registers), or tiles
    const uint32_t per_wave = rows <= 16 ? 1 : rows <= 32 && a.dim <= 128 ? 2 : 0;
    const uint32_t most = per_wave ? 16 * per_wave : 128;
    const uint64_t tiles = static_cast<uint64_t>(a.n_tokens) * group / most + a.n_requests + 2;
    const uint64_t all_rows = static_cast<uint64_t>(a.n_tokens) * a.heads;
    // a launch holds fewer than 2^32 threads
    if ((tiles * a.kv_heads) >> 23 || all_rows >> 31) return false;
    a.n_tiles = static_cast<uint32_t>(tiles);
    // Few tiles are cut into ranges of even length, as many as the card holds
    // workgroups at once (4 requests of 32768 keys, 128 dimensions: 2 workgroups a
    // CU 94 us, 3 109, 1 103).  More of them, or requests long enough to lag behind
    // the others, into about four rounds of workgroups, of no short ranges (64 of
    // up to 16384 keys: uncut 398 us, two rounds 348, four 338, twelve 370); else
    // reading the lengths and joining cost more than they even out (256 of up to
    // 1024 keys: uncut 110 us, cut 160; of up to 4096 372 and 389; 48 of up to 2048
    // with 16 heads of 64 dimensions 53 and 60).
    // `held`, the workgroups that the card holds at once, is that of one block of rows a
    // wave.  Of two, a CU holds one less (two up to 64 dimensions, one above), so that
    // theirs run in about two rounds.  Counted as they are, 8 tokens of 8192 keys would
    // take 20 us instead of 32 and 64 requests of 8 of 4096 239 instead of 262, but 20
    // of 6 of 30000 456 instead of 397 (32 heads over 8, 128 dimensions).
    const uint64_t tiles_in_all = (rows + most - 1) / most * requests;
    const uint64_t longest = std::min<uint64_t>(room, max_kv ? max_kv : room);
    const uint32_t on_a_cu = per_wave && a.dim <= 64 ? 3 : a.dim <= (per_wave ? 128 : 192) ? 2 : 1;
    const uint64_t held = on_a_cu * cus / a.kv_heads + 1;
    bool few = 2 * tiles_in_all <= held;
    // Tiles of 128 rows leave as much to join however many keys they see, so that
    // cutting has to shorten the longest by about 800 keys (one request, 256 tokens
    // of 1024 uncut 33 us, cut 29; 600 of 2048 60 and 52; 1000 of 4096 111 and 102;
    // but 512 of 512 23 and 29; 1024 of 1024 38 and 48; 16 of 64 of 1024 36.5 and 37.2).
    if (!per_wave) few = few && longest * (held - tiles_in_all) > 800 * held;
    const bool long_ones = per_wave && longest >= 4096 && tiles_in_all <= (longest >= 16384 ? 16 : 2) * held;
    // Tiles for more than half of the card, but perhaps of requests so uneven that the
    // longest would be waited for: the device looks at the lengths (5 of 1924 tokens
    // of up to 42670, 4 heads: uncut 955 us, cut 410; 16 of 100 of 4096 104 and 83).
    // With more tiles it costs more than it gains: rows to be joined, and ranges in
    // the requests' order where uncut tiles go longest first (8 of 1000 of 8192, 192
    // tiles for 65 places: 179 and 201).
    const bool uneven =
        !per_wave && !few && a.n_requests > 1 && a.dim <= 128 && longest >= 4096 && tiles_in_all <= held;
    const bool cut = (few || long_ones || uneven) && all_rows >> 24 == 0;
    a.if_uneven = uneven;
    a.step = per_wave ? DC_KEYS * DC_WAVES : 64;
    a.least_len = !few ? 1024 : per_wave ? DC_KEYS * DC_WAVES : 256;
    uint64_t ranges = tiles;
    if (cut && longest > a.least_len) {
        a.share = static_cast<uint32_t>(few ? held - tiles_in_all : uneven ? held : 4 * held);
        ranges += a.share;
    }
    a.n_ranges = static_cast<uint32_t>(ranges);
    *rows_a_wave = per_wave;
    return true;
}

// Segment i of the tokens: request i - 1's; the first and the last one hold
// those before and behind all requests, which see nothing.
__device__ __forceinline__ int32_t segment_start(const AttnArgs& a, uint32_t i)
{
    if (i == 0) return 0;
    if (i > a.n_requests + 1) return static_cast<int32_t>(a.n_tokens);
    return min(max(a.starts[i - 1], 0), static_cast<int32_t>(a.n_tokens));
}

// How many keys a segment's request has; `n`: what its length says.
__device__ __forceinline__ uint32_t segment_keys(const AttnArgs& a, uint32_t i, int32_t& n)
{
    n = 0;
    if (i == 0 || i > a.n_requests) return 0;
    n = a.sel ? a.sel_len[i - 1] : a.kv_len[i - 1];
    // (Not `n <= 0 ? 0 : min(room, n)`: the compiler moves the min before the test and then takes n for positive.)
    return static_cast<uint32_t>(min(static_cast<uint64_t>(a.cols) << a.page_lg, static_cast<uint64_t>(max(n, 0))));
}

// Segment i's tiles of `most` rows are numbered from here, which leaves each
// segment room for all of its rows.
__device__ __forceinline__ uint32_t tile_base(uint32_t i, int32_t start, uint32_t group, uint32_t most)
{
    return static_cast<uint32_t>(static_cast<uint64_t>(static_cast<uint32_t>(start)) * group / most) + i;
}

// A workgroup's work: a tile of rows of a segment (row m is token m / group,
// head m % group of those that share a key head) and a range of its keys.
struct Work {
    uint32_t request;
    bool real;            // a request's, not the tokens' outside
    int32_t token0;       // the segment's first token
    uint32_t tokens;
    uint32_t row0, rows;  // rows [row0, rows) are this tile's and those behind it
    uint32_t keys;        // the request's
    int32_t len;          // what its length says
    uint32_t k0, k1;      // the range
    uint32_t range;       // its number
    bool whole;           // the tile's only range: its results need not be joined
    bool none;            // nothing to do
};

__device__ __forceinline__ uint32_t lane_value(uint32_t x, uint32_t lane)
{
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), static_cast<int>(lane)));
}

// Up to 128 requests of few rows are put in order, too: 128 of up to 2000 keys 62 ->
// 55 us, 79 of up to 790 39.6 -> 36.7.  More of them would cost more than it evens
// out (256 of up to 1024 102 -> 116), and so do tiles (106 of 429 tokens 460 -> 485).
constexpr uint32_t FIND_WAVES = 4, FIND_SORTED = 130;

// What the workgroup's number `id` stands for.  A wave looks at 64 segments at
// a time, each lane at one.
// IF_UNEVEN: it may be left to the lengths whether tiles are cut.  BY_CLASS: of more
// requests than lanes, too, those with many keys go first.
template <bool IF_UNEVEN, bool BY_CLASS>
__device__ __forceinline__ Work find_work(const AttnArgs& a, uint32_t id, uint32_t most)
{
    const uint32_t group = a.heads / a.kv_heads, n = a.n_requests + 2, lane = __lane_id();
    uint32_t lo = 0, start = 0, end = 0, keys = 0, tile = 0, count = 1, part = 0, at = 0;
    int32_t said = 0;
    bool cut = a.share != 0;
    uint64_t all = 0;
    if (cut) {
        uint32_t longest = 0;
#pragma unroll 2
        for (uint32_t i0 = 0; i0 < n; i0 += 64) {
            const uint32_t i = min(i0 + lane, n);
            start = static_cast<uint32_t>(segment_start(a, i));
            end = static_cast<uint32_t>(segment_start(a, i + 1));
            keys = segment_keys(a, i, said);
            const uint32_t rows = end > start ? (end - start) * group : 0u;
            all += static_cast<uint64_t>((rows + most - 1) / most) * keys;
            if (IF_UNEVEN) longest = max(longest, rows ? keys : 0u);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o, 64);
        if (IF_UNEVEN && a.if_uneven) {
#pragma unroll
            for (int o = 32; o > 0; o >>= 1)
                longest = max(longest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(longest), o, 64)));
            cut = static_cast<uint64_t>(longest) * a.share * 2 > all * 5;
        }
    }
    if (!cut) {
        if (n <= 64) {
            // the requests with the most keys go first, and of each its last rows, which see the most
            const uint32_t i = min(lane, n);
            start = static_cast<uint32_t>(segment_start(a, i));
            end = static_cast<uint32_t>(segment_start(a, i + 1));
            keys = segment_keys(a, i, said);
            const uint32_t rows = end > start ? (end - start) * group : 0u;
            const uint32_t mine = i < n ? (rows + most - 1) / most : 0u;
            uint32_t before = 0;
            for (uint32_t j0 = 0; j0 < n; j0 += 8) {  // (segments from n on have no tiles)
#pragma unroll
                for (uint32_t j = j0; j < j0 + 8; ++j) {
                    const uint32_t other = lane_value(keys, j), tiles = lane_value(mine, j);
                    // more keys, or as many and an earlier segment
                    const int32_t below = static_cast<int32_t>(keys) - (j < lane ? 1 : 0);
                    before += static_cast<int32_t>(other) > below ? tiles : 0u;
                }
            }
            const uint64_t here = __ballot(before <= id && id - before < mine);
            if (!here) {
                Work w{};
                w.none = true;
                return w;
            }
            at = lo = static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(here))) - 1;
            tile = lane_value(mine, at) - 1 - (id - lane_value(before, at));
        } else if (BY_CLASS && n <= FIND_SORTED) {
            // the same by classes of keys, two to a power of two: first the tiles of each,
            // then the request among those of the class that holds the id
            __shared__ uint32_t s_class[FIND_WAVES][64];
            uint32_t* sums = s_class[threadIdx.x >> 6];
            auto look = [&](uint32_t i0, uint32_t& mine) {
                const uint32_t i = min(i0 + lane, n);
                start = static_cast<uint32_t>(segment_start(a, i));
                end = static_cast<uint32_t>(segment_start(a, i + 1));
                keys = segment_keys(a, i, said);
                const uint32_t rows = end > start ? (end - start) * group : 0u;
                mine = i < n ? (rows + most - 1) / most : 0u;
                const uint32_t top = keys ? 31u - static_cast<uint32_t>(__clz(static_cast<int>(keys))) : 0u;
                return keys > 1 ? top * 2 + ((keys >> (top - 1)) & 1u) : keys;
            };
            sums[lane] = 0;
            wave_lds_fence();
            uint32_t mine;
#pragma unroll 2
            for (uint32_t i0 = 0; i0 < n; i0 += 64) {
                const uint32_t c = look(i0, mine);
                if (mine) atomicAdd(&sums[c], mine);
            }
            wave_lds_fence();
            const uint32_t of_class = sums[63u - lane], upto_class = wave_incl_scan(of_class);
            const uint64_t in = __ballot(upto_class > id);
            bool found = false;
            if (in) {
                const uint32_t first = static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(in))) - 1;
                const uint32_t rest = id - lane_value(upto_class - of_class, first);
                uint32_t before = 0;
                for (uint32_t i0 = 0; i0 < n && !found; i0 += 64) {
                    const uint32_t c = look(i0, mine);
                    mine = c == 63u - first ? mine : 0u;
                    const uint32_t upto = before + wave_incl_scan(mine);
                    const uint64_t past = __ballot(upto > rest);
                    if (past) {
                        at = static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(past))) - 1;
                        lo = i0 + at;
                        tile = lane_value(upto, at) - 1 - rest;  // the last rows first
                        found = true;
                    }
                    before = lane_value(upto, 63);
                }
            }
            if (!found) {
                Work w{};
                w.none = true;
                return w;
            }
        } else {
            for (uint32_t len = n; len > 64;) {  // base(lo) <= id < base(lo + len)
                const uint32_t step = (len + 63) / 64, i = lo + lane * step;
                const bool below = lane * step < len && tile_base(i, segment_start(a, i), group, most) <= id;
                const uint32_t from = (max(1u, static_cast<uint32_t>(__popcll(__ballot(below)))) - 1) * step;
                lo += from;
                len = min(step, len - from);
            }
            const uint32_t i = min(lo + lane, n);
            start = static_cast<uint32_t>(segment_start(a, i));
            end = static_cast<uint32_t>(segment_start(a, i + 1));
            keys = segment_keys(a, i, said);
            const uint32_t base = tile_base(i, static_cast<int32_t>(start), group, most);
            at = max(1u, static_cast<uint32_t>(__popcll(__ballot(lo + lane < n && base <= id)))) - 1;
            lo += at;
            tile = id - lane_value(base, at);
        }
    } else {
        // ranges of one length for all, so that about `share` of them result
        const uint64_t even = (all + a.share - 1) / a.share;
        const uint32_t len = max(a.least_len, static_cast<uint32_t>(min(even, static_cast<uint64_t>(0x7FFFFFFF))));
        uint32_t before = 0;
        bool found = false;
        for (uint32_t i0 = 0; i0 < n && !found; i0 += 64) {
            const uint32_t i = min(i0 + lane, n);
            if (n > 64) {
                start = static_cast<uint32_t>(segment_start(a, i));
                end = static_cast<uint32_t>(segment_start(a, i + 1));
                keys = segment_keys(a, i, said);
            }
            const uint32_t rows = end > start ? (end - start) * group : 0u;
            count = max(1u, (keys + len - 1) / len);
            const uint32_t mine = i < n ? (rows + most - 1) / most * count : 0u;
            const uint32_t upto = before + wave_incl_scan(mine);
            const uint64_t past = __ballot(upto > id);
            if (past) {
                at = static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(past))) - 1;
                lo = i0 + at;
                part = id - lane_value(upto - mine, at);
                count = lane_value(count, at);
                tile = part / count;
                part %= count;
                found = true;
            }
            before = lane_value(upto, 63);
        }
        if (!found) {
            Work w{};
            w.none = true;
            return w;
        }
    }
    Work w;
    w.real = lo > 0 && lo <= a.n_requests;
    w.request = w.real ? lo - 1 : 0;
    w.token0 = static_cast<int32_t>(lane_value(start, at));
    const uint32_t last = lane_value(end, at);
    w.tokens = last > static_cast<uint32_t>(w.token0) ? last - static_cast<uint32_t>(w.token0) : 0u;
    w.rows = w.tokens * group;
    w.row0 = tile * most;
    w.keys = lane_value(keys, at);
    w.len = static_cast<int32_t>(lane_value(static_cast<uint32_t>(said), at));
    w.none = w.row0 >= w.rows;
    w.range = id;
    w.whole = count == 1;
    const uint32_t even = ((w.keys + count - 1) / count + a.step - 1) / a.step * a.step;
    w.k0 = part * even;
    w.k1 = part + 1 == count ? w.keys : min(w.keys, w.k0 + even);
    // (A number behind the last segment's tiles has no entry: there are more numbers than entries.)
    if (a.share && part == 0 && !w.none && threadIdx.x == 0)
        a.ranges[tile_base(lo, w.token0, group, most) + tile] = make_uint2(id, count);
    return w;
}

// Which ranges hold a token's row, and where.
struct Joined {
    uint32_t first, count, row;  // `row` within the tile
};

__device__ __forceinline__ Joined find_joined(const AttnArgs& a, uint32_t token, uint32_t head, uint32_t most)
{
    const uint32_t group = a.heads / a.kv_heads, n = a.n_requests + 2, lane = __lane_id();
    // the token's segment: the last that starts at or before it
    uint32_t lo = 0, len = n, start = 0;
    while (true) {
        const uint32_t step = (len + 63) / 64, i = lo + min(lane * step, len);
        start = static_cast<uint32_t>(segment_start(a, i));
        const uint32_t at =
            max(1u, static_cast<uint32_t>(__popcll(__ballot(lane * step < len && start <= token)))) - 1;
        start = lane_value(start, at);
        lo += at * step;
        if (step == 1) break;
        len = min(step, len - at * step);
    }
    const uint32_t row = (token - start) * group + head % group;
    // (Offsets that do not ascend may lead to no tile's entry, but to none outside.)
    const uint32_t tile = min(tile_base(lo, static_cast<int32_t>(start), group, most) + row / most, a.n_tiles - 1);
    const uint2 range = a.ranges[tile];
    const uint32_t first = min(range.x, a.n_ranges);
    return {first, range.y == 1 ? 0u : min(range.y, a.n_ranges - first), row % most};
}

__device__ __forceinline__ uint64_t part_place(const AttnArgs& a, const Joined& j, uint32_t head, uint32_t most,
                                               uint32_t r)
{
    return (static_cast<uint64_t>(j.first + r) * a.kv_heads + head / (a.heads / a.kv_heads)) * most + j.row;
}

}  // namespace

}  // namespace crimpl

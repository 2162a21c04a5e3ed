// How the work of cr_paged_weights is split: which kernels take it, the sizes of their
// launches, and the sums that they leave for one another.  Included by weights.hip, and by
// a check that runs it on the CPU.
#pragma once
#include <algorithm>
#include <cstdint>

namespace crimpl {

namespace {

// Up to this many rows that share a key head in a request, wt_rows, whose products read their
// keys from LDS again for every 16 rows; wt_tiles keeps them in registers, but takes its time
// for few rows too.  us of either, 32 requests of 4096 positions and one of 16384, 8 key heads:
//   64 dimensions, 64 rows: 47 and 60, 13 and 12     128 rows: 71 and 66, 18 and 14
//   128, 48 rows: 75 and 86, 14 and 15               64 rows: 88 and 86, 17 and 15
//   256, 24 rows: 145 and 145, 24 and 21             16 rows: 114 and 145, 19 and 21
constexpr uint32_t few_rows(uint32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 48 : 24; }

// wt_rows: waves of a workgroup, a wave's LDS, and the positions that it holds the keys of.
constexpr int WR_NT = 256;
constexpr uint32_t WR_WAVES = WR_NT / 64;
constexpr uint32_t WR_BYTES = 8192;
constexpr uint32_t row_tiles(uint32_t chunks) { return WR_BYTES / (chunks * 16) / 16 > 4 ? 4 : WR_BYTES / (chunks * 16) / 16; }
constexpr uint32_t row_cols(uint32_t dim) { return row_tiles(dim <= 64 ? 8 : dim <= 128 ? 16 : 32) * 16; }

// wt_tiles: blocks of 32 positions whose keys a wave holds; positions of a workgroup's tile.
constexpr int WT_NT = 256;
constexpr uint32_t tile_blocks(uint32_t dim) { return dim <= 192 ? 2 : 1; }
constexpr uint32_t tile_cols(uint32_t dim) { return tile_blocks(dim) * 32 * (WT_NT / 64); }

struct WeightsShape {
    uint32_t n_tokens, heads, kv_heads, dim, n_requests;
    uint64_t room;             // positions of a table's row
    uint32_t max_new, max_kv;  // the caller's, 0 where it does not know
    bool some;                 // the caller says how many rows of each request count
    uint32_t cus;
};

struct WeightsWork {
    bool many;   // wt_tiles takes all requests; otherwise wt_rows does, or
    bool mixed;  // those of more than `few` rows go to wt_tiles, listed by a launch before
    uint32_t few;
    // wt_rows: waves that share the heads, how often a wave's LDS is filled with positions that it
    // looks up at once, and workgroups of a request.
    uint32_t head_waves, halves, spans, rows_grid;
    // wt_tiles: parts of a request's rows, of part_rows or more each (or, of listed requests, how many
    // parts there may be in all), and tiles of positions that a launch has for a request.  A launch
    // takes `batch` requests and `side` of their parts, or `side` of the list.
    uint32_t part_rows, parts, side, batch, tiles, tiles_grid;
    uint64_t sums;  // floats that a launch leaves for wt_join
    // wt_join: workgroups of a request, and requests at a time.
    uint32_t join_per_request, join_side;
};

// A launch holds fewer than 2^32 threads.  Workgroups come back for more positions where it does not
// hold one for all of them, so that the caller's hints never decide whether it is answered.
constexpr uint64_t WT_LAUNCH = (1u << 23) - 1;
// The sums of a launch of wt_tiles take at most 512 MB: every part of rows leaves one for each key head and
// each position that a table has room for.  More parts go launch after launch; where one takes more, wt_rows
// takes them all.  (8 key heads, tables of 131072 positions: 128 parts.)
constexpr uint64_t WT_SUMS = 1u << 27;

inline WeightsWork weights_work(const WeightsShape& a)
{
    WeightsWork w{};
    const uint64_t most = a.max_kv ? std::min<uint64_t>(a.room, a.max_kv) : a.room;
    // Rows of a request that share a key head, as far as the caller says.
    const uint32_t group = a.heads / a.kv_heads;
    // (q may hold more tokens than are counted: a prompt's last ones, with starts moved up to them)
    const uint64_t counted = a.max_new ? std::min<uint64_t>(a.n_tokens, static_cast<uint64_t>(a.max_new) * a.n_requests) : a.n_tokens;
    const uint64_t total = counted * group, mean = (total + a.n_requests - 1) / a.n_requests;
    w.few = few_rows(a.dim);
    const uint32_t cols = tile_cols(a.dim);
    w.tiles = static_cast<uint32_t>((most + cols - 1) / cols);
    const uint64_t longest = static_cast<uint64_t>(a.max_new) * group;
    const bool uneven = a.n_requests > 1 && !a.some;
    w.many = (uneven || !a.max_new ? mean : longest) > w.few;
    // Where requests have few rows on average, but one of them may have many (a prompt among single
    // tokens), each kernel takes its own kind, which a launch before lists.  One new token a request on
    // average is taken for single tokens.
    w.mixed = uneven && !w.many && total > 2 * w.few && (a.max_new ? longest > 2 * w.few : counted > a.n_requests);
    // Parts of the rows: as many workgroups as fill the card a few times, no longer sums than 2048
    // rows (in requests of the mean: a launch has as many parts of each), and no parts of fewer than
    // 256 where it can be helped, which end in more sums to be joined (32 requests of 100 tokens,
    // group 3: 39 us, with parts of 64 or 128 rows 44; a prompt of 500 18, not 15).
    const uint64_t even = total * w.tiles * a.kv_heads / (8ull * a.cus);
    w.part_rows = static_cast<uint32_t>(std::min<uint64_t>(2048, std::max<uint64_t>(256, even))) / 64 * 64;
    // A table may have room for far more positions than its requests hold, and a list for more parts than
    // there are.  Where the caller does not say how many positions there are, workgroups come back for
    // more of them instead of being launched for none (1024 requests of 500 positions in tables of 65536,
    // a prompt of 2048 among them: 320 us, not 1130; with max_kv 193).
    const uint64_t places = (a.max_kv ? 256ull : 64ull) * a.cus;
    auto at_most = [](uint64_t n, uint64_t most) { return std::max<uint64_t>(1, std::min(n, most)); };
    const uint64_t per = a.kv_heads * a.room, most_side = std::min(per ? WT_SUMS / per : WT_SUMS, WT_LAUNCH / a.kv_heads);
    w.many = w.many && most_side;
    w.mixed = w.mixed && most_side;
    if (w.mixed) {
        // A request counts as one of many rows from more rows on, where the list would have room for little
        // but requests of one part.
        const uint64_t full = total / w.part_rows + 1;
        if (full + std::min<uint64_t>(total / (w.few + 1), a.n_requests) > most_side)
            w.few = std::max(w.few, static_cast<uint32_t>(total / std::max(most_side, full)));
        const uint64_t listed = full + std::min<uint64_t>(total / (w.few + 1), a.n_requests);
        if (listed >> 20) {
            w.mixed = false;  // too long a list: wt_rows answers them all
        } else {
            w.parts = static_cast<uint32_t>(listed);
            w.side = static_cast<uint32_t>(std::min(listed, most_side));
            w.tiles = static_cast<uint32_t>(at_most(w.tiles, places / (static_cast<uint64_t>(w.side) * a.kv_heads)));
            w.tiles_grid = w.side * w.tiles * a.kv_heads;
            w.sums = w.side * per;
        }
    }
    if (w.many) {
        w.parts = static_cast<uint32_t>(std::max<uint64_t>(1, (mean + w.part_rows - 1) / w.part_rows));
        w.side = static_cast<uint32_t>(std::min<uint64_t>(w.parts, most_side));
        const uint64_t each = static_cast<uint64_t>(w.side) * a.kv_heads;  // workgroups of a request and a tile
        w.batch = static_cast<uint32_t>(std::min<uint64_t>(a.n_requests, most_side / w.side));
        if (!a.max_kv) w.tiles = static_cast<uint32_t>(at_most(w.tiles, places / (each * w.batch)));
        w.tiles = static_cast<uint32_t>(at_most(w.tiles, WT_LAUNCH / (each * w.batch)));
        w.tiles_grid = static_cast<uint32_t>(each * w.batch * w.tiles);
        w.sums = w.side * w.batch * per;
    } else {
        w.head_waves = a.kv_heads >= 3 ? 4 : a.kv_heads;
        // A wave looks up 64 positions at once and fills its LDS with them two or four times where there
        // is work for many rounds of the card, which saves look-ups (64 requests of 16384 positions, 8
        // heads of 128: 174 -> 167 us), and fills it once where the last round counts (32 requests of
        // 4096: 27 us, not 32).
        const uint32_t fill = WR_WAVES / w.head_waves * row_cols(a.dim);
        w.halves = row_cols(a.dim) <= 32 && most * a.n_requests > 16ull * a.cus * fill ? 64 / row_cols(a.dim) : 1;
        const uint32_t span = w.halves * fill;
        uint64_t spans = (most + span - 1) / span;
        if (!a.max_kv) spans = at_most(spans, places / a.n_requests);
        spans = at_most(spans, WT_LAUNCH / a.n_requests);
        w.spans = static_cast<uint32_t>(spans);
        w.rows_grid = static_cast<uint32_t>(spans * a.n_requests);
    }
    if (w.many || w.mixed) {
        // (fewer than 2^32 threads; of listed requests, which may be few or none, a few rounds of the card)
        const uint32_t requests = w.mixed ? std::min(w.parts, a.n_requests) : w.batch;
        uint64_t wanted = (most + 63) / 64;
        if (!a.max_kv) wanted = at_most(wanted, places / requests);
        w.join_per_request = static_cast<uint32_t>(std::min<uint64_t>(wanted, ((1u << 22) - 1) / (w.mixed ? 1u : requests)));
        w.join_side = w.mixed ? std::max(1u, std::min(requests, 8u * a.cus / w.join_per_request)) : requests;
    }
    return w;
}

}  // namespace

}  // namespace crimpl

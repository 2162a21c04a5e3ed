// Eviction from a paged cache, for serving language models (no reference
// implementation): which tokens of each request stay, by the attention weight that
// they got, and the moves that close the holes.
//
// Entry i of a request of L is safe if its slot is pinned, or if its position is one
// of the first `sinks` or the last `recent`.  With m = max(min(L, keep), safe ones),
// the m that come first by (safe, weight descending, i ascending) stay.  Holes among
// [0, m) are filled from [m, L) in order, so that sources and destinations never
// meet and every token in [0, m) that stays lies where it lay.
#include <algorithm>

#include "internal.hpp"
#include "set_bits.hpp"

namespace crimpl {

namespace {

constexpr int EV_NT = 1024;
constexpr uint32_t EV_WAVES = EV_NT / 64;
constexpr uint32_t EV_ROW = 256;       // entries that a wave takes at a time, four a lane
constexpr uint32_t EV_SAFE = 0xFFFFFFFFu;  // above the order of every weight
constexpr uint32_t EV_BINS = 2048;     // of a digit of 11 bits
constexpr uint32_t EV_COPIES = 4;      // of the first digit's counts

struct EvictArgs {
    const float* weights;
    uint64_t weights_stride;
    const int32_t* positions;  // or nullptr: an entry's place
    uint64_t positions_stride;
    const int32_t* kept;
    const int32_t* seen;
    const int32_t* kv_len;
    const int32_t* keep;
    const int32_t* table;
    uint32_t cols;
    uint64_t table_stride;
    uint32_t page_lg, n_pages, n_requests;
    uint32_t room;
    SetBits pinned;
    bool pins;
    uint32_t sinks, recent;
    float* weights_out;
    uint64_t weights_out_stride;
    int32_t* positions_out;
    uint64_t positions_out_stride;
    int32_t* len;
    int2* moves;
    uint64_t moves_stride;
    int32_t* n_moves;
    int32_t* freed;
    uint32_t freed_cap;
    int32_t* counts;
    uint32_t* keys;       // [n_requests][room rounded up to EV_ROW]
    uint32_t keys_stride;
};

__device__ __forceinline__ uint32_t request_len(const EvictArgs& a, uint32_t r)
{
    return static_cast<uint32_t>(min(max(a.kv_len[r], 0), static_cast<int32_t>(a.room)));
}

// Whole numbers in the order of the weights; NaN is the lowest, -0 counts as +0.
__device__ __forceinline__ uint32_t weight_order(float w)
{
    const uint32_t b = __float_as_uint(w + 0.0f);
    return w != w ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ int32_t slot_at(const EvictArgs& a, uint32_t r, uint32_t i)
{
    const uint32_t page = static_cast<uint32_t>(a.table[r * a.table_stride + (i >> a.page_lg)]);
    return page < a.n_pages ? static_cast<int32_t>((page << a.page_lg) + (i & ((1u << a.page_lg) - 1u))) : -1;
}

struct Ages {  // of a request's entries
    const int32_t* row;
    uint32_t kept;
    int64_t first;  // position of entry 0, were it one of the new ones
    int64_t sinks, recent;
    __device__ __forceinline__ Ages(const EvictArgs& a, uint32_t r, uint32_t len)
    {
        row = a.positions ? a.positions + r * a.positions_stride : nullptr;
        kept = a.positions ? static_cast<uint32_t>(min(max(a.kept[r], 0), static_cast<int32_t>(len))) : 0u;
        const int64_t seen = a.seen ? static_cast<int64_t>(a.seen[r]) : static_cast<int64_t>(len);
        first = seen - len;
        sinks = a.sinks;
        recent = seen - static_cast<int64_t>(a.recent);
    }
    __device__ __forceinline__ int64_t position(uint32_t i) const { return i < kept ? row[i] : first + i; }
    __device__ __forceinline__ bool safe(int64_t p) const { return p < sinks || p >= recent; }
};

__device__ __forceinline__ uint32_t lanes_below(unsigned long long m)
{
    const uint32_t lane = __lane_id();
    return static_cast<uint32_t>(__popcll(m & ((1ull << lane) - 1ull)));
}

// Finds the digit in which the n-th largest of the counted values lies (n >= 1, at
// most their number): counts are EV_BINS, the highest digit first taken.  Every
// thread gets the digit and how many values have a higher one.
__device__ __forceinline__ void find_digit(const uint32_t* s_bins, uint32_t copies, uint32_t n, uint32_t* s_scan,
                                           uint32_t* s_found, uint32_t& digit, uint32_t& above)
{
    constexpr uint32_t PER = EV_BINS / EV_NT;
    const uint32_t t = threadIdx.x;
    uint32_t c[PER], mine = 0, total;
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        const uint32_t bin = EV_BINS - 1 - (t * PER + j);
        c[j] = 0;
        for (uint32_t k = 0; k < copies; ++k) c[j] += s_bins[k * EV_BINS + bin];
        mine += c[j];
    }
    uint32_t before = block_excl_scan<EV_NT>(mine, s_scan, total);
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        if (before < n && n <= before + c[j]) {
            s_found[0] = EV_BINS - 1 - (t * PER + j);
            s_found[1] = before;
        }
        before += c[j];
    }
    __syncthreads();
    digit = s_found[0];
    above = s_found[1];
    __syncthreads();
}

// A workgroup a request.
__global__ __launch_bounds__(EV_NT) void ev_pick(EvictArgs a)
{
    __shared__ uint32_t s_bins[EV_COPIES * EV_BINS];
    __shared__ uint32_t s_scan[EV_WAVES], s_found[2], s_safe;
    const uint32_t r = blockIdx.x, t = threadIdx.x, lane = __lane_id(), wave = t >> 6;
    const uint32_t len = request_len(a, r);
    const uint32_t rows = (len + EV_ROW - 1) / EV_ROW, per_wave = (rows + EV_WAVES - 1) / EV_WAVES;
    const uint32_t row0 = min(wave * per_wave, rows), row1 = min(row0 + per_wave, rows);
    uint32_t* keys = a.keys + static_cast<uint64_t>(r) * a.keys_stride;
    const float* weights = a.weights + r * a.weights_stride;
    const Ages ages(a, r, len);
    const uint32_t keep = static_cast<uint32_t>(max(a.keep[r], 0));
    const bool all = keep >= len;
    for (uint32_t i = t; i < EV_COPIES * EV_BINS; i += EV_NT) s_bins[i] = 0;
    if (t == 0) s_safe = 0;
    __syncthreads();

    // Every entry's place in the order, and how many have each first digit.
    if (!all) {
        uint32_t n_safe = 0;
        for (uint32_t row = row0; row < row1; ++row) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t i = row * EV_ROW + j * 64 + lane;
                if (i >= len) continue;
                bool safe = ages.safe(ages.position(i));
                if (a.pins) {
                    const int32_t slot = slot_at(a, r, i);
                    if (slot >= 0 && static_cast<uint32_t>(slot) < a.pinned.end)
                        safe |= (a.pinned.word(static_cast<uint32_t>(slot) >> 5) >> (slot & 31)) & 1u;
                }
                const uint32_t key = safe ? EV_SAFE : weight_order(weights[i]);
                keys[i] = key;
                n_safe += safe ? 1u : 0u;
                if (!safe) atomicAdd(&s_bins[(wave % EV_COPIES) * EV_BINS + (key >> 21)], 1u);
            }
        }
        n_safe = wave_sum(n_safe);
        if (lane == 0) atomicAdd(&s_safe, n_safe);
    }
    __syncthreads();
    const uint32_t n_safe = s_safe;
    const uint32_t m = all ? len : max(keep, n_safe);
    // Of the others, the m - n_safe largest stay: those above `last`, and the first `ties` that equal it.
    uint32_t last = EV_SAFE, ties = 0;
    if (!all && m > n_safe) {
        uint32_t n = m - n_safe, digit, above, prefix;
        find_digit(s_bins, EV_COPIES, n, s_scan, s_found, digit, above);
        n -= above;
        prefix = digit << 21;
        for (int shift = 10; shift >= 0; shift -= 10) {
            const uint32_t bits = shift == 10 ? 11 : 10, mask = (1u << bits) - 1u;
            for (uint32_t i = t; i < EV_BINS; i += EV_NT) s_bins[i] = 0;
            __syncthreads();
            for (uint32_t row = row0; row < row1; ++row) {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const uint32_t i = row * EV_ROW + j * 64 + lane;
                    if (i >= len) continue;
                    const uint32_t key = keys[i];
                    if (key != EV_SAFE && (key >> (shift + bits)) == (prefix >> (shift + bits)))
                        atomicAdd(&s_bins[(key >> shift) & mask], 1u);
                }
            }
            __syncthreads();
            find_digit(s_bins, 1, n, s_scan, s_found, digit, above);
            n -= above;
            prefix |= digit << shift;
        }
        last = prefix;
        ties = n;
    }

    // Which stay, wave by wave over even parts of the row: ties first, then holes and movers.
    uint32_t tie0 = 0, hole0, move0, total;
    auto each = [&](auto f) {
        for (uint32_t row = row0; row < row1; ++row) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t i = row * EV_ROW + j * 64 + lane;
                f(i, i < len ? (all ? EV_SAFE : keys[i]) : 0u, i < len);
            }
        }
    };
    const bool tied = ties != 0;
    if (tied) {
        uint32_t n = 0;
        each([&](uint32_t, uint32_t key, bool in) { n += in && key == last ? 1u : 0u; });
        n = wave_sum(n);
        if (lane == 0) s_scan[wave] = n;
        __syncthreads();
        for (uint32_t w = 0; w < wave; ++w) tie0 += s_scan[w];
        __syncthreads();
    }
    auto stays = [&](uint32_t key, bool in, uint32_t& tie) {
        bool stay = in && (key > last || key == EV_SAFE);
        if (tied) {
            const bool eq = in && key == last;
            const unsigned long long same = __ballot(eq);
            stay |= eq && tie + lanes_below(same) < ties;
            tie += static_cast<uint32_t>(__popcll(same));
        }
        return stay;
    };
    {
        uint32_t holes = 0, movers = 0, tie = tie0;
        each([&](uint32_t i, uint32_t key, bool in) {
            const bool stay = stays(key, in, tie);
            holes += static_cast<uint32_t>(__popcll(__ballot(i < m && !stay)));
            movers += static_cast<uint32_t>(__popcll(__ballot(i >= m && stay)));
        });
        hole0 = move0 = total = 0;
        if (lane == 0) s_scan[wave] = holes | 0u;
        __syncthreads();
        for (uint32_t w = 0; w < EV_WAVES; ++w) {
            if (w < wave) hole0 += s_scan[w];
            total += s_scan[w];
        }
        __syncthreads();
        if (lane == 0) s_scan[wave] = movers;
        __syncthreads();
        for (uint32_t w = 0; w < wave; ++w) move0 += s_scan[w];
    }
    int2* moves = a.moves + r * a.moves_stride;
    float* w_out = a.weights_out + r * a.weights_out_stride;
    int32_t* p_out = a.positions_out ? a.positions_out + r * a.positions_out_stride : nullptr;
    {
        uint32_t hole = hole0, tie = tie0;
        each([&](uint32_t i, uint32_t key, bool in) {
            const bool stay = stays(key, in, tie);
            const bool open = i < m && !stay;
            const unsigned long long opens = __ballot(open);
            if (open) moves[hole + lanes_below(opens)].y = static_cast<int32_t>(i);
            hole += static_cast<uint32_t>(__popcll(opens));
            if (i < m && stay) {
                w_out[i] = weights[i];
                if (p_out) p_out[i] = static_cast<int32_t>(ages.position(i));
            }
        });
    }
    __threadfence_block();
    __syncthreads();
    {
        uint32_t mover = move0, tie = tie0;
        each([&](uint32_t i, uint32_t key, bool in) {
            const bool stay = stays(key, in, tie);
            const bool go = i >= m && stay;
            const unsigned long long goes = __ballot(go);
            if (go) {
                const uint32_t j = mover + lanes_below(goes);
                const uint32_t to = static_cast<uint32_t>(moves[j].y);
                w_out[to] = weights[i];
                if (p_out) p_out[to] = static_cast<int32_t>(ages.position(i));
                moves[j] = make_int2(slot_at(a, r, i), slot_at(a, r, to));
            }
            mover += static_cast<uint32_t>(__popcll(goes));
        });
    }
    if (t == 0) {
        a.len[r] = static_cast<int32_t>(m);
        a.n_moves[r] = static_cast<int32_t>(total);
    }
}

// The pages that get free, requests in order: a workgroup a request, which counts
// those of the requests before it.
constexpr int EF_NT = 256;

__device__ __forceinline__ uint32_t pages_freed(const EvictArgs& a, uint32_t r, uint32_t& first)
{
    const uint64_t page = 1ull << a.page_lg;
    first = static_cast<uint32_t>((static_cast<uint64_t>(a.len[r]) + page - 1) >> a.page_lg);
    return static_cast<uint32_t>((request_len(a, r) + page - 1) >> a.page_lg) - first;
}

__global__ __launch_bounds__(EF_NT) void ev_free(EvictArgs a)
{
    __shared__ uint32_t s_sum[EF_NT / 64];
    const uint32_t r = blockIdx.x, t = threadIdx.x;
    const bool last = r + 1 == a.n_requests;
    uint32_t before = 0, moves = 0, first;
    for (uint32_t i = t; i < r; i += EF_NT) before += pages_freed(a, i, first);
    if (last)
        for (uint32_t i = t; i < a.n_requests; i += EF_NT) moves += static_cast<uint32_t>(a.n_moves[i]);
    before = block_sum<EF_NT>(before, s_sum);
    if (last) moves = block_sum<EF_NT>(moves, s_sum);
    const uint32_t n = pages_freed(a, r, first);
    for (uint32_t i = t; i < n; i += EF_NT)
        if (before + i < a.freed_cap) a.freed[before + i] = a.table[r * a.table_stride + first + i];
    if (last && t == 0) {
        a.counts[0] = static_cast<int32_t>(before + n);
        a.counts[1] = static_cast<int32_t>(moves);
    }
}

// ---- move ------------------------------------------------------------------------
struct MoveArgs {
    char* base[2];
    uint64_t page[2], slot[2], head[2];  // strides in bytes
    const int2* moves;
    uint64_t moves_stride;
    const int32_t* n_moves;
    uint32_t cap, heads, units;  // units: pieces of sizeof(U) bytes in a head's row
    uint64_t n_slots;
    uint32_t page_lg, per;       // workgroups of a request
};

constexpr int MV_NT = 256;

// Bound by memory.  A thread moves one piece of the keys and of the values at a time.
template <class U>
__global__ __launch_bounds__(MV_NT) void ev_move(MoveArgs a)
{
    const uint32_t r = blockIdx.x / a.per, row = a.heads * a.units;
    const uint32_t n = static_cast<uint32_t>(min(max(a.n_moves[r], 0), static_cast<int32_t>(a.cap)));
    const int2* moves = a.moves + r * a.moves_stride;
    const uint64_t pieces = static_cast<uint64_t>(n) * row;
    for (uint64_t i = (blockIdx.x % a.per) * static_cast<uint64_t>(MV_NT) + threadIdx.x; i < pieces;
         i += static_cast<uint64_t>(a.per) * MV_NT) {
        const uint32_t j = static_cast<uint32_t>(i / row), in = static_cast<uint32_t>(i % row);
        const uint32_t head = in / a.units, unit = in % a.units;
        const int2 move = moves[j];
        if (move.x < 0 || move.y < 0 || static_cast<uint32_t>(move.x) >= a.n_slots ||
            static_cast<uint32_t>(move.y) >= a.n_slots)
            continue;
        const uint32_t mask = (1u << a.page_lg) - 1u;
        U x[2];
#pragma unroll
        for (int c = 0; c < 2; ++c)
            x[c] = __builtin_nontemporal_load(reinterpret_cast<const U*>(
                a.base[c] + (static_cast<uint32_t>(move.x) >> a.page_lg) * a.page[c] +
                (static_cast<uint32_t>(move.x) & mask) * a.slot[c] + head * a.head[c] + unit * sizeof(U)));
#pragma unroll
        for (int c = 0; c < 2; ++c)
            __builtin_nontemporal_store(
                x[c], reinterpret_cast<U*>(a.base[c] + (static_cast<uint32_t>(move.y) >> a.page_lg) * a.page[c] +
                                           (static_cast<uint32_t>(move.y) & mask) * a.slot[c] + head * a.head[c] +
                                           unit * sizeof(U)));
    }
}

}  // namespace

}  // namespace crimpl

using namespace crimpl;

extern "C" int cr_paged_evict(const cr_paged_evict_args* args, cr_stream_t stream)
{
    if (!args) {
        set_error("cr_paged_evict: invalid argument");
        return CR_ERR_INVALID;
    }
    const cr_paged_evict_args& p = *args;
    if (!power_of_two(p.page_size)) {
        set_error("cr_paged_evict: invalid argument (page size %u)", p.page_size);
        return CR_ERR_INVALID;
    }
    const uint64_t room = static_cast<uint64_t>(p.table_cols) * p.page_size;
    if (!p.d_counts || p.table_stride < p.table_cols ||
        (p.n_requests && (!p.d_kv_len || !p.d_keep || !p.d_len || !p.d_n_moves)) ||
        (room && p.n_requests && (!p.d_weights || !p.d_weights_out || !p.d_table || p.weights_stride < room ||
                  p.weights_out_stride < room)) ||
        (p.d_positions && (!p.d_kept || !p.d_positions_out || p.positions_stride < room)) ||
        (p.d_positions_out && p.positions_out_stride < room) || p.moves_stride < p.moves_cap ||
        p.moves_cap < room / 2 || (p.moves_cap && p.n_requests && !p.d_moves) || (p.freed_cap && !p.d_freed)) {
        set_error("cr_paged_evict: invalid argument (rows hold table_cols * page_size entries, half as many moves)");
        return CR_ERR_INVALID;
    }
    const uint64_t n_slots = static_cast<uint64_t>(p.n_pages) * p.page_size;
    if (n_slots >> 31 || room >> 30 || p.n_requests >> 20 || p.sinks >> 31 || p.recent >> 31) {
        set_error("cr_paged_evict: supported up to 2^31 - 1 slots, 2^30 - 1 positions and 2^20 - 1 requests");
        return CR_ERR_UNSUPPORTED;
    }
    hipStream_t s = as_stream(stream);
    if (p.n_requests == 0) return fill_u32(reinterpret_cast<uint32_t*>(p.d_counts), 0, 2, s);
    EvictArgs a{};
    a.weights = p.d_weights;
    a.weights_stride = p.weights_stride;
    a.positions = p.d_positions;
    a.positions_stride = p.positions_stride;
    a.kept = p.d_kept;
    a.seen = p.d_seen;
    a.kv_len = p.d_kv_len;
    a.keep = p.d_keep;
    a.table = p.d_table;
    a.cols = p.table_cols;
    a.table_stride = p.table_stride;
    a.page_lg = static_cast<uint32_t>(__builtin_ctz(p.page_size));
    a.n_pages = p.n_pages;
    a.n_requests = p.n_requests;
    a.room = static_cast<uint32_t>(room);
    a.pins = p.pinned != nullptr;
    a.sinks = p.sinks;
    a.recent = p.recent;
    a.weights_out = p.d_weights_out;
    a.weights_out_stride = p.weights_out_stride;
    a.positions_out = p.d_positions_out;
    a.positions_out_stride = p.positions_out_stride;
    a.len = p.d_len;
    a.moves = reinterpret_cast<int2*>(p.d_moves);
    a.moves_stride = p.moves_stride;
    a.n_moves = p.d_n_moves;
    a.freed = p.d_freed;
    a.freed_cap = p.freed_cap;
    a.counts = p.d_counts;
    a.keys_stride = (a.room + EV_ROW - 1) / EV_ROW * EV_ROW;
    const bool direct = p.pinned && is_direct(p.pinned);
    const uint32_t n_words = static_cast<uint32_t>((n_slots + 31) / 32);
    Carver cv;
    const size_t o_keys = cv.add(static_cast<size_t>(p.n_requests) * a.keys_stride * 4);
    const size_t o_words = cv.add(p.pinned && !direct ? n_words * 4ull : 0);
    Scratch sc;
    CR_RET(sc.alloc(std::max<size_t>(256, cv.total), s));
    a.keys = sc.at<uint32_t>(o_keys);
    if (p.pinned)
        CR_RET(set_bits(p.pinned, direct, sc.at<uint32_t>(o_words), n_words, static_cast<uint32_t>(n_slots), stream,
                        &a.pinned));
    CR_TIMED("ev_pick", s);
    ev_pick<<<p.n_requests, EV_NT, 0, s>>>(a);
    ev_free<<<p.n_requests, EF_NT, 0, s>>>(a);
    CR_LAUNCH_CHECK();
    return CR_OK;
}

extern "C" int cr_paged_move(const int32_t* d_moves, uint32_t moves_cap, uint64_t moves_stride,
                             const int32_t* d_n_moves, uint32_t n_requests, const cr_paged_cache* cache,
                             cr_stream_t stream)
{
    if (!cache || !cache->k || !cache->v || !power_of_two(cache->page_size) || cache->dtype > CR_BF16 ||
        (n_requests && (!d_n_moves || (moves_cap && !d_moves))) || moves_stride < moves_cap) {
        set_error("cr_paged_move: invalid argument");
        return CR_ERR_INVALID;
    }
    const uint64_t es = cache->dtype == CR_F32 ? 4 : 2;
    MoveArgs a{};
    a.base[0] = static_cast<char*>(cache->k);
    a.base[1] = static_cast<char*>(cache->v);
    a.page[0] = cache->k_page_stride * es;
    a.page[1] = cache->v_page_stride * es;
    a.slot[0] = cache->k_slot_stride * es;
    a.slot[1] = cache->v_slot_stride * es;
    a.head[0] = cache->k_head_stride * es;
    a.head[1] = cache->v_head_stride * es;
    a.moves = reinterpret_cast<const int2*>(d_moves);
    a.moves_stride = moves_stride;
    a.n_moves = d_n_moves;
    a.cap = moves_cap;
    a.heads = cache->n_heads;
    a.n_slots = static_cast<uint64_t>(cache->n_pages) * cache->page_size;
    a.page_lg = static_cast<uint32_t>(__builtin_ctz(cache->page_size));
    uint64_t all = cache->head_dim * es;
    for (int c = 0; c < 2; ++c) all |= reinterpret_cast<uintptr_t>(a.base[c]) | a.page[c] | a.slot[c] | a.head[c];
    const uint32_t unit = all % 16 == 0 ? 16 : static_cast<uint32_t>(es);
    a.units = static_cast<uint32_t>(cache->head_dim * es / unit);
    const uint64_t row = static_cast<uint64_t>(a.heads) * a.units;
    if (row == 0 || moves_cap == 0 || n_requests == 0) return CR_OK;
    if (row >> 24 || moves_cap >> 31 || n_requests >> 20) {
        set_error("cr_paged_move: too many elements for one call");
        return CR_ERR_UNSUPPORTED;
    }
    // About eight workgroups a CU, shared evenly by the requests.
    const uint64_t most = (moves_cap * row + MV_NT - 1) / MV_NT;
    a.per = static_cast<uint32_t>(std::min<uint64_t>(most, std::max(1u, 8 * num_cus() / n_requests)));
    const uint32_t grid = a.per * n_requests;
    hipStream_t s = as_stream(stream);
    CR_TIMED("ev_move", s);
    if (unit == 16)
        ev_move<cr_v4u><<<grid, MV_NT, 0, s>>>(a);
    else if (es == 4)
        ev_move<uint32_t><<<grid, MV_NT, 0, s>>>(a);
    else
        ev_move<uint16_t><<<grid, MV_NT, 0, s>>>(a);
    CR_LAUNCH_CHECK();
    return CR_OK;
}

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
#include <type_traits>

#include "internal.hpp"
#include "rows.hpp"
#include "set_bits.hpp"

namespace crimpl {

namespace {

constexpr int EV_NT = 1024;
constexpr uint32_t EV_SAFE = 0xFFFFFFFFu;  // above the order of every weight
constexpr uint32_t EV_BINS = 2048;         // of a digit of 11 bits
constexpr uint32_t EV_COPIES = 4;          // of the first digit's counts
constexpr uint32_t EV_ALL = 0xFFFFFFFFu;   // ties: all that equal the last stay
constexpr uint32_t EV_NO_DIGIT = 2046;     // a first digit above those of all weights and below that of EV_SAFE

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
    bool wide;            // rows can be read four entries at a time
    // Long rows, in segments: the entries' places in the order, and what the launches leave
    // for one another.
    uint32_t segments;
    uint32_t* keys;       // [n_requests][segments][SG_SIZE]
    uint2* undecided;     // the same: (key, entry)
    uint32_t* bins;       // [n_requests][segments][EV_BINS / 2], two counts a word
    uint4* counts_of;     // [n_requests][segments]
    uint4* from;          // [n_requests][segments]
    uint4* picked;        // [n_requests][2]
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

// Finds the digit in which the n-th largest of the counted values lies (n >= 1, at
// most their number).  count(bin): how many have it.  Every thread gets the digit, how
// many values have a higher one, and how many have it.
template <int NT, class F>
__device__ __forceinline__ void find_digit(F count, uint32_t n, uint32_t* s_scan, uint32_t* s_found, uint32_t& digit,
                                           uint32_t& above, uint32_t& here)
{
    constexpr uint32_t PER = EV_BINS / NT;
    const uint32_t t = threadIdx.x;
    uint32_t c[PER], mine = 0, total;
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        c[j] = count(EV_BINS - 1 - (t * PER + j));
        mine += c[j];
    }
    uint32_t before = block_excl_scan<NT>(mine, s_scan, total);
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
        if (before < n && n <= before + c[j]) {
            s_found[0] = EV_BINS - 1 - (t * PER + j);
            s_found[1] = before;
            s_found[2] = c[j];
        }
        before += c[j];
    }
    __syncthreads();
    digit = s_found[0];
    above = s_found[1];
    here = s_found[2];
    __syncthreads();
}

// Four neighbours each of ROWS parts of a request's row: entries first[j] + e.
template <uint32_t ROWS>
struct Entries {
    float weight[ROWS][4];
    int32_t position[ROWS][4];
};

template <class T>
__device__ __forceinline__ void store4(T* row, uint32_t i, uint32_t on, bool wide, const T (&x)[4])
{
    if (wide && on == 15u) {
        typedef T V __attribute__((ext_vector_type(4)));
        *reinterpret_cast<V*>(row + i) = V{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if ((on >> e) & 1u) row[i + e] = x[e];
    }
}

// Weights and positions of entries i0 + j * 256 + e < len (len > 0; any values behind them).
// No load waits for another: rows that can be read four at a time are read up to their end.
template <uint32_t ROWS>
__device__ __forceinline__ void load_entries(const EvictArgs& a, const Ages& ages, uint32_t r, uint32_t i0, uint32_t len,
                                             Entries<ROWS>& x)
{
    const float* weights = a.weights + r * a.weights_stride;
    if (a.wide) {
        typedef float VF __attribute__((ext_vector_type(4)));
        typedef int32_t VI __attribute__((ext_vector_type(4)));
        VF w[ROWS];
        VI p[ROWS];
#pragma unroll
        for (uint32_t j = 0; j < ROWS; ++j) w[j] = *reinterpret_cast<const VF*>(weights + min(i0 + j * 256, a.room - 4));
        if (ages.kept) {
#pragma unroll
            for (uint32_t j = 0; j < ROWS; ++j) p[j] = *reinterpret_cast<const VI*>(ages.row + min(i0 + j * 256, a.room - 4));
        }
#pragma unroll
        for (uint32_t j = 0; j < ROWS; ++j)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                x.weight[j][e] = w[j][e];
                if (ages.kept) x.position[j][e] = p[j][e];
            }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < ROWS; ++j)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) x.weight[j][e] = weights[min(i0 + j * 256 + e, len - 1)];
        if (ages.kept) {
#pragma unroll
            for (uint32_t j = 0; j < ROWS; ++j)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) x.position[j][e] = ages.row[min(i0 + j * 256 + e, ages.kept - 1)];
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < ROWS; ++j)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const uint32_t i = i0 + j * 256 + e;
            if (i >= ages.kept) x.position[j][e] = static_cast<int32_t>(ages.first + i);
        }
}

// The pinned ones of them, as bits.
template <uint32_t ROWS>
__device__ __forceinline__ void load_pinned(const EvictArgs& a, uint32_t r, uint32_t i0, uint32_t len, uint32_t (&on)[ROWS])
{
#pragma unroll
    for (uint32_t j = 0; j < ROWS; ++j) on[j] = 0;
    if (!a.pins || a.pinned.end == 0) return;
    const int32_t* table = a.table + r * a.table_stride;
    constexpr uint32_t MOST = ROWS * 4;
    auto look = [&](auto& word, auto& shift, auto& in, auto n_of, auto entry) {  // side by side
        constexpr uint32_t N = decltype(n_of)::value;
        uint32_t slot[N], x[N];
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) {
            const uint32_t i = min(entry(j), len - 1), page = static_cast<uint32_t>(table[i >> a.page_lg]);
            slot[j] = (page << a.page_lg) + (i & ((1u << a.page_lg) - 1u));
            in[j] = page < a.n_pages && slot[j] < a.pinned.end;
        }
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) {
            word[j] = in[j] ? slot[j] >> 5 : 0u;
            shift[j] = slot[j] & 31u;
        }
        a.pinned.words(word, x);
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) word[j] = in[j] ? x[j] >> shift[j] : 0u;
    };
    if (a.page_lg >= 2) {  // four neighbours lie in one page and one word
        uint32_t word[ROWS], shift[ROWS];
        bool in[ROWS];
        look(word, shift, in, std::integral_constant<uint32_t, ROWS>{}, [&](uint32_t j) { return i0 + j * 256; });
#pragma unroll
        for (uint32_t j = 0; j < ROWS; ++j) on[j] = word[j] & 15u;
    } else {
        uint32_t word[MOST], shift[MOST];
        bool in[MOST];
        look(word, shift, in, std::integral_constant<uint32_t, MOST>{},
             [&](uint32_t j) { return i0 + j / 4 * 256 + j % 4; });
#pragma unroll
        for (uint32_t j = 0; j < MOST; ++j) on[j / 4] |= (word[j] & 1u) << (j % 4);
    }
}

// Their places in the order (0 behind the request's last).
template <uint32_t ROWS>
__device__ __forceinline__ void keys_of(const EvictArgs& a, const Ages& ages, uint32_t i0, uint32_t len, const Entries<ROWS>& x,
                                        const uint32_t (&pinned)[ROWS], uint32_t (&key)[ROWS][4])
{
#pragma unroll
    for (uint32_t j = 0; j < ROWS; ++j)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const uint32_t i = i0 + j * 256 + e;
            const int64_t at = i < ages.kept ? static_cast<int64_t>(x.position[j][e]) : ages.first + i;
            key[j][e] = i >= len ? 0u : ages.safe(at) || ((pinned[j] >> e) & 1u) ? EV_SAFE : weight_order(x.weight[j][e]);
        }
}

// Bits e of the entries i + e < m of four.
__device__ __forceinline__ uint32_t below4(uint32_t i, uint32_t m)
{
    return i >= m ? 0u : m - i >= 4 ? 15u : (1u << (m - i)) - 1u;
}

// Which of four stay: those above `last`, the safe ones, and of those that equal it the
// ones before whom fewer than `ties` do; tie: how many do before the first.
__device__ __forceinline__ uint32_t stays4(const uint32_t (&key)[4], uint32_t in, uint32_t last, uint32_t ties, uint32_t tie)
{
    uint32_t stay = 0;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
        const bool eq = key[e] == last && ((in >> e) & 1u) && last != EV_SAFE;
        stay |= (key[e] > last || key[e] == EV_SAFE || (eq && tie < ties) ? 1u : 0u) << e;
        tie += eq ? 1u : 0u;
    }
    return stay & in;
}

__device__ __forceinline__ uint32_t ties4(const uint32_t (&key)[4], uint32_t in, uint32_t last)
{
    uint32_t n = 0;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) n += key[e] == last && ((in >> e) & 1u) && last != EV_SAFE ? 1u : 0u;
    return n;
}

// What lies in the entries `on` of four from i afterwards, where they stay.
__device__ __forceinline__ void keep4(const EvictArgs& a, uint32_t r, uint32_t i, uint32_t on, const float (&weight)[4],
                                      const int32_t (&position)[4])
{
    store4(a.weights_out + r * a.weights_out_stride, i, on, a.wide, weight);
    if (a.positions_out) store4(a.positions_out + r * a.positions_out_stride, i, on, a.wide, position);
}

// Move j of request r: entry `from` goes to place `to`; of N of them (those that are
// not there: the same twice), so that no look-up waits for another.
template <uint32_t N>
__device__ __forceinline__ void move_entries(const EvictArgs& a, const Ages& ages, uint32_t r, const uint32_t (&from)[N],
                                             const uint32_t (&to)[N], const uint32_t (&j)[N], const bool (&on)[N])
{
    float w[N];
    int32_t p[N], page[2][N];
    const int32_t* table = a.table + r * a.table_stride;
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) {
        w[k] = a.weights[r * a.weights_stride + from[k]];
        page[0][k] = table[from[k] >> a.page_lg];
        page[1][k] = table[to[k] >> a.page_lg];
        p[k] = static_cast<int32_t>(ages.first + from[k]);
    }
    if (ages.kept) {
        int32_t x[N];
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) x[k] = ages.row[min(from[k], ages.kept - 1)];
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) p[k] = from[k] < ages.kept ? x[k] : p[k];
    }
    const uint32_t mask = (1u << a.page_lg) - 1u;
    auto slot = [&](int32_t page, uint32_t i) {
        return static_cast<uint32_t>(page) < a.n_pages
                   ? static_cast<int32_t>((static_cast<uint32_t>(page) << a.page_lg) + (i & mask))
                   : -1;
    };
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) {
        if (!on[k]) continue;
        a.weights_out[r * a.weights_out_stride + to[k]] = w[k];
        if (a.positions_out) a.positions_out[r * a.positions_out_stride + to[k]] = p[k];
        a.moves[r * a.moves_stride + j[k]] = make_int2(slot(page[0][k], from[k]), slot(page[1][k], to[k]));
    }
}
constexpr uint32_t EV_MOVES = 4;  // a thread's at a time

// How many of the entries are safe, and how many stay in all.
__device__ __forceinline__ uint32_t staying(uint32_t len, uint32_t keep, uint32_t n_safe)
{
    return keep >= len ? len : max(keep, n_safe);
}

// The pages of a request's first m entries, and how many it holds behind them.
__device__ __forceinline__ uint32_t pages_freed(const EvictArgs& a, uint32_t len, uint32_t m, uint32_t& first)
{
    const uint64_t page = 1ull << a.page_lg;
    first = static_cast<uint32_t>((m + page - 1) >> a.page_lg);
    return static_cast<uint32_t>((len + page - 1) >> a.page_lg) - first;
}

// Their list, behind `before` pages of other requests.
template <int NT>
__device__ __forceinline__ uint32_t list_freed(const EvictArgs& a, uint32_t r, uint32_t len, uint32_t m, uint32_t before)
{
    uint32_t first;
    const uint32_t n = pages_freed(a, len, m, first);
    for (uint32_t i = threadIdx.x; i < n; i += NT)
        if (before + i < a.freed_cap) a.freed[before + i] = a.table[r * a.table_stride + first + i];
    return n;
}

// Entries of a request that one workgroup takes: what its registers hold, which is read once
// and not written down in between (64 requests of 16384, moves included: 187 us, by the launches
// for longer rows 198).
constexpr uint64_t EV_WHOLE = 16384;

// A workgroup a request of at most E * NT entries, whose places in the order stay in
// registers: four neighbours a lane, 256 a wave at a time.  The last that stays is found by
// its digits, of 11, 11 and 10 bits, counted in LDS; what bounds it is the chain of those
// counts and scans, not the bytes (1003 entries: 7.5 us).
template <int NT, uint32_t E>
__global__ __launch_bounds__(NT) void ev_pick(EvictArgs a)
{
    constexpr uint32_t ROWS = E / 4, WAVES = NT / 64, HOLES = E * NT / 2;
    __shared__ uint32_t s_mem[EV_COPIES * EV_BINS > HOLES ? EV_COPIES * EV_BINS : HOLES];  // counts, then holes
    __shared__ uint32_t s_movers[HOLES];
    __shared__ uint32_t s_scan[WAVES], s_found[3], s_of[2][WAVES];
    const uint32_t r = blockIdx.x, t = threadIdx.x, lane = __lane_id(), wave = t >> 6;
    const uint32_t len = request_len(a, r);
    const Ages ages(a, r, len);
    const uint32_t keep = static_cast<uint32_t>(max(a.keep[r], 0));
    const uint32_t i0 = wave * 64 * E + lane * 4;  // row j: from i0 + j * 256
    uint32_t key[ROWS][4], n_safe = 0;
    Entries<ROWS> x;
    if (len) load_entries<ROWS>(a, ages, r, i0, len, x);
    if (keep >= len) {  // all stay
#pragma unroll
        for (uint32_t j = 0; j < ROWS; ++j) keep4(a, r, i0 + j * 256, below4(i0 + j * 256, len), x.weight[j], x.position[j]);
        if (t == 0) {
            a.len[r] = static_cast<int32_t>(len);
            a.n_moves[r] = 0;
            if (a.n_requests == 1) a.counts[0] = a.counts[1] = 0;
        }
        return;
    }
    {
        uint32_t pinned[ROWS];
        load_pinned<ROWS>(a, r, i0, len, pinned);
        for (uint32_t i = t; i < EV_COPIES * EV_BINS; i += NT) s_mem[i] = 0;
        keys_of<ROWS>(a, ages, i0, len, x, pinned, key);
    }
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < ROWS; ++j)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            if (i0 + j * 256 + e >= len) continue;
            n_safe += key[j][e] == EV_SAFE ? 1u : 0u;
            if (key[j][e] != EV_SAFE) atomicAdd(&s_mem[wave % EV_COPIES * EV_BINS + (key[j][e] >> 21)], 1u);
        }
    n_safe = block_sum<NT>(n_safe, s_scan);
    const uint32_t m = staying(len, keep, n_safe);
    // Of the others, the m - n_safe largest stay.
    uint32_t last = EV_SAFE, ties = 0;
    if (m > n_safe) {
        uint32_t n = m - n_safe, digit, above, here;
        find_digit<NT>(
            [&](uint32_t bin) {
                uint32_t c = 0;
#pragma unroll
                for (uint32_t k = 0; k < EV_COPIES; ++k) c += s_mem[k * EV_BINS + bin];
                return c;
            },
            n, s_scan, s_found, digit, above, here);
        n -= above;
        last = digit << 21;
#pragma unroll
        for (int shift = 10; shift >= 0; shift -= 10) {
            const uint32_t bits = shift == 10 ? 11 : 10, mask = (1u << bits) - 1u;
            for (uint32_t i = t; i < EV_BINS; i += NT) s_mem[i] = 0;
            __syncthreads();
#pragma unroll
            for (uint32_t j = 0; j < ROWS; ++j)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (i0 + j * 256 + e < len && key[j][e] >> (shift + bits) == last >> (shift + bits))
                        atomicAdd(&s_mem[(key[j][e] >> shift) & mask], 1u);
            __syncthreads();
            find_digit<NT>([&](uint32_t bin) { return s_mem[bin]; }, n, s_scan, s_found, digit, above, here);
            n -= above;
            last |= digit << shift;
        }
        ties = n < here ? n : EV_ALL;
    }
    // Which stay, and how many holes and movers lie before each lane's four: both counts and
    // the ties' fit one word for a wave's 256.
    uint32_t tie0 = 0;
    const bool ranked = ties != 0 && ties != EV_ALL;
    if (ranked) {
        uint32_t n = 0;
#pragma unroll
        for (uint32_t j = 0; j < ROWS; ++j) n += ties4(key[j], below4(i0 + j * 256, len), last);
        n = wave_sum(n);
        if (lane == 0) s_scan[wave] = n;
        __syncthreads();
        for (uint32_t w = 0; w < wave; ++w) tie0 += s_scan[w];
    }
    uint32_t stay[ROWS], rank[ROWS], holes = 0, movers = 0;
#pragma unroll
    for (uint32_t j = 0; j < ROWS; ++j) {
        const uint32_t i = i0 + j * 256, in = below4(i, len), mine = below4(i, m);
        uint32_t tie = tie0;
        if (ranked) {
            const uint32_t n = ties4(key[j], in, last), upto = wave_incl_scan(n);
            tie = tie0 + upto - n;
            tie0 += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), 63));
        }
        stay[j] = stays4(key[j], in, last, ties, tie);
        const uint32_t n = __popc(mine & ~stay[j]) | static_cast<uint32_t>(__popc(stay[j] & ~mine)) << 16;
        const uint32_t upto = wave_incl_scan(n);
        rank[j] = (holes | movers << 16) + upto - n;  // (of a wave: at most 64 E of either)
        const uint32_t all = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), 63));
        holes += all & 0xFFFFu;
        movers += all >> 16;
    }
    __syncthreads();
    if (lane == 0) {
        s_of[0][wave] = holes;
        s_of[1][wave] = movers;
    }
    __syncthreads();
    uint32_t hole0 = 0, move0 = 0, total = 0;
    for (uint32_t w = 0; w < WAVES; ++w) {
        hole0 += w < wave ? s_of[0][w] : 0u;
        move0 += w < wave ? s_of[1][w] : 0u;
        total += s_of[0][w];
    }
#pragma unroll
    for (uint32_t j = 0; j < ROWS; ++j) {
        const uint32_t i = i0 + j * 256, mine = below4(i, m);
        const uint32_t open = mine & ~stay[j], go = stay[j] & ~mine;
        uint32_t hole = hole0 + (rank[j] & 0xFFFFu), mover = move0 + (rank[j] >> 16);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            if ((open >> e) & 1u) s_mem[hole++] = i + e;
            if ((go >> e) & 1u) s_movers[mover++] = i + e;
        }
        keep4(a, r, i, mine & stay[j], x.weight[j], x.position[j]);
    }
    __syncthreads();
    for (uint32_t j0 = t; j0 < total; j0 += EV_MOVES * NT) {
        uint32_t from[EV_MOVES], to[EV_MOVES], at[EV_MOVES];
        bool on[EV_MOVES];
#pragma unroll
        for (uint32_t i = 0; i < EV_MOVES; ++i) {
            at[i] = min(j0 + i * NT, total - 1);
            on[i] = j0 + i * NT < total;
            from[i] = s_movers[at[i]];
            to[i] = s_mem[at[i]];
        }
        move_entries<EV_MOVES>(a, ages, r, from, to, at, on);
    }
    uint32_t freed = 0;
    if (a.n_requests == 1) freed = list_freed<NT>(a, r, len, m, 0);
    if (t == 0) {
        a.len[r] = static_cast<int32_t>(m);
        a.n_moves[r] = static_cast<int32_t>(total);
        if (a.n_requests == 1) {
            a.counts[0] = static_cast<int32_t>(freed);
            a.counts[1] = static_cast<int32_t>(total);
        }
    }
}

// ---- long rows: a workgroup per segment ----------------------------------------------
// The same in launches that leave one another their counts: keys and first digits
// (sg_keys), the digit in which the last that stays lies (sg_digit), those that have it
// (sg_split), which of them stay and where each segment's holes and movers begin
// (sg_decide), and what lies where (sg_place); ev_finish then moves the weights.  Four
// requests of 131072 entries: 7.9, 5.2, 4.3, 8.3, 6.4 and 5.4 us, most of each the launch
// and the chain of loads behind it (a workgroup a request, which read its row for every digit:
// 480 in all).
constexpr int SG_NT = 256;
constexpr uint32_t SG_WAVES = SG_NT / 64;
constexpr uint32_t SG_ROWS = 4;                             // of 256 entries, a wave's
constexpr uint32_t SG_SIZE = SG_WAVES * SG_ROWS * 256;

__global__ __launch_bounds__(SG_NT) void sg_keys(EvictArgs a)
{
    __shared__ uint32_t s_bins[2][EV_BINS];
    __shared__ uint32_t s_scan[SG_WAVES];
    const uint32_t r = blockIdx.x / a.segments, seg = blockIdx.x % a.segments, t = threadIdx.x;
    const uint32_t lane = __lane_id(), wave = t >> 6, len = request_len(a, r);
    if (seg * SG_SIZE >= len) return;
    const Ages ages(a, r, len);
    uint32_t key[SG_ROWS][4], pinned[SG_ROWS], n_safe = 0;
    const uint32_t i0 = seg * SG_SIZE + wave * SG_ROWS * 256 + lane * 4;
    Entries<SG_ROWS> x;
    load_pinned<SG_ROWS>(a, r, i0, len, pinned);
    load_entries<SG_ROWS>(a, ages, r, i0, len, x);
    keys_of<SG_ROWS>(a, ages, i0, len, x, pinned, key);
    for (uint32_t i = t; i < EV_BINS; i += SG_NT) s_bins[0][i] = s_bins[1][i] = 0;
    __syncthreads();
    uint32_t* keys = a.keys + static_cast<uint64_t>(blockIdx.x) * SG_SIZE;
#pragma unroll
    for (uint32_t j = 0; j < SG_ROWS; ++j) {
        const uint32_t in = (wave * SG_ROWS + j) * 256 + lane * 4;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            if (seg * SG_SIZE + in + e >= len) continue;
            n_safe += key[j][e] == EV_SAFE ? 1u : 0u;
            if (key[j][e] != EV_SAFE) atomicAdd(&s_bins[wave % 2][key[j][e] >> 21], 1u);
        }
        *reinterpret_cast<uint4*>(keys + in) = make_uint4(key[j][0], key[j][1], key[j][2], key[j][3]);
    }
    n_safe = block_sum<SG_NT>(n_safe, s_scan);
    uint32_t* bins = a.bins + static_cast<uint64_t>(blockIdx.x) * (EV_BINS / 2);
    for (uint32_t i = t; i < EV_BINS / 2; i += SG_NT)  // (a segment's counts are at most SG_SIZE)
        bins[i] = (s_bins[0][2 * i] + s_bins[1][2 * i]) | (s_bins[0][2 * i + 1] + s_bins[1][2 * i + 1]) << 16;
    if (t == 0) a.counts_of[blockIdx.x].w = n_safe;
}

// picked[2 r]: m, the digit, how many stay of those that have it, the request's segments.
__global__ __launch_bounds__(EV_NT) void sg_digit(EvictArgs a)
{
    __shared__ uint32_t s_scan[EV_NT / 64], s_found[3];
    const uint32_t r = blockIdx.x, t = threadIdx.x, len = request_len(a, r);
    const uint32_t keep = static_cast<uint32_t>(max(a.keep[r], 0)), segments = (len + SG_SIZE - 1) / SG_SIZE;
    const uint64_t seg0 = static_cast<uint64_t>(r) * a.segments;
    uint32_t n_safe = 0;
    for (uint32_t i = t; i < segments; i += EV_NT) n_safe += a.counts_of[seg0 + i].w;
    n_safe = block_sum<EV_NT>(n_safe, s_scan);
    const uint32_t m = staying(len, keep, n_safe);
    uint32_t digit = EV_NO_DIGIT, above = 0, here;
    if (m > n_safe) {
        static_assert(EV_BINS == 2 * EV_NT, "a word of two counts per thread");
        const uint32_t word = (EV_BINS - 1 - t * 2) / 2;
        uint32_t lo = 0, hi = 0;
        constexpr uint32_t AHEAD = 32;
        for (uint32_t i = 0; i < segments; i += AHEAD) {
            uint32_t x[AHEAD];
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k) x[k] = a.bins[(seg0 + min(i + k, segments - 1)) * (EV_BINS / 2) + word];
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k) {
                lo += i + k < segments ? x[k] & 0xFFFFu : 0u;
                hi += i + k < segments ? x[k] >> 16 : 0u;
            }
        }
        find_digit<EV_NT>([&](uint32_t bin) { return bin & 1u ? hi : lo; }, m - n_safe, s_scan, s_found, digit, above, here);
    }
    if (t == 0) a.picked[2 * r] = make_uint4(m, digit, m > n_safe ? m - n_safe - above : 0u, segments);
}

// Rank of a lane's count among the workgroup's, wave by wave in order; s_wave: a slot a wave.
__device__ __forceinline__ uint32_t wave_base(uint32_t mine, uint32_t* s_wave)
{
    __syncthreads();
    if (__lane_id() == 0) s_wave[threadIdx.x >> 6] = mine;
    __syncthreads();
    uint32_t base = 0;
#pragma unroll
    for (uint32_t w = 0; w < SG_WAVES; ++w) base += w < threadIdx.x >> 6 ? s_wave[w] : 0u;
    return base;
}

__device__ __forceinline__ void load_keys(const EvictArgs& a, uint32_t (&key)[SG_ROWS][4])
{
    const uint32_t* keys = a.keys + static_cast<uint64_t>(blockIdx.x) * SG_SIZE;
#pragma unroll
    for (uint32_t j = 0; j < SG_ROWS; ++j) {
        const uint4 x = *reinterpret_cast<const uint4*>(keys + ((threadIdx.x >> 6) * SG_ROWS + j) * 256 + __lane_id() * 4);
        key[j][0] = x.x;
        key[j][1] = x.y;
        key[j][2] = x.z;
        key[j][3] = x.w;
    }
}

// counts_of: the undecided, and of the others the holes and the movers.
__global__ __launch_bounds__(SG_NT) void sg_split(EvictArgs a)
{
    __shared__ uint32_t s_wave[SG_WAVES], s_scan[SG_WAVES];
    const uint32_t r = blockIdx.x / a.segments, seg = blockIdx.x % a.segments, lane = __lane_id(), wave = threadIdx.x >> 6;
    const uint32_t len = request_len(a, r);
    if (seg * SG_SIZE >= len) return;
    uint32_t key[SG_ROWS][4], open[SG_ROWS], rank[SG_ROWS], n_open = 0, holes = 0, movers = 0;
    load_keys(a, key);
    const uint4 picked = a.picked[2 * r];
    const uint32_t m = picked.x, digit = picked.y;
#pragma unroll
    for (uint32_t j = 0; j < SG_ROWS; ++j) {
        const uint32_t i = seg * SG_SIZE + (wave * SG_ROWS + j) * 256 + lane * 4, in = below4(i, len), mine = below4(i, m);
        uint32_t stay = 0;
        open[j] = 0;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            stay |= (key[j][e] >> 21 > digit ? 1u : 0u) << e;
            open[j] |= (key[j][e] >> 21 == digit ? 1u : 0u) << e;
        }
        open[j] &= in;
        stay &= in;
        holes += __popc(mine & ~stay & ~open[j]);
        movers += __popc(stay & ~mine);
        const uint32_t n = __popc(open[j]), upto = wave_incl_scan(n);
        rank[j] = n_open + upto - n;
        n_open += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), 63));
    }
    const uint32_t base = wave_base(n_open, s_wave);
    uint2* to = a.undecided + static_cast<uint64_t>(blockIdx.x) * SG_SIZE;
#pragma unroll
    for (uint32_t j = 0; j < SG_ROWS; ++j) {
        const uint32_t i = seg * SG_SIZE + (wave * SG_ROWS + j) * 256 + lane * 4;
        uint32_t at = base + rank[j];
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if ((open[j] >> e) & 1u) to[at++] = make_uint2(key[j][e], i + e);
    }
    holes = block_sum<SG_NT>(holes, s_scan);
    movers = block_sum<SG_NT>(movers, s_scan);
    const uint32_t all = block_sum<SG_NT>(lane == 0 ? n_open : 0u, s_scan);
    if (threadIdx.x == 0) a.counts_of[blockIdx.x] = make_uint4(all, holes, movers, 0);
}

// picked[2 r + 1]: the last key that stays and how many that equal it do, the moves.
// from: the ties, holes and movers before each segment.
__global__ __launch_bounds__(EV_NT) void sg_decide(EvictArgs a)
{
    constexpr uint32_t WAVES = EV_NT / 64;
    __shared__ uint32_t s_bins[EV_BINS], s_scan[WAVES], s_found[3];
    const uint32_t r = blockIdx.x, t = threadIdx.x, lane = __lane_id(), wave = t >> 6;
    const uint4 picked = a.picked[2 * r];
    const uint32_t m = picked.x, segments = picked.w;
    const uint64_t seg0 = static_cast<uint64_t>(r) * a.segments;
    uint32_t n = picked.z, last = EV_SAFE, ties = 0;
    // a wave a segment, its undecided in order
    auto each = [&](uint32_t seg, auto f) {
        const uint2* from = a.undecided + (seg0 + seg) * SG_SIZE;
        const uint32_t all = a.counts_of[seg0 + seg].x;
        for (uint32_t i0 = 0; i0 < all; i0 += 64) {
            const uint2 x = from[min(i0 + lane, all - 1)];
            f(i0 + lane < all, x.x, x.y);
        }
    };
    if (n) {
        last = picked.y << 21;
#pragma unroll
        for (int shift = 10; shift >= 0; shift -= 10) {
            const uint32_t bits = shift == 10 ? 11 : 10, mask = (1u << bits) - 1u;
            uint32_t digit, above, here;
            for (uint32_t i = t; i < EV_BINS; i += EV_NT) s_bins[i] = 0;
            __syncthreads();
            for (uint32_t seg = wave; seg < segments; seg += WAVES)
                each(seg, [&](bool in, uint32_t key, uint32_t) {
                    if (in && key >> (shift + bits) == last >> (shift + bits)) atomicAdd(&s_bins[(key >> shift) & mask], 1u);
                });
            __syncthreads();
            find_digit<EV_NT>([&](uint32_t bin) { return s_bins[bin]; }, n, s_scan, s_found, digit, above, here);
            n -= above;
            last |= digit << shift;
            ties = n < here ? n : EV_ALL;
        }
    }
    const bool ranked = ties != 0 && ties != EV_ALL;
    // A wave takes neighbouring segments, at most as many as it has lanes; lane k keeps what is
    // counted of the k-th of them.
    uint32_t ties0 = 0, holes0 = 0, movers0 = 0;
    auto before_wave = [&](uint32_t mine, uint32_t* s_wave, uint32_t& all) {  // of the waves before; adds all to `all`
        if (lane == 63) s_wave[wave] = mine;
        __syncthreads();
        uint32_t before = all;
        for (uint32_t w = 0; w < WAVES; ++w) {
            before += w < wave ? s_wave[w] : 0u;
            all += s_wave[w];
        }
        return before;
    };
    for (uint32_t s0 = 0; s0 < segments; s0 += WAVES * 64) {
        const uint32_t per = (min(segments - s0, WAVES * 64) + WAVES - 1) / WAVES, first = s0 + wave * per;
        const uint32_t n_mine = first < segments ? min(per, segments - first) : 0u;
        __syncthreads();
        uint32_t tie = 0;
        if (ranked) {
            for (uint32_t k = 0; k < n_mine; ++k) {
                uint32_t same = 0;
                each(first + k, [&](bool in, uint32_t key, uint32_t) {
                    same += static_cast<uint32_t>(__popcll(__ballot(in && key == last)));
                });
                tie = lane == k ? same : tie;
            }
            const uint32_t upto = wave_incl_scan(tie);
            tie = before_wave(upto, s_scan, ties0) + upto - tie;
        }
        uint32_t holes = 0, movers = 0;
        for (uint32_t k = 0; k < n_mine; ++k) {
            const uint4 c = a.counts_of[seg0 + first + k];
            uint32_t h = c.y, g = c.z, run = static_cast<uint32_t>(__shfl(static_cast<int>(tie), static_cast<int>(k), 64));
            each(first + k, [&](bool in, uint32_t key, uint32_t i) {
                const unsigned long long same = __ballot(in && key == last && ties);
                const uint32_t rank = run + static_cast<uint32_t>(__popcll(same & ((1ull << lane) - 1ull)));
                const bool stay = key > last || (key == last && rank < ties);
                run += static_cast<uint32_t>(__popcll(same));
                h += static_cast<uint32_t>(__popcll(__ballot(in && !stay && i < m)));
                g += static_cast<uint32_t>(__popcll(__ballot(in && stay && i >= m)));
            });
            holes = lane == k ? h : holes;
            movers = lane == k ? g : movers;
        }
        const uint32_t upto_holes = wave_incl_scan(holes), upto_movers = wave_incl_scan(movers);
        const uint32_t hole = before_wave(upto_holes, s_bins, holes0) + upto_holes - holes;
        const uint32_t move = before_wave(upto_movers, s_bins + WAVES, movers0) + upto_movers - movers;
        if (lane < n_mine) a.from[seg0 + first + lane] = make_uint4(tie, hole, move, 0);
    }
    if (t == 0) {
        a.picked[2 * r + 1] = make_uint4(last, ties, holes0, 0);
        a.len[r] = static_cast<int32_t>(m);
        a.n_moves[r] = static_cast<int32_t>(holes0);
    }
}

// What stays in its place; the moves as pairs of entries.
__global__ __launch_bounds__(SG_NT) void sg_place(EvictArgs a)
{
    __shared__ uint32_t s_wave[SG_WAVES];
    const uint32_t r = blockIdx.x / a.segments, seg = blockIdx.x % a.segments, lane = __lane_id(), wave = threadIdx.x >> 6;
    const uint32_t len = request_len(a, r);
    if (seg * SG_SIZE >= len) return;
    const Ages ages(a, r, len);
    uint32_t key[SG_ROWS][4];
    Entries<SG_ROWS> x;
    load_keys(a, key);
    load_entries<SG_ROWS>(a, ages, r, seg * SG_SIZE + wave * SG_ROWS * 256 + lane * 4, len, x);
    const uint32_t m = a.picked[2 * r].x;
    const uint4 picked = a.picked[2 * r + 1], from = a.from[blockIdx.x];
    const uint32_t last = picked.x, ties = picked.y;
    uint32_t tie0 = from.x;
    const bool ranked = ties != 0 && ties != EV_ALL;
    if (ranked) {
        uint32_t n = 0;
#pragma unroll
        for (uint32_t j = 0; j < SG_ROWS; ++j)
            n += ties4(key[j], below4(seg * SG_SIZE + (wave * SG_ROWS + j) * 256 + lane * 4, len), last);
        tie0 += wave_base(wave_sum(n), s_wave);
    }
    uint32_t stay[SG_ROWS], rank[SG_ROWS], counts = 0;
#pragma unroll
    for (uint32_t j = 0; j < SG_ROWS; ++j) {
        const uint32_t i = seg * SG_SIZE + (wave * SG_ROWS + j) * 256 + lane * 4, in = below4(i, len), mine = below4(i, m);
        uint32_t tie = tie0;
        if (ranked) {
            const uint32_t n = ties4(key[j], in, last), upto = wave_incl_scan(n);
            tie += upto - n;
            tie0 += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), 63));
        }
        stay[j] = stays4(key[j], in, last, ties, tie);
        const uint32_t n = __popc(mine & ~stay[j]) | static_cast<uint32_t>(__popc(stay[j] & ~mine)) << 16;
        const uint32_t upto = wave_incl_scan(n);
        rank[j] = counts + upto - n;
        counts += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), 63));
    }
    const uint32_t base = wave_base(counts, s_wave);  // (at most SG_SIZE of either)
    int2* moves = a.moves + r * a.moves_stride;
#pragma unroll
    for (uint32_t j = 0; j < SG_ROWS; ++j) {
        const uint32_t i = seg * SG_SIZE + (wave * SG_ROWS + j) * 256 + lane * 4, mine = below4(i, m);
        uint32_t hole = from.y + ((base + rank[j]) & 0xFFFFu), move = from.z + ((base + rank[j]) >> 16);
        const uint32_t open = mine & ~stay[j], go = stay[j] & ~mine;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            if ((open >> e) & 1u) moves[hole++].y = static_cast<int32_t>(i + e);
            if ((go >> e) & 1u) moves[move++].x = static_cast<int32_t>(i + e);
        }
        keep4(a, r, i, mine & stay[j], x.weight[j], x.position[j]);
    }
}

// The pages that get free, requests in order: a workgroup a request, which counts
// those of the requests before it (one request in one workgroup does without).  Of
// long rows, the moves' weights and slots too, which a workgroup a segment shares.
constexpr int EF_NT = 256;

__global__ __launch_bounds__(EF_NT) void ev_finish(EvictArgs a, uint32_t per)
{
    __shared__ uint32_t s_sum[EF_NT / 64];
    const uint32_t r = blockIdx.x / per, part = blockIdx.x % per, t = threadIdx.x;
    if (a.segments) {
        const Ages ages(a, r, request_len(a, r));
        const uint32_t n = static_cast<uint32_t>(a.n_moves[r]);
        for (uint32_t j0 = part * EF_NT + t; j0 < n; j0 += EV_MOVES * per * EF_NT) {
            uint32_t from[EV_MOVES], to[EV_MOVES], at[EV_MOVES];
            bool on[EV_MOVES];
#pragma unroll
            for (uint32_t i = 0; i < EV_MOVES; ++i) {
                on[i] = j0 + i * per * EF_NT < n;
                at[i] = on[i] ? j0 + i * per * EF_NT : j0;
                const int2 x = a.moves[r * a.moves_stride + at[i]];
                from[i] = static_cast<uint32_t>(x.x);
                to[i] = static_cast<uint32_t>(x.y);
            }
            move_entries<EV_MOVES>(a, ages, r, from, to, at, on);
        }
    }
    if (part) return;
    const bool last = r + 1 == a.n_requests;
    uint32_t before = 0, moves = 0, first;
    for (uint32_t i = t; i < r; i += EF_NT)
        before += pages_freed(a, request_len(a, i), static_cast<uint32_t>(a.len[i]), first);
    if (last)
        for (uint32_t i = t; i < a.n_requests; i += EF_NT) moves += static_cast<uint32_t>(a.n_moves[i]);
    before = block_sum<EF_NT>(before, s_sum);
    if (last) moves = block_sum<EF_NT>(moves, s_sum);
    const uint32_t n = list_freed<EF_NT>(a, r, request_len(a, r), static_cast<uint32_t>(a.len[r]), before);
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

// Bound by memory: a thread asks for MV_AHEAD pieces of the keys and of the values at
// a time, past the caches.  64 requests, 8 heads of 128 in bf16, 90000 tokens: 155 us,
// 4.7 TB/s read and written, where a copy of 1 GiB reaches 5.1.
constexpr uint32_t MV_AHEAD = 2;

template <class U>
__global__ __launch_bounds__(MV_NT) void ev_move(MoveArgs a)
{
    const uint32_t r = blockIdx.x / a.per, row = a.heads * a.units;
    const uint32_t n = static_cast<uint32_t>(min(max(a.n_moves[r], 0), static_cast<int32_t>(a.cap)));
    const int2* moves = a.moves + r * a.moves_stride;
    const uint32_t step = a.per * MV_NT, i = blockIdx.x % a.per * MV_NT + threadIdx.x, mask = (1u << a.page_lg) - 1u;
    uint64_t j = i / row;  // the thread's move, and its piece of it
    uint32_t in = i % row;
    while (j < n) {
        U x[MV_AHEAD][2];
        char* to[MV_AHEAD][2];
#pragma unroll
        for (uint32_t k = 0; k < MV_AHEAD; ++k) {
            to[k][0] = to[k][1] = nullptr;
            if (j < n) {
                const uint32_t head = in / a.units, unit = in % a.units;
                const int2 move = moves[j];
                const uint32_t from = static_cast<uint32_t>(move.x), into = static_cast<uint32_t>(move.y);
                if (move.x >= 0 && move.y >= 0 && from < a.n_slots && into < a.n_slots) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint64_t off = head * a.head[c] + unit * sizeof(U);
                        x[k][c] = __builtin_nontemporal_load(reinterpret_cast<const U*>(
                            a.base[c] + (from >> a.page_lg) * a.page[c] + (from & mask) * a.slot[c] + off));
                        to[k][c] = a.base[c] + (into >> a.page_lg) * a.page[c] + (into & mask) * a.slot[c] + off;
                    }
                }
            }
            j += step / row;
            in += step % row;
            if (in >= row) {
                in -= row;
                ++j;
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < MV_AHEAD; ++k) {
            if (!to[k][0]) continue;
#pragma unroll
            for (int c = 0; c < 2; ++c) __builtin_nontemporal_store(x[k][c], reinterpret_cast<U*>(to[k][c]));
        }
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
    // What is written is read again behind it: not over the lengths that are asked.
    auto meets = [&](const int32_t* x) {
        auto over = [&](const int32_t* y) { return x && y && x < y + p.n_requests && y < x + p.n_requests; };
        return over(p.d_len) || over(p.d_n_moves);
    };
    if (meets(p.d_kv_len) || meets(p.d_keep) || meets(p.d_kept) || meets(p.d_seen)) {
        set_error("cr_paged_evict: invalid argument (the lengths that are written lie over those that are read)");
        return CR_ERR_INVALID;
    }
    auto rows = [&](const void* x, uint64_t stride) { return Rows(x, x ? p.n_requests : 0, stride * 4, 1, 0, room * 4); };
    if (rows_overwrite(rows(p.d_weights_out, p.weights_out_stride), rows(p.d_weights, p.weights_stride)) ||
        rows_overwrite(rows(p.d_positions_out, p.positions_out_stride), rows(p.d_positions, p.positions_stride))) {
        set_error("cr_paged_evict: invalid argument (the rows that are written lie over others of those that are read)");
        return CR_ERR_INVALID;
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
    auto four = [](const void* p, uint64_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 4 == 0; };
    a.wide = room >= 4 && room % 4 == 0 && four(p.d_weights, p.weights_stride) && four(p.d_weights_out, p.weights_out_stride) &&
             (!p.d_positions || four(p.d_positions, p.positions_stride)) &&
             (!p.d_positions_out || four(p.d_positions_out, p.positions_out_stride));
    // One workgroup a request while its entries fit the registers.
    const bool whole = room <= EV_WHOLE;
    a.segments = whole ? 0 : static_cast<uint32_t>((room + SG_SIZE - 1) / SG_SIZE);
    const uint64_t segments = static_cast<uint64_t>(a.segments) * p.n_requests;
    if (segments >> 23) {  // a launch holds fewer than 2^32 threads
        set_error("cr_paged_evict: too many positions for one call");
        return CR_ERR_UNSUPPORTED;
    }
    const bool direct = p.pinned && is_direct(p.pinned);
    // What the set can hold: slots behind are not pinned, and take no room where its bits are written out.
    uint64_t pin_end = n_slots;
    if (p.pinned && p.pinned->universe_size)
        pin_end = std::min(n_slots, (std::max<uint64_t>((p.pinned->universe_size - 1u) >> 16, p.pinned->max_key) + 1) << 16);
    const uint32_t n_words = static_cast<uint32_t>((pin_end + 31) / 32);
    Carver cv;
    const size_t o_keys = cv.add(segments * SG_SIZE * 4), o_open = cv.add(segments * SG_SIZE * 8);
    const size_t o_bins = cv.add(segments * EV_BINS * 2), o_counts = cv.add(segments * 16), o_from = cv.add(segments * 16);
    const size_t o_picked = cv.add(whole ? 0 : p.n_requests * 32ull);
    const size_t o_words = cv.add(p.pinned && !direct ? std::max<size_t>(4, n_words * 4ull) : 0);
    Scratch sc;
    if (cv.total) CR_RET(sc.alloc(cv.total, s));
    a.keys = sc.at<uint32_t>(o_keys);
    a.undecided = sc.at<uint2>(o_open);
    a.bins = sc.at<uint32_t>(o_bins);
    a.counts_of = sc.at<uint4>(o_counts);
    a.from = sc.at<uint4>(o_from);
    a.picked = sc.at<uint4>(o_picked);
    if (p.pinned)
        CR_RET(set_bits(p.pinned, direct, sc.at<uint32_t>(o_words), n_words, static_cast<uint32_t>(pin_end), stream,
                        &a.pinned));
    CR_TIMED("ev_pick", s);
    const uint32_t n = p.n_requests, parts = static_cast<uint32_t>(segments);
    // Four entries a thread while a workgroup has threads for them: fewer waves scan and wait faster
    // than idle ones (1003 entries 7.5 us, with 1024 threads 10; 512 requests of 2000, freed pages
    // included, 16, with 1024 threads 22.6, with 8 entries 17.4; 16 a thread cost 4 us).
    if (room <= 1024) {
        ev_pick<256, 4><<<n, 256, 0, s>>>(a);
    } else if (room <= 2048) {
        ev_pick<512, 4><<<n, 512, 0, s>>>(a);
    } else if (room <= 4096) {
        ev_pick<1024, 4><<<n, 1024, 0, s>>>(a);
    } else if (whole) {
        ev_pick<512, 32><<<n, 512, 0, s>>>(a);
    } else {
        sg_keys<<<parts, SG_NT, 0, s>>>(a);
        sg_digit<<<n, EV_NT, 0, s>>>(a);
        sg_split<<<parts, SG_NT, 0, s>>>(a);
        sg_decide<<<n, EV_NT, 0, s>>>(a);
        sg_place<<<parts, SG_NT, 0, s>>>(a);
    }
    const uint32_t per = whole ? 1 : a.segments;
    if (!whole || n > 1) ev_finish<<<n * per, EF_NT, 0, s>>>(a, per);
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
    // About 32 workgroups a CU, shared evenly by the requests, of which some have no moves.
    const uint64_t most = (moves_cap * row + MV_NT - 1) / MV_NT;
    a.per = static_cast<uint32_t>(std::min<uint64_t>(most, std::max(1u, 32 * num_cus() / n_requests)));
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

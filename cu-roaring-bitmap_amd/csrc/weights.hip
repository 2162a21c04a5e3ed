// Attention weights of a paged cache's tokens, for serving language models (no
// reference implementation): what eviction goes by.
//
//   out_i = (i is older than the rows counted, or a layer before has been: decay * past_i, else 0)
//           + sum over rows (t, h) that see i of e^(scale * q_th . k_i - lse_th)
//
// with the log-sums that the attention of the same rows left.
#include <algorithm>
#include <type_traits>

#include "internal.hpp"
#include "elements.hpp"
#include "rows.hpp"
#include "set_bits.hpp"
#include "weights_work.hpp"

namespace crimpl {

namespace {

constexpr uint32_t WT_DIM_MAX = 256;

typedef short v8s __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct Half : F16 {
    static __device__ __forceinline__ f32x4 mfma16(v8s x, v8s y, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), c, 0, 0,
                                                      0);
    }
    static __device__ __forceinline__ f32x16 mfma32(v8s x, v8s y, f32x16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), c, 0, 0,
                                                      0);
    }
};
struct BHalf : BF16 {
    static __device__ __forceinline__ f32x4 mfma16(v8s x, v8s y, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, x), __builtin_bit_cast(v8b, y), c, 0, 0,
                                                       0);
    }
    static __device__ __forceinline__ f32x16 mfma32(v8s x, v8s y, f32x16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, x), __builtin_bit_cast(v8b, y), c, 0, 0,
                                                       0);
    }
};

constexpr float LOG2E = 1.44269504088896340736f;

struct WeightArgs {
    const uint16_t* q;
    uint64_t q_token, q_head;
    const uint16_t* k;
    uint64_t k_page, k_slot, k_head;
    const float* lse;
    uint32_t n_tokens, heads, kv_heads, dim, n_requests;
    uint32_t n_pages, page_lg;
    const int32_t* starts;
    const int32_t* fresh;  // or nullptr: up to the next start
    const int32_t* kv_len;
    const int32_t* table;
    uint32_t cols;
    uint64_t table_stride;
    SetBits visible;
    bool gated;
    const float* past;
    uint64_t past_stride;
    float decay;
    float* out;
    uint64_t out_stride;
    float scale2;  // scale * log2(e)
    bool causal, continued;
    // Few rows: waves that share the heads, workgroups of a request, and how often a wave's LDS
    // is filled with positions that it looks up at once.
    uint32_t head_waves, spans, halves;
    // Many rows: parts of a request's rows, of part_rows or more each; tiles of positions
    // that the launch has for a request; and the sums of the `side` parts from part `first` on
    // (of the list: from entry `first` on) that the launch takes, [n_requests][side][key heads][room].
    uint32_t parts, part_rows, tiles, room, first, side;
    float* sums;
    // Requests of both kinds: the parts of those with many rows, (request, part of it) [max_listed],
    // each request's first of them (or NONE), how many there are, and the requests that have some.
    uint32_t few, max_listed;
    uint2* listed;
    uint32_t* first_of;
    uint32_t* counts;  // parts, requests
    uint32_t* many;    // [max_listed]
};
constexpr uint32_t NONE = 0xFFFFFFFFu;

struct Counted {  // a request's rows and positions
    uint32_t token0, tokens, keys;
    int64_t older;  // positions before the first counted token's
};

__device__ __forceinline__ Counted counted_of(const WeightArgs& a, uint32_t r)
{
    const int32_t n = static_cast<int32_t>(a.n_tokens);
    const int32_t t0 = min(max(a.starts[r], 0), n);
    const int32_t t1 = a.fresh ? t0 + min(max(a.fresh[r], 0), n - t0) : min(max(a.starts[r + 1], t0), n);
    const int32_t len = max(a.kv_len[r], 0);
    const uint64_t room = static_cast<uint64_t>(a.cols) << a.page_lg;
    return {static_cast<uint32_t>(t0), static_cast<uint32_t>(t1 - t0),
            static_cast<uint32_t>(min(room, static_cast<uint64_t>(len))), static_cast<int64_t>(a.kv_len[r]) - (t1 - t0)};
}

// 16 bytes a lane from memory to LDS, lane after lane from `to`, which is the same for the wave.
// ONCE: data that no other workgroup reads.
template <bool ONCE>
__device__ __forceinline__ void load_to_lds(const uint16_t* from, uint16_t* to)
{
    constexpr int NONTEMPORAL = 2;
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) const void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, ONCE ? NONTEMPORAL : 0);
}

// How rows lie in LDS: turned by pieces of 16 bytes so that the rows of a fragment share no
// banks.
template <uint32_t DIM>
struct Lines {
    static constexpr uint32_t CHUNKS = DIM <= 64 ? 8 : DIM <= 128 ? 16 : 32;  // 16-byte pieces of a row
    static constexpr uint32_t STRIDE = CHUNKS * 8;                             // its elements
    static constexpr uint32_t TURN = CHUNKS < 16 ? CHUNKS - 1 : 15;
};

// ---- few rows: bound by reading the keys -------------------------------------------------
// A workgroup per span of a request's positions.  Its waves share the key heads, and
// where there are fewer heads than waves the span; a wave takes the keys of its
// positions, one head after another, through LDS of its own, to which they go whole
// lines at a time and without passing through registers, and which hands them out as the
// columns of 16x16x32 products whose rows are the queries.  A product's 16 rows are not all
// used where fewer share a key head, which costs nothing: reading is what takes the time.
// 64 requests of up to 16384 positions, 8 key heads of 128 in bf16, groups of 4: 166 us,
// 6.5 TB/s (keys through registers and the caches 211, as they came 243; 16 KB of LDS a wave
// in place of 8, 174); one of 1003 positions: 6 us.
template <class E, uint32_t DIM>
__global__ __launch_bounds__(WR_NT) void wt_rows(WeightArgs a)
{
    using L = Lines<DIM>;
    constexpr uint32_t STEPS = DIM / 32, TILES = row_tiles(L::CHUNKS), COLS = TILES * 16;
    constexpr uint32_t PER = 64 / L::CHUNKS, LOADS = COLS / PER;  // rows that an instruction covers, instructions
    __shared__ alignas(16) uint16_t s_key[WR_WAVES][COLS * L::STRIDE];
    __shared__ uint64_t s_at[WR_WAVES][64];
    __shared__ uint32_t s_from[WR_WAVES][64];
    __shared__ float s_sum[WR_WAVES][64];
    const uint32_t lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15u, g = lane >> 4;
    const uint32_t r = blockIdx.x / a.spans, tile_waves = WR_WAVES / a.head_waves;
    const uint32_t head_wave = wave % a.head_waves, tile_wave = wave / a.head_waves;
    if (a.listed && a.first_of[r] != NONE) return;  // wt_tiles takes the request
    const Counted t = counted_of(a, r);
    const uint32_t group = a.heads / a.kv_heads, rows = t.tokens * group, per_wave = a.halves * COLS, step = tile_waves * per_wave;
    uint16_t* sk = s_key[wave];
    if (a.dim < DIM) {  // pieces behind the head dimension: zeros, as the queries that they meet
#pragma unroll
        for (uint32_t x = 0; x < LOADS; ++x) {
            const uint32_t row = x * PER + lane / L::CHUNKS, pos = lane % L::CHUNKS;
            if ((pos ^ (row & L::TURN)) * 8 >= a.dim) *reinterpret_cast<v8s*>(sk + row * L::STRIDE + pos * 8) = v8s{};
        }
    }
    // (more than once where the caller's most positions are fewer than there are)
    for (uint32_t first = blockIdx.x % a.spans * step; first < t.keys; first += a.spans * step) {
        // Lane l looks after position l of the wave's: where its keys lie, and the first row that
        // sees it, of rows numbered from 1.
        const uint32_t p0 = first + tile_wave * per_wave;
        if (lane < per_wave) {
            const uint32_t p = p0 + lane;
            uint64_t at = 0;
            uint32_t from = 0xFFFFFFFFu;
            if (p < t.keys) {
                const uint32_t page = static_cast<uint32_t>(a.table[r * a.table_stride + (p >> a.page_lg)]);
                const uint32_t off = p & ((1u << a.page_lg) - 1u), slot = (page << a.page_lg) + off;
                bool see = page < a.n_pages;
                if (see && a.gated) see = slot < a.visible.end && ((a.visible.word(slot >> 5) >> (slot & 31u)) & 1u);
                const int64_t token = a.causal ? max(static_cast<int64_t>(0), static_cast<int64_t>(p) - t.older) : 0;
                if (see && token < t.tokens) {
                    at = page * a.k_page + off * a.k_slot;
                    from = static_cast<uint32_t>(token) * group + 1;
                }
            }
            s_at[wave][lane] = at;
            s_from[wave][lane] = from;
        }
        wave_lds_fence();
        for (uint32_t half = 0; half < a.halves; ++half) {
            uint64_t at[LOADS];
            uint32_t on = 0, from[TILES];
            float sum[TILES], part[TILES];  // long sums in two steps, which lose less
#pragma unroll
            for (uint32_t x = 0; x < LOADS; ++x) {
                const uint32_t row = x * PER + lane / L::CHUNKS, d = (lane % L::CHUNKS ^ (row & L::TURN)) * 8;
                at[x] = s_at[wave][half * COLS + row] + d;
                on |= (s_from[wave][half * COLS + row] != 0xFFFFFFFFu && d < a.dim ? 1u : 0u) << x;
            }
            bool any = false;
#pragma unroll
            for (uint32_t i = 0; i < TILES; ++i) {
                from[i] = s_from[wave][half * COLS + i * 16 + c16];
                any = any || __ballot(from[i] != 0xFFFFFFFFu) != 0;
                sum[i] = part[i] = 0.0f;
            }
            for (uint32_t h = head_wave; any && h < a.kv_heads; h += a.head_waves) {
                const uint16_t* kp = a.k + h * a.k_head;
#pragma unroll
                for (uint32_t x = 0; x < LOADS; ++x)
                    if ((on >> x) & 1u) load_to_lds<true>(kp + at[x], sk + x * PER * L::STRIDE);
                for (uint32_t row0 = 0; row0 < rows; row0 += 16) {
                    v8s q[STEPS];
                    const uint32_t mine = min(row0 + c16, rows - 1);
                    const uint16_t* qp =
                        a.q + (t.token0 + mine / group) * a.q_token + (h * group + mine % group) * a.q_head;
#pragma unroll
                    for (uint32_t s = 0; s < STEPS; ++s) {
                        const uint32_t d = s * 32 + g * 8;
                        q[s] = d < a.dim ? *reinterpret_cast<const v8s*>(qp + d) : v8s{};
                    }
                    float lse2[4];
                    uint32_t number[4];  // 0: counts for nothing
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        const uint32_t at_row = row0 + g * 4 + e, row = min(at_row, rows - 1);
                        const float z = a.lse[static_cast<uint64_t>(t.token0 + row / group) * a.heads + h * group + row % group];
                        lse2[e] = z * LOG2E;  // (rounded: 1.3e-6 of a weight at a log-sum of 32, less below it)
                        number[e] = at_row < rows && z != -__builtin_inff() ? at_row + 1 : 0u;
                    }
                    // the wave's own keys are in LDS
                    if (row0 == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
                    for (uint32_t i = 0; i < TILES; ++i) {
                        f32x4 x = {0, 0, 0, 0};
                        const uint32_t row = i * 16 + c16;
#pragma unroll
                        for (uint32_t s = 0; s < STEPS; ++s) {
                            const v8s key = *reinterpret_cast<const v8s*>(sk + row * L::STRIDE + ((s * 4 + g) ^ (row & L::TURN)) * 8);
                            x = E::mfma16(q[s], key, x);
                        }
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) {
                            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], a.scale2, -lse2[e]));
                            part[i] += number[e] >= from[i] ? w : 0.0f;
                        }
                    }
                    if (row0 % 1024 == 1008 || row0 + 16 >= rows) {
#pragma unroll
                        for (uint32_t i = 0; i < TILES; ++i) {
                            sum[i] += part[i];
                            part[i] = 0.0f;
                        }
                    }
                }
                wave_lds_fence();  // its keys are read before the next head's arrive
            }
#pragma unroll
            for (uint32_t i = 0; i < TILES; ++i) {
                sum[i] += __shfl_xor(sum[i], 16, 64);
                sum[i] += __shfl_xor(sum[i], 32, 64);
                if (g == 0) s_sum[wave][half * COLS + i * 16 + c16] = sum[i];
            }
        }
        __syncthreads();
        // the heads' sums joined in a fixed order
        for (uint32_t i = threadIdx.x; i < step; i += WR_NT) {
            const uint32_t p = first + i, of = i / per_wave, in = i % per_wave;
            if (p >= t.keys) break;
            float all = 0.0f;
            for (uint32_t w = 0; w < a.head_waves; ++w) all += s_sum[of * a.head_waves + w][in];
            const float past =
                a.past && (a.continued || static_cast<int64_t>(p) < t.older) ? a.past[r * a.past_stride + p] * a.decay : 0.0f;
            a.out[r * a.out_stride + p] = past + all;
        }
        __syncthreads();
    }
}

// ---- many rows ------------------------------------------------------------------------
// A workgroup takes a part of a request's rows, one key head and a tile of 256
// positions, 64 a wave, whose keys stay in registers as the columns of 32x32x16
// products; the queries pass by through LDS, 64 rows at a time, where the next ones
// arrive meanwhile without passing through registers.  A lane sums what its two
// columns get; the parts' sums are joined by another kernel, heads and parts in order.
// Bound by the matrix units and the exponential of each product beside them: a prompt of
// 16384 tokens, 8 key heads of 128, groups of 4, takes 1.13 ms, 970 TFLOP/s (1.18 with two
// waves a SIMD, 1.27 with every row tested for what it sees).
__device__ __attribute__((aligned(16))) uint16_t wt_zeros[WT_DIM_MAX];
constexpr uint32_t WT_ROWS = 64;   // rows that arrive at a time

template <uint32_t DIM>
struct Stage : Lines<DIM> {
    static constexpr uint32_t PER = WT_NT / Lines<DIM>::CHUNKS, LOADS = WT_ROWS / PER;  // rows that the workgroup loads at once
};

// The first row that sees a position, at or behind all that its tokens are.
__device__ __forceinline__ int64_t first_row(const WeightArgs& a, const Counted& t, uint32_t p, uint32_t group)
{
    return a.causal ? max(static_cast<int64_t>(0), static_cast<int64_t>(p) - t.older) * group : 0;
}

// The rows of each of a request's parts.
__device__ __forceinline__ uint32_t part_size(const WeightArgs& a, uint32_t rows)
{
    return max(a.part_rows, ((rows + a.parts - 1) / a.parts + 63u) / 64u * 64u);
}

// The rows [first, end) of part i that a tile whose first position is p counts.
__device__ __forceinline__ void rows_of_part(const WeightArgs& a, const Counted& t, uint32_t p, uint32_t group, uint32_t i,
                                             uint32_t& first, uint32_t& end)
{
    const uint32_t rows = t.tokens * group, size = part_size(a, rows);
    const uint64_t from = static_cast<uint64_t>(i) * size;
    const uint64_t sees = static_cast<uint64_t>(first_row(a, t, p, group)) / 32 * 32;
    end = static_cast<uint32_t>(min(static_cast<uint64_t>(rows), from + size));
    first = static_cast<uint32_t>(min(static_cast<uint64_t>(end), max(from, sees)));
}

// LISTED: where a bitmap leaves positions out, the seen ones of a tile are put side by side first, so
// that nothing is worked out for the others (8 requests of 100 tokens and 8192 positions, 96
// dimensions: with 60% of them seen 2 us less of 38, with 30% 6 of 36; a prompt of 8192 with 30%
// 193 us, not 280).  Where a wave has one block anyway, above 192 dimensions, it would gain little and
// the lists cost 7% with 60% seen.
template <class E, uint32_t DIM, bool LISTED>
__global__ __launch_bounds__(WT_NT) __attribute__((amdgpu_waves_per_eu(DIM <= 128 ? 3 : 2))) void wt_tiles(WeightArgs a)
{
    using S = Stage<DIM>;
    constexpr uint32_t STEPS = DIM / 16, NB = tile_blocks(DIM), COLS = tile_cols(DIM);
    // separate arrays: what is read is not what is being loaded
    __shared__ alignas(16) uint16_t s_q0[WT_ROWS * S::STRIDE], s_q1[WT_ROWS * S::STRIDE];
    __shared__ uint64_t s_at[4][WT_ROWS];
    __shared__ alignas(16) float s_lse[4][WT_ROWS];
    __shared__ uint64_t s_key[LISTED ? COLS : 1];  // where the seen positions' keys are, and the positions
    __shared__ uint32_t s_col[LISTED ? COLS : 1], s_seen[WT_NT / 64];
    const uint32_t lane = __lane_id(), wave = threadIdx.x >> 6, c32 = lane & 31u, h = lane >> 5;
    const uint32_t kh = blockIdx.x % a.kv_heads, part = blockIdx.x / a.kv_heads / a.tiles;
    if (a.listed && a.first + part >= a.counts[0]) return;
    const uint2 of = a.listed ? a.listed[a.first + part] : make_uint2(part / a.side, a.first + part % a.side);
    const uint32_t r = of.x, group = a.heads / a.kv_heads;
    const Counted t = counted_of(a, r);
    const uint32_t rows = t.tokens * group;
    const uint32_t lrow = threadIdx.x / S::CHUNKS, lpos = threadIdx.x % S::CHUNKS;
    const uint32_t wave_row = __builtin_amdgcn_readfirstlane(wave) * (64 / S::CHUNKS);
    if (a.dim < DIM) {  // pieces behind the head dimension: zeros, as the keys that they meet
#pragma unroll
        for (uint32_t x = 0; x < S::LOADS; ++x) {
            const uint32_t lr = x * S::PER + lrow, at = lr * S::STRIDE + lpos * 8;
            if ((lpos ^ (lr & S::TURN)) * 8 >= a.dim) {
                *reinterpret_cast<v8s*>(s_q0 + at) = v8s{};
                *reinterpret_cast<v8s*>(s_q1 + at) = v8s{};
            }
        }
    }
    // (more than once where the caller's most positions are fewer than there are)
    for (uint32_t first = blockIdx.x / a.kv_heads % a.tiles * COLS; first < t.keys; first += a.tiles * COLS) {
        uint32_t row0, row1;
        rows_of_part(a, t, first, group, of.y, row0, row1);
        if (row0 >= row1) continue;
        // Whether one of the rows sees position p, and where its keys lie.
        auto look_up = [&](uint32_t p, uint32_t page, uint64_t& at) __attribute__((always_inline)) {
            const uint32_t off = p & ((1u << a.page_lg) - 1u), slot = (page << a.page_lg) + off;
            bool see = p < t.keys && page < a.n_pages && first_row(a, t, p, group) < row1;
            if ((LISTED || a.gated) && see) see = slot < a.visible.end && ((a.visible.word(slot >> 5) >> (slot & 31u)) & 1u);
            at = see ? page * a.k_page + off * a.k_slot : 0;
            return see;
        };
        auto page_of = [&](uint32_t p) __attribute__((always_inline)) {
            return static_cast<uint32_t>(a.table[r * a.table_stride + (min(p, t.keys - 1) >> a.page_lg)]);
        };
        auto sum_at = [&](uint32_t p) __attribute__((always_inline)) -> float& {
            return a.sums[(static_cast<uint64_t>(part) * a.kv_heads + kh) * a.room + p];
        };
        // The lane's columns: as the positions lie, or, where a bitmap leaves some out, the ones that
        // are seen side by side, in blocks of 32 that the waves take in turn.
        uint32_t page[NB];
        bool mine_seen = false;
        uint64_t mine_at = 0;
        const uint32_t mine = first + threadIdx.x;
        if constexpr (LISTED) {
            if (threadIdx.x < COLS) mine_seen = look_up(mine, page_of(mine), mine_at);
            if (threadIdx.x < COLS && mine < t.keys && !mine_seen) sum_at(mine) = 0.0f;
        } else {
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) page[b] = page_of(first + (wave * NB + b) * 32 + c32);
        }

        // Where a stage's rows are, and their log-sums: lane l looks after row l.
        const uint32_t n_stages = (row1 - row0 + WT_ROWS - 1) / WT_ROWS;
        auto note = [&](uint32_t i) __attribute__((always_inline)) {
            const uint32_t row = min(row0 + i * WT_ROWS + lane, rows - 1);
            const uint64_t token = t.token0 + row / group;
            const uint32_t head = kh * group + row % group;
            const float z = a.lse[token * a.heads + head];
            const bool none = z == -__builtin_inff();  // counts for nothing, whatever it holds
            const uint16_t* at = none ? wt_zeros : a.q + token * a.q_token + head * a.q_head;
            s_at[i % 4][lane] = reinterpret_cast<uint64_t>(at);
            // (rounded: 1.3e-6 of a weight at a log-sum of 32, less below it; what the product loses, given back,
            // would be an operation more for each exponential)
            s_lse[i % 4][lane] = none ? __builtin_inff() : z * LOG2E;
        };
        auto load = [&](uint32_t i, uint16_t* sq) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t x = 0; x < S::LOADS; ++x) {
                const uint32_t lr = x * S::PER + lrow, d = (lpos ^ (lr & S::TURN)) * 8;
                if (d < a.dim)
                    load_to_lds<false>(reinterpret_cast<const uint16_t*>(s_at[i % 4][lr]) + d,
                                       sq + (x * S::PER + wave_row) * S::STRIDE);
            }
        };
        auto load_key = [&](v8s (&to)[STEPS], const uint16_t* of, bool on) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t st = 0; st < STEPS; ++st) {
                const uint32_t d = st * 16 + h * 8;
                to[st] = on && d < a.dim ? *reinterpret_cast<const v8s*>(of + kh * a.k_head + d) : v8s{};
            }
        };
        __syncthreads();  // the tile before is done with LDS
        v8s key[NB][STEPS];
        uint32_t from[NB], latest = 0;  // the first row that sees the lane's positions, if any
        uint32_t turn = 0, n_mine = 0;
        bool none = false;
        if constexpr (LISTED) {
            const unsigned long long seen = __ballot(mine_seen);
            if (lane == 0) s_seen[wave] = static_cast<uint32_t>(__popcll(seen));
            __syncthreads();
            uint32_t total = 0, before = 0;
#pragma unroll
            for (uint32_t w = 0; w < WT_NT / 64; ++w) {
                before += w < wave ? s_seen[w] : 0u;
                total += s_seen[w];
            }
            if (mine_seen) {
                const uint32_t i = before + static_cast<uint32_t>(__popcll(seen & ((1ull << lane) - 1ull)));
                s_col[i] = mine;
                s_key[i] = mine_at;
            }
            __syncthreads();
            total = __builtin_amdgcn_readfirstlane(total);
            none = total == 0;
            turn = __builtin_amdgcn_readfirstlane((wave + blockIdx.x) % 4);
            n_mine = (total + 31) / 32 > turn ? ((total + 31) / 32 - turn + 3) / 4 : 0u;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const uint32_t c = (turn + 4 * b) * 32 + c32;
                from[b] = c < total ? static_cast<uint32_t>(first_row(a, t, s_col[c], group)) : 0xFFFFFFFFu;
                load_key(key[b], a.k + (c < total ? s_key[c] : 0), c < total);
            }
        } else {
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const uint32_t p = first + (wave * NB + b) * 32 + c32;
                uint64_t at;
                const bool see = look_up(p, page[b], at);
                from[b] = see ? static_cast<uint32_t>(first_row(a, t, p, group)) : 0xFFFFFFFFu;
                if (__ballot(see)) n_mine = NB;
                load_key(key[b], a.k + at, see);
            }
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) latest = max(latest, from[b] != 0xFFFFFFFFu ? from[b] : 0u);
        if (wave < 2) note(wave);
        if (LISTED) __syncthreads();
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) latest = max(latest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(latest), o, 64)));
        latest = __builtin_amdgcn_readfirstlane(latest);
        float sum[NB] = {};
        const uint32_t q_at = c32 * S::STRIDE + (h ^ (c32 & S::TURN)) * 8;  // of step st: q_at ^ st * 16
        auto add = [&](const auto& x, const f32x4 (&z)[4], auto counts) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t b = 0; b < sizeof(x) / sizeof(f32x16); ++b) {
                float w[16];
#pragma unroll
                for (uint32_t e = 0; e < 16; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[b][e], a.scale2, -z[e / 4][e % 4]));
                    if (!counts(b, e)) w[e] = 0.0f;
                }
#pragma unroll
                for (uint32_t o = 8; o > 0; o >>= 1)
#pragma unroll
                    for (uint32_t e = 0; e < o; ++e) w[e] += w[e + o];
                sum[b] += w[0];
            }
        };
        auto multiply_by = [&](uint32_t i, const uint16_t* sq, auto n_of) __attribute__((always_inline)) {
            constexpr uint32_t N = decltype(n_of)::value;
#pragma unroll
            for (uint32_t y = 0; y < WT_ROWS / 32; ++y) {
                const uint32_t base = row0 + i * WT_ROWS + y * 32;
                if (base >= row1) break;
                f32x16 x[N];
#pragma unroll
                for (uint32_t b = 0; b < N; ++b)
#pragma unroll
                    for (uint32_t e = 0; e < 16; ++e) x[b][e] = 0.0f;
                // Three waves a SIMD leave 128 dimensions no registers to keep all addresses in: the
                // second half's are worked out from the first's.
                uint32_t half = DIM == 128 ? 64u : 0u;
                if constexpr (DIM == 128) asm volatile("" : "+v"(half));
#pragma unroll
                for (uint32_t st = 0; st < STEPS; ++st) {
                    const v8s q = *reinterpret_cast<const v8s*>(
                        sq + y * 32 * S::STRIDE +
                        (DIM == 128 && st >= 4 ? (q_at ^ (st * 16 - 64)) ^ half : q_at ^ (st * 16)));
#pragma unroll
                    for (uint32_t b = 0; b < N; ++b) x[b] = E::mfma32(q, key[b][st], x[b]);
                }
                f32x4 z[4];
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    z[e] = *reinterpret_cast<const f32x4*>(&s_lse[i % 4][y * 32 + e * 8 + h * 4]);
                // Apart, so that rows which all see all are not tested one by one.
                if (base >= latest && base + 32 <= row1)
                    add(x, z, [](uint32_t, uint32_t) { return true; });
                else
                    add(x, z, [&](uint32_t b, uint32_t e) {
                        const uint32_t row = base + e / 4 * 8 + h * 4 + e % 4;
                        return row >= from[b] && row < row1;
                    });
            }
        };
        auto multiply = [&](uint32_t i, const uint16_t* sq) __attribute__((always_inline)) {
            if (n_mine == NB)
                multiply_by(i, sq, std::integral_constant<uint32_t, NB>{});
            else if (LISTED && n_mine)
                multiply_by(i, sq, std::integral_constant<uint32_t, 1>{});
        };
        if (!LISTED) __syncthreads();  // (the rows' places are noted)
        if (!none) load(0, s_q0);
        // Each wave waits for its own loads to LDS before all meet.
        auto arrived = [&]() __attribute__((always_inline)) {
            __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
            __syncthreads();
        };
        for (uint32_t i = 0; !none && i < n_stages; i += 2) {
            arrived();
            if (i + 1 < n_stages) load(i + 1, s_q1);
            if (wave == 2 && i + 2 < n_stages) note(i + 2);
            multiply(i, s_q0);
            if (i + 1 >= n_stages) break;
            arrived();
            if (i + 2 < n_stages) load(i + 2, s_q0);
            if (wave == 3 && i + 3 < n_stages) note(i + 3);
            multiply(i + 1, s_q1);
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            sum[b] += __shfl_xor(sum[b], 32, 64);
            const uint32_t p = LISTED ? s_col[(turn + 4 * b) * 32 + c32] : first + (wave * NB + b) * 32 + c32;
            if (h == 0 && (LISTED ? from[b] != 0xFFFFFFFFu : p < t.keys)) sum_at(p) = from[b] != 0xFFFFFFFFu ? sum[b] : 0.0f;
        }
    }
}

// The parts' sums joined: 64 positions a workgroup, whose waves share the heads and
// parts.  LISTED: of the listed requests, `side` at a time.  Four waves, of which many
// fit a CU: 8 requests of 100 tokens and 8192 positions take 34.5 us in all, with sixteen
// 37.7; a prompt of 2048, whose positions have 64 sums each, 47.6, with eight 45.1, with
// two 53.3.
constexpr int WJ_NT = 256;

// What rows [first, end) of key head kh give seen position p, row by row: those whose log-sum is
// -inf nothing, whatever the position's key holds.
template <class E>
__device__ float sum_of_rows(const WeightArgs& a, const Counted& t, uint32_t r, uint32_t p, uint32_t kh, uint32_t first, uint32_t end)
{
    const uint32_t group = a.heads / a.kv_heads, page = static_cast<uint32_t>(a.table[r * a.table_stride + (p >> a.page_lg)]);
    const uint16_t* key = a.k + page * a.k_page + (p & ((1u << a.page_lg) - 1u)) * a.k_slot + kh * a.k_head;
    float sum = 0.0f;
    if (page >= a.n_pages) return sum;
    for (int64_t row = max(static_cast<int64_t>(first), first_row(a, t, p, group)); row < end && sum == sum; ++row) {
        const uint64_t token = t.token0 + static_cast<uint32_t>(row) / group;
        const uint32_t head = kh * group + static_cast<uint32_t>(row) % group;
        const float z = a.lse[token * a.heads + head];
        if (z == -__builtin_inff()) continue;
        const uint16_t* q = a.q + token * a.q_token + head * a.q_head;
        float x = 0.0f;
        for (uint32_t d = 0; d < a.dim; ++d) x = __builtin_fmaf(E::up(q[d]), E::up(key[d]), x);
        sum += __builtin_amdgcn_exp2f(__builtin_fmaf(x, a.scale2, -(z * LOG2E)));
    }
    return sum;
}

template <class E, bool LISTED>
__global__ __launch_bounds__(WJ_NT) void wt_join(WeightArgs a, uint32_t per_request, uint32_t side, uint32_t cols)
{
    constexpr uint32_t WAVES = WJ_NT / 64;
    __shared__ float s_sum[WAVES][64];
    const uint32_t lane = __lane_id(), wave = threadIdx.x >> 6, group = a.heads / a.kv_heads;
    const uint32_t n_requests = LISTED ? a.counts[1] : a.n_requests;
    for (uint32_t k = blockIdx.x / per_request; k < n_requests; k = LISTED ? k + side : n_requests) {
        const uint32_t r = LISTED ? a.many[k] : k;
        const Counted t = counted_of(a, r);
        const uint32_t rows = t.tokens * group, size = part_size(a, rows);
        // The request's parts that this launch has sums of, which lie from part `at` on.
        uint32_t lo = a.first, hi = min((rows + size - 1) / size, a.first + a.side);  // (those behind have no rows)
        uint64_t at = static_cast<uint64_t>(r) * a.side;
        bool begins = a.first == 0;  // the launch has the first of them
        if (LISTED) {
            const uint32_t part0 = a.first_of[r];
            begins = part0 >= a.first;
            lo = begins ? 0u : a.first - part0;
            hi = part0 >= a.first + a.side ? 0u : min((rows + size - 1) / size, a.first + a.side - part0);
            if (lo >= hi) continue;
            at = begins ? part0 - a.first : 0u;
        }
        hi = max(lo, hi);
        for (uint32_t p0 = blockIdx.x % per_request * 64; p0 < t.keys; p0 += per_request * 64) {
            const uint32_t p = p0 + lane;
            float sum = 0.0f;
            uint32_t skip = lo;  // parts that see nothing of the position's tile: the first ones
            for (uint32_t first, end; skip < hi; ++skip) {
                rows_of_part(a, t, p0 / cols * cols, group, skip, first, end);
                if (first < end) break;
            }
            if (p < t.keys)
#pragma unroll 4
                for (uint32_t i = (skip - lo) * a.kv_heads + wave; i < (hi - lo) * a.kv_heads; i += WAVES)
                    sum += a.sums[(at * a.kv_heads + i) * a.room + p];
            // Not a number: the key holds something that wt_tiles has multiplied rows which count for nothing
            // with too.  (A test a product there would cost registers that three waves a SIMD do not have.)
            if (sum != sum) {
                sum = 0.0f;
                for (uint32_t i = (skip - lo) * a.kv_heads + wave; i < (hi - lo) * a.kv_heads; i += WAVES) {
                    float more = a.sums[(at * a.kv_heads + i) * a.room + p];
                    if (more != more) {
                        uint32_t first, end;
                        rows_of_part(a, t, p0 / cols * cols, group, lo + i / a.kv_heads, first, end);
                        more = sum_of_rows<E>(a, t, r, p, i % a.kv_heads, first, end);
                    }
                    sum += more;
                }
            }
            s_sum[wave][lane] = sum;
            __syncthreads();
            if (wave == 0 && p < t.keys) {
                float all = 0.0f;
#pragma unroll
                for (uint32_t w = 0; w < WAVES; ++w) all += s_sum[w][lane];
                const float past =
                    !begins ? a.out[r * a.out_stride + p]
                    : a.past && (a.continued || static_cast<int64_t>(p) < t.older) ? a.past[r * a.past_stride + p] * a.decay : 0.0f;
                a.out[r * a.out_stride + p] = past + all;
            }
            __syncthreads();
        }
    }
}

// Lists the parts of the requests with many rows, a workgroup's work.  What the list has no room for,
// where requests count the same rows, stays with wt_rows.  255 single tokens and 2048 of one
// prompt, 4096 positions each, take 408 us in all, by wt_rows alone 2190, by wt_tiles alone 674.
constexpr int WS_NT = 1024;

__global__ __launch_bounds__(WS_NT) void wt_split(WeightArgs a)
{
    __shared__ uint32_t s_scan[WS_NT / 64], s_end;
    const uint32_t group = a.heads / a.kv_heads;
    uint32_t parts = 0, requests = 0;
    if (threadIdx.x == 0) s_end = 0;
    __syncthreads();
    for (uint32_t r0 = 0; r0 < a.n_requests; r0 += WS_NT) {
        const uint32_t r = r0 + threadIdx.x;
        uint32_t n = 0, total, here;
        if (r < a.n_requests) {
            const uint32_t rows = counted_of(a, r).tokens * group;
            n = rows > a.few ? (rows + a.part_rows - 1) / a.part_rows : 0u;
            n = n <= a.max_listed ? n : 0u;
        }
        const uint32_t first = parts + block_excl_scan<WS_NT>(n, s_scan, total);
        const bool fits = n && first + n <= a.max_listed;
        const uint32_t k = requests + block_excl_scan<WS_NT>(fits ? 1u : 0u, s_scan, here);
        if (r < a.n_requests) a.first_of[r] = fits ? first : NONE;
        if (fits) {
            a.many[k] = r;
            for (uint32_t i = 0; i < n; ++i) a.listed[first + i] = make_uint2(r, i);
        }
        if (fits) atomicMax(&s_end, first + n);  // (behind one that does not fit none does)
        parts = min(parts + total, a.max_listed + 1);
        requests += here;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        a.counts[0] = s_end;
        a.counts[1] = requests;
    }
}

template <class E, uint32_t DIM>
void launch_dim(const WeightArgs& a, uint32_t grid, hipStream_t s)
{
    if (!a.sums) {
        wt_rows<E, DIM><<<grid, WR_NT, 0, s>>>(a);
        return;
    }
    if constexpr (tile_blocks(DIM) == 2) {
        if (a.gated) {
            wt_tiles<E, DIM, true><<<grid, WT_NT, 0, s>>>(a);
            return;
        }
    }
    wt_tiles<E, DIM, false><<<grid, WT_NT, 0, s>>>(a);
}

template <class E>
void launch_weights(const WeightArgs& a, uint32_t grid, hipStream_t s)
{
    if (a.dim <= 64)
        launch_dim<E, 64>(a, grid, s);
    else if (a.dim <= 96)
        launch_dim<E, 96>(a, grid, s);
    else if (a.dim <= 128)
        launch_dim<E, 128>(a, grid, s);
    else if (a.dim <= 192)
        launch_dim<E, 192>(a, grid, s);
    else
        launch_dim<E, 256>(a, grid, s);
}

}  // namespace

}  // namespace crimpl

using namespace crimpl;

extern "C" int cr_paged_weights(const cr_paged_weights_args* args, const cr_paged_cache* cache, cr_stream_t stream)
{
    if (!args || !cache) {
        set_error("cr_paged_weights: invalid argument");
        return CR_ERR_INVALID;
    }
    const cr_paged_weights_args& p = *args;
    if (p.n_requests == 0) return CR_OK;
    if (!power_of_two(cache->page_size)) {
        set_error("cr_paged_weights: invalid argument (page size %u)", cache->page_size);
        return CR_ERR_INVALID;
    }
    const uint64_t n_slots = static_cast<uint64_t>(cache->n_pages) * cache->page_size;
    const uint64_t room = static_cast<uint64_t>(p.table_cols) * cache->page_size;
    if (!p.d_starts || !p.d_kv_len || (p.n_tokens && (!p.q || !p.lse)) || cache->n_heads == 0 || p.n_heads == 0 ||
        p.n_heads % cache->n_heads || cache->head_dim == 0 || (cache->n_pages && !cache->k) ||
        p.table_stride < p.table_cols || (room && (!p.d_table || !p.d_out)) || p.out_stride < room ||
        (p.d_past && p.past_stride < room)) {
        set_error("cr_paged_weights: invalid argument (%u query heads, %u key heads; a row holds table_cols * page_size "
                  "weights)", p.n_heads, cache->n_heads);
        return CR_ERR_INVALID;
    }
    // The strides that lead anywhere: that of an axis of one entry may be any number.
    auto over = [](uint32_t extent, uint64_t x) { return extent > 1 ? x : 0; };
    const uint64_t strides = over(p.n_tokens, p.q_token_stride) | over(p.n_heads, p.q_head_stride) |
                             over(cache->n_pages, cache->k_page_stride) | over(cache->page_size, cache->k_slot_stride) |
                             over(cache->n_heads, cache->k_head_stride) | cache->head_dim;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(cache->k);
    if ((cache->dtype != CR_F16 && cache->dtype != CR_BF16) || cache->head_dim > WT_DIM_MAX || strides % 8 || at % 16) {
        set_error("cr_paged_weights: f16 or bf16 rows of at most %u dimensions (a multiple of 8), 16-byte aligned, are "
                  "supported (type %u, %u dimensions)", WT_DIM_MAX, cache->dtype, cache->head_dim);
        return CR_ERR_UNSUPPORTED;
    }
    if (n_slots >> 31 || room >> 31 || p.n_tokens >> 31 || p.n_heads > 65535 || p.n_requests >> 22 ||
        (static_cast<uint64_t>(p.n_tokens) * p.n_heads) >> 31 || (room * p.n_requests) >> 36) {
        set_error("cr_paged_weights: supported up to 2^31 - 1 slots, positions and rows, 65535 heads, 2^22 - 1 requests and "
                  "2^36 - 1 weights");
        return CR_ERR_UNSUPPORTED;
    }
    auto rows = [&](const void* x, uint64_t stride) { return Rows(x, x ? p.n_requests : 0, stride * 4, 1, 0, room * 4); };
    if (rows_overwrite(rows(p.d_out, p.out_stride), rows(p.d_past, p.past_stride))) {
        set_error("cr_paged_weights: invalid argument (the weights that are written lie over others of those that are read)");
        return CR_ERR_INVALID;
    }
    WeightArgs a{};
    a.q = static_cast<const uint16_t*>(p.q);
    a.q_token = p.q_token_stride;
    a.q_head = p.q_head_stride;
    a.k = static_cast<const uint16_t*>(cache->k);
    a.k_page = cache->k_page_stride;
    a.k_slot = cache->k_slot_stride;
    a.k_head = cache->k_head_stride;
    a.lse = p.lse;
    a.n_tokens = p.n_tokens;
    a.heads = p.n_heads;
    a.kv_heads = cache->n_heads;
    a.dim = cache->head_dim;
    a.n_requests = p.n_requests;
    a.n_pages = cache->n_pages;
    a.page_lg = static_cast<uint32_t>(__builtin_ctz(cache->page_size));
    a.starts = p.d_starts;
    a.fresh = p.d_new;
    a.kv_len = p.d_kv_len;
    a.table = p.d_table;
    a.cols = p.table_cols;
    a.table_stride = p.table_stride;
    a.gated = p.visible != nullptr;
    a.past = p.d_past;
    a.past_stride = p.past_stride;
    a.decay = p.decay;
    a.out = p.d_out;
    a.out_stride = p.out_stride;
    a.scale2 = static_cast<float>(static_cast<double>(p.scale) * 1.44269504088896340736);
    a.causal = p.causal != 0;
    a.continued = p.continued != 0;
    a.room = static_cast<uint32_t>(room);
    if (room == 0) return CR_OK;
    const WeightsWork w = weights_work({p.n_tokens, p.n_heads, cache->n_heads, cache->head_dim, p.n_requests, room, p.max_new,
                                        p.max_kv, p.d_new != nullptr, num_cus()});
    a.few = w.few;
    a.head_waves = w.head_waves;
    a.halves = w.halves;
    a.spans = w.spans;
    a.part_rows = w.part_rows;
    a.parts = w.mixed ? 1u << 30 : w.parts;  // (of listed requests as many as the rows need)
    a.side = w.side;
    a.tiles = w.tiles;
    a.max_listed = w.parts;
    Carver cv;
    const size_t o_sums = cv.add(w.sums * 4), o_listed = cv.add(w.mixed ? w.parts * 8ull : 0);
    const size_t o_many = cv.add(w.mixed ? w.parts * 4ull + 16 : 0), o_first = cv.add(w.mixed ? p.n_requests * 4ull : 0);
    hipStream_t s = as_stream(stream);
    const bool direct = p.visible && is_direct(p.visible);
    const uint32_t n_words = static_cast<uint32_t>((n_slots + 31) / 32);
    const size_t o_words = cv.add(p.visible && !direct ? std::max<size_t>(4, n_words * 4ull) : 0);
    Scratch sc;
    if (cv.total) CR_RET(sc.alloc(cv.total, s));
    if (p.visible)
        CR_RET(set_bits(p.visible, direct, sc.at<uint32_t>(o_words), n_words, static_cast<uint32_t>(n_slots), stream,
                        &a.visible));
    if (w.mixed) {
        a.listed = sc.at<uint2>(o_listed);
        a.counts = sc.at<uint32_t>(o_many);
        a.many = a.counts + 4;
        a.first_of = sc.at<uint32_t>(o_first);
        CR_TIMED("wt_split", s);
        wt_split<<<1, WS_NT, 0, s>>>(a);
    }
    auto launch = [&](const WeightArgs& a, uint32_t workgroups) {
        if (cache->dtype == CR_F16)
            launch_weights<Half>(a, workgroups, s);
        else
            launch_weights<BHalf>(a, workgroups, s);
    };
    auto join = [&](const WeightArgs& a, uint32_t side, auto type) {
        using E = decltype(type);
        const uint32_t grid = w.join_per_request * side, cols = tile_cols(a.dim);
        if (w.mixed)
            wt_join<E, true><<<grid, WJ_NT, 0, s>>>(a, w.join_per_request, side, cols);
        else
            wt_join<E, false><<<grid, WJ_NT, 0, s>>>(a, w.join_per_request, side, cols);
    };
    if (!w.many) {
        CR_TIMED("wt_rows", s);
        launch(a, w.rows_grid);
    }
    if (w.side) a.sums = sc.at<float>(o_sums);
    for (uint32_t r = 0; w.side && r < p.n_requests; r += w.mixed ? p.n_requests : w.batch) {
        WeightArgs b = a;  // of requests from r on
        uint32_t at_once = w.join_side, grid = w.tiles_grid;
        if (w.many) {
            b.starts += r;
            if (b.fresh) b.fresh += r;
            b.kv_len += r;
            b.table += r * b.table_stride;
            if (b.past) b.past += r * b.past_stride;
            b.out += r * b.out_stride;
            b.n_requests = at_once = std::min(w.batch, p.n_requests - r);
            grid = grid / w.batch * at_once;
        }
        for (b.first = 0; b.first < w.parts; b.first += w.side) {
            {
                CR_TIMED("wt_tiles", s);
                launch(b, grid);
            }
            CR_TIMED("wt_join", s);
            if (cache->dtype == CR_F16)
                join(b, at_once, Half{});
            else
                join(b, at_once, BHalf{});
        }
    }
    CR_LAUNCH_CHECK();
    return CR_OK;
}

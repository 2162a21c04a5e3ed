// Attention weights of a paged cache's tokens, for serving language models (no
// reference implementation): what eviction goes by.
//
//   out_i = (i is older than the rows counted, or a layer before has been: decay * past_i, else 0)
//           + sum over rows (t, h) that see i of e^(scale * q_th . k_i - lse_th)
//
// with the log-sums that the attention of the same rows left.
#include <algorithm>

#include "internal.hpp"
#include "set_bits.hpp"

namespace crimpl {

namespace {

constexpr uint32_t WT_DIM_MAX = 256;

typedef short v8s __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Half {
    static __device__ __forceinline__ f32x4 mfma16(v8s x, v8s y, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), c, 0, 0,
                                                      0);
    }
};
struct BHalf {
    static __device__ __forceinline__ f32x4 mfma16(v8s x, v8s y, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, x), __builtin_bit_cast(v8b, y), c, 0, 0,
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
    uint32_t head_waves, spans;  // waves that share the heads; workgroups of a request
};

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

constexpr int WR_NT = 256;
constexpr uint32_t WR_WAVES = WR_NT / 64;
constexpr uint32_t WR_TILES = 4;  // of 16 positions, a wave's

// A workgroup per span of a request's positions.  Its waves share the key heads, and
// where there are fewer heads than waves the span; a wave keeps the keys of its
// positions in registers, one head after another, as the columns of 16x16x32 products
// whose rows are the queries.
template <class E, uint32_t DIM>
__global__ __launch_bounds__(WR_NT) void wt_rows(WeightArgs a)
{
    constexpr uint32_t STEPS = DIM / 32;
    __shared__ float s_sum[WR_WAVES][WR_TILES * 16];
    const uint32_t lane = __lane_id(), wave = threadIdx.x >> 6, c16 = lane & 15u, g = lane >> 4;
    const uint32_t r = blockIdx.x / a.spans, tile_waves = WR_WAVES / a.head_waves;
    const uint32_t head_wave = wave % a.head_waves, tile_wave = wave / a.head_waves;
    const Counted t = counted_of(a, r);
    const uint32_t group = a.heads / a.kv_heads, rows = t.tokens * group, step = tile_waves * WR_TILES * 16;
    // (more than once where the caller's most positions are fewer than there are)
    for (uint32_t first = blockIdx.x % a.spans * step; first < t.keys; first += a.spans * step) {
        const uint32_t p0 = first + tile_wave * WR_TILES * 16;
        uint64_t at[WR_TILES];
        uint32_t from[WR_TILES];  // the first row that sees the lane's position
        float sum[WR_TILES], part[WR_TILES];  // long sums in two steps, which lose less
#pragma unroll
        for (uint32_t i = 0; i < WR_TILES; ++i) {
            const uint32_t p = p0 + i * 16 + c16;
            sum[i] = part[i] = 0.0f;
            at[i] = 0;
            from[i] = 0xFFFFFFFFu;
            if (p < t.keys) {
                const uint32_t page = static_cast<uint32_t>(a.table[r * a.table_stride + (p >> a.page_lg)]);
                const uint32_t off = p & ((1u << a.page_lg) - 1u), slot = (page << a.page_lg) + off;
                bool see = page < a.n_pages;
                if (see && a.gated)
                    see = slot < a.visible.end && ((a.visible.word(slot >> 5) >> (slot & 31u)) & 1u);
                const int64_t token = a.causal ? max(static_cast<int64_t>(0), static_cast<int64_t>(p) - t.older) : 0;
                if (see && token < t.tokens) {
                    at[i] = page * a.k_page + off * a.k_slot;
                    from[i] = static_cast<uint32_t>(token) * group;
                }
            }
        }
        for (uint32_t h = head_wave; h < a.kv_heads; h += a.head_waves) {
            v8s key[WR_TILES][STEPS];
#pragma unroll
            for (uint32_t i = 0; i < WR_TILES; ++i)
#pragma unroll
                for (uint32_t s = 0; s < STEPS; ++s) {
                    const uint32_t d = s * 32 + g * 8;
                    key[i][s] = v8s{};
                    if (from[i] != 0xFFFFFFFFu && d < a.dim)
                        key[i][s] = __builtin_nontemporal_load(
                            reinterpret_cast<const v8s*>(a.k + at[i] + h * a.k_head + d));
                }
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
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    const uint32_t row = min(row0 + g * 4 + e, rows - 1);
                    const float z = a.lse[static_cast<uint64_t>(t.token0 + row / group) * a.heads + h * group + row % group];
                    lse2[e] = z == -__builtin_inff() ? __builtin_inff() : z * LOG2E;
                }
#pragma unroll
                for (uint32_t i = 0; i < WR_TILES; ++i) {
                    f32x4 x = {0, 0, 0, 0};
#pragma unroll
                    for (uint32_t s = 0; s < STEPS; ++s) x = E::mfma16(q[s], key[i][s], x);
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        const uint32_t row = row0 + g * 4 + e;
                        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], a.scale2, -lse2[e]));
                        part[i] += row >= from[i] && row < rows ? w : 0.0f;
                    }
                }
                if (row0 % 1024 == 1008 || row0 + 16 >= rows) {
#pragma unroll
                    for (uint32_t i = 0; i < WR_TILES; ++i) {
                        sum[i] += part[i];
                        part[i] = 0.0f;
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < WR_TILES; ++i) {
            sum[i] += __shfl_xor(sum[i], 16, 64);
            sum[i] += __shfl_xor(sum[i], 32, 64);
            if (g == 0) s_sum[wave][i * 16 + c16] = sum[i];
        }
        __syncthreads();
        // the heads' sums joined in a fixed order
        const uint32_t in = threadIdx.x % (WR_TILES * 16), of = threadIdx.x / (WR_TILES * 16);
        const uint32_t p = first + of * WR_TILES * 16 + in;
        if (of < tile_waves && p < t.keys) {
            float all = 0.0f;
            for (uint32_t w = 0; w < a.head_waves; ++w) all += s_sum[of * a.head_waves + w][in];
            const float past =
                a.past && (a.continued || static_cast<int64_t>(p) < t.older) ? a.past[r * a.past_stride + p] * a.decay : 0.0f;
            a.out[r * a.out_stride + p] = past + all;
        }
        __syncthreads();
    }
}

template <class E>
void launch_weights(const WeightArgs& a, uint32_t grid, hipStream_t s)
{
    if (a.dim <= 64)
        wt_rows<E, 64><<<grid, WR_NT, 0, s>>>(a);
    else if (a.dim <= 96)
        wt_rows<E, 96><<<grid, WR_NT, 0, s>>>(a);
    else if (a.dim <= 128)
        wt_rows<E, 128><<<grid, WR_NT, 0, s>>>(a);
    else if (a.dim <= 192)
        wt_rows<E, 192><<<grid, WR_NT, 0, s>>>(a);
    else
        wt_rows<E, 256><<<grid, WR_NT, 0, s>>>(a);
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
    if (n_slots >> 31 || room >> 31 || p.n_tokens >> 31 || p.n_heads > 65535 || p.n_requests >> 24 ||
        (static_cast<uint64_t>(p.n_tokens) * p.n_heads) >> 31) {
        set_error("cr_paged_weights: supported up to 2^31 - 1 slots, positions and rows, 65535 heads and 2^24 - 1 "
                  "requests");
        return CR_ERR_UNSUPPORTED;
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
    const uint64_t most = p.max_kv ? std::min<uint64_t>(room, p.max_kv) : room;
    a.head_waves = a.kv_heads >= 3 ? 4 : a.kv_heads;
    const uint32_t span = WR_WAVES / a.head_waves * WR_TILES * 16;
    a.spans = static_cast<uint32_t>((most + span - 1) / span);
    if (a.spans == 0) return CR_OK;
    const uint64_t grid = static_cast<uint64_t>(a.spans) * a.n_requests;
    if (grid >> 23) {  // a launch holds fewer than 2^32 threads
        set_error("cr_paged_weights: too many positions for one call");
        return CR_ERR_UNSUPPORTED;
    }
    hipStream_t s = as_stream(stream);
    const bool direct = p.visible && is_direct(p.visible);
    const uint32_t n_words = static_cast<uint32_t>((n_slots + 31) / 32);
    Scratch sc;
    if (p.visible && !direct) CR_RET(sc.alloc(std::max<size_t>(256, n_words * 4ull), s));
    if (p.visible)
        CR_RET(set_bits(p.visible, direct, sc.at<uint32_t>(0), n_words, static_cast<uint32_t>(n_slots), stream,
                        &a.visible));
    CR_TIMED("wt_rows", s);
    if (cache->dtype == CR_F16)
        launch_weights<Half>(a, static_cast<uint32_t>(grid), s);
    else
        launch_weights<BHalf>(a, static_cast<uint32_t>(grid), s);
    CR_LAUNCH_CHECK();
    return CR_OK;
}

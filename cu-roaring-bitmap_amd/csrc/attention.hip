// Attention of new tokens over a paged key/value cache (no reference
// implementation).
//
// For token t and head h, over the keys j that the token sees:
//   s_j = scale * q_t . k_j,  o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),
//   lse = m + log(sum_j e^(s_j - m)),  m = max_j s_j.
#include <algorithm>

#include "internal.hpp"

namespace crimpl {

namespace {

constexpr uint32_t AT_DIM_MAX = 256;

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
};

struct Half {
    static __device__ __forceinline__ float up(uint16_t x) { return static_cast<float>(__builtin_bit_cast(_Float16, x)); }
    static __device__ __forceinline__ uint16_t down(float x) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x)); }
};
struct BHalf {
    static __device__ __forceinline__ float up(uint16_t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }
    static __device__ __forceinline__ uint16_t down(float x) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x)); }
};

constexpr int AT_NT = 256;

// A workgroup per (token, head), a tile of AT_NT keys at a time.
template <class E>
__global__ __launch_bounds__(AT_NT) void at_simple(AttnArgs a)
{
    __shared__ float s_q[AT_DIM_MAX], s_p[AT_NT], s_red[AT_NT / 64];
    __shared__ int32_t s_slot[AT_NT];
    const uint32_t t = threadIdx.x, token = blockIdx.x, h = blockIdx.y, kh = h / (a.heads / a.kv_heads);
    uint32_t lo = 0, hi = a.n_requests;
    int64_t limit = 0;
    if (a.n_requests && a.starts[0] <= static_cast<int32_t>(token) && static_cast<int32_t>(token) < a.starts[a.n_requests]) {
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (a.starts[mid] <= static_cast<int32_t>(token)) lo = mid;
            else hi = mid;
        }
        const int64_t room = static_cast<int64_t>(a.cols) << a.page_lg;
        const int64_t len = min(room, static_cast<int64_t>(max(a.sel ? a.sel_len[lo] : a.kv_len[lo], 0)));
        limit = len;
        if (a.causal) {
            const int64_t at = a.sel ? a.limits[token] : static_cast<int64_t>(a.kv_len[lo]) - a.starts[lo + 1] + token + 1;
            limit = max(static_cast<int64_t>(0), min(len, at));
        }
    }
    for (uint32_t d = t; d < a.dim; d += AT_NT) s_q[d] = E::up(a.q[token * a.q_token + h * a.q_head + d]) * a.scale;
    float m = -__builtin_inff(), l = 0, o = 0;
    for (int64_t j0 = 0; j0 < limit; j0 += AT_NT) {
        __syncthreads();
        const int64_t j = j0 + t;
        float s = -__builtin_inff();
        int32_t slot = -1;
        if (j < limit) {
            if (a.sel) slot = a.sel[lo * a.sel_stride + j];
            else {
                const int32_t page = a.table[lo * a.table_stride + (j >> a.page_lg)];
                if (static_cast<uint32_t>(page) < a.n_pages) slot = (page << a.page_lg) + static_cast<int32_t>(j & ((1 << a.page_lg) - 1));
            }
            if (static_cast<uint64_t>(static_cast<uint32_t>(slot)) >> a.page_lg >= a.n_pages) slot = -1;
        }
        s_slot[t] = slot;
        if (slot >= 0) {
            const uint16_t* k = a.k + (slot >> a.page_lg) * a.k_page + (slot & ((1 << a.page_lg) - 1)) * a.k_slot + kh * a.k_head;
            s = 0;
            for (uint32_t d = 0; d < a.dim; ++d) s += s_q[d] * E::up(k[d]);
        }
        float top = s;
        for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
        if ((t & 63) == 0) s_red[t >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
        const float now = fmaxf(m, top);
        if (now == -__builtin_inff()) continue;
        const float fix = __expf(m - now);
        m = now;
        s_p[t] = __expf(s - now);
        __syncthreads();
        o *= fix;
        l *= fix;
        for (uint32_t i = 0; i < AT_NT; ++i) {
            if (s_slot[i] < 0) continue;
            l += s_p[i];
            if (t < a.dim)
                o += s_p[i] * E::up(a.v[(s_slot[i] >> a.page_lg) * a.v_page + (s_slot[i] & ((1 << a.page_lg) - 1)) * a.v_slot + kh * a.v_head + t]);
        }
    }
    if (t < a.dim) a.out[token * a.out_token + h * a.out_head + t] = E::down(l > 0 ? o / l : 0.0f);
    if (a.lse && t == 0) a.lse[static_cast<uint64_t>(token) * a.heads + h] = l > 0 ? m + __logf(l) : -__builtin_inff();
}

}  // namespace

}  // namespace crimpl

using namespace crimpl;

extern "C" int cr_paged_attention(const cr_paged_attention_args* args, const cr_paged_cache* cache, cr_stream_t stream)
{
    if (!args || !cache) {
        set_error("cr_paged_attention: invalid argument");
        return CR_ERR_INVALID;
    }
    const cr_paged_attention_args& p = *args;
    if (p.n_tokens == 0 || p.n_heads == 0) return CR_OK;
    const bool pow2 = cache->page_size && (cache->page_size & (cache->page_size - 1)) == 0;
    if (!p.q || !p.out || !p.d_starts || (p.n_requests && !p.d_kv_len) || !pow2 || cache->n_heads == 0 ||
        p.n_heads % cache->n_heads || cache->head_dim == 0 || (cache->n_pages && (!cache->k || !cache->v)) ||
        (p.table_cols && p.n_requests && !p.d_table) || p.table_stride < p.table_cols ||
        (p.d_sel && (!p.d_sel_len || !p.d_limits ||
                     p.sel_stride < static_cast<uint64_t>(p.table_cols) * cache->page_size))) {
        set_error("cr_paged_attention: invalid argument (%u query heads, %u key heads, page size %u)", p.n_heads,
                  cache->n_heads, cache->page_size);
        return CR_ERR_INVALID;
    }
    const uint64_t strides = p.q_token_stride | p.q_head_stride | p.out_token_stride | p.out_head_stride |
                             cache->k_page_stride | cache->k_slot_stride | cache->k_head_stride |
                             cache->v_page_stride | cache->v_slot_stride | cache->v_head_stride | cache->head_dim;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out) |
                         reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v);
    if ((cache->dtype != CR_F16 && cache->dtype != CR_BF16) || cache->head_dim > AT_DIM_MAX || strides % 8 || at % 16) {
        set_error("cr_paged_attention: f16 or bf16 rows of at most %u dimensions (a multiple of 8), 16-byte aligned, "
                  "are supported (type %u, %u dimensions)", AT_DIM_MAX, cache->dtype, cache->head_dim);
        return CR_ERR_UNSUPPORTED;
    }
    const uint64_t n_slots = static_cast<uint64_t>(cache->n_pages) * cache->page_size;
    const uint64_t room = static_cast<uint64_t>(p.table_cols) * cache->page_size;
    if (n_slots >> 31 || room >> 31 || p.n_tokens >> 31 || p.n_heads > 65535 || p.n_requests >> 24) {
        set_error("cr_paged_attention: supported up to 2^31 - 1 slots, positions and tokens, 65535 heads and 2^24 - 1 "
                  "requests");
        return CR_ERR_UNSUPPORTED;
    }
    AttnArgs a{};
    a.q = static_cast<const uint16_t*>(p.q);
    a.q_token = p.q_token_stride;
    a.q_head = p.q_head_stride;
    a.out = static_cast<uint16_t*>(p.out);
    a.out_token = p.out_token_stride;
    a.out_head = p.out_head_stride;
    a.lse = p.lse;
    a.n_tokens = p.n_tokens;
    a.heads = p.n_heads;
    a.kv_heads = cache->n_heads;
    a.dim = cache->head_dim;
    a.n_requests = p.n_requests;
    a.k = static_cast<const uint16_t*>(cache->k);
    a.v = static_cast<const uint16_t*>(cache->v);
    a.k_page = cache->k_page_stride;
    a.k_slot = cache->k_slot_stride;
    a.k_head = cache->k_head_stride;
    a.v_page = cache->v_page_stride;
    a.v_slot = cache->v_slot_stride;
    a.v_head = cache->v_head_stride;
    a.n_pages = cache->n_pages;
    a.page_lg = static_cast<uint32_t>(__builtin_ctz(cache->page_size));
    a.starts = p.d_starts;
    a.kv_len = p.d_kv_len;
    a.table = p.d_table;
    a.cols = p.table_cols;
    a.table_stride = p.table_stride;
    a.sel = p.d_sel;
    a.sel_stride = p.sel_stride;
    a.sel_len = p.d_sel_len;
    a.limits = p.d_limits;
    a.scale = p.scale;
    a.causal = p.causal;
    hipStream_t s = as_stream(stream);
    CR_TIMED("at_simple", s);
    if (cache->dtype == CR_F16)
        at_simple<Half><<<dim3(p.n_tokens, p.n_heads), AT_NT, 0, s>>>(a);
    else
        at_simple<BHalf><<<dim3(p.n_tokens, p.n_heads), AT_NT, 0, s>>>(a);
    CR_LAUNCH_CHECK();
    return CR_OK;
}

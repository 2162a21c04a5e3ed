// A paged key/value cache's bookkeeping, for serving language models (no
// reference implementation).
//
//   cr_paged_plan    block tables and slot maps from the requests' lengths, the
//                    pages taken from a Roaring bitmap of free ones
//   cr_paged_append  new keys and values into their slots
//   cr_paged_select  the slots of each request that a Roaring bitmap lets through
//
// Lengths, tables and slots stay on the device: no call waits for the stream.
// Whatever those arrays hold, accesses stay inside the buffers that the host
// arguments describe.
#include <algorithm>

#include "internal.hpp"

namespace crimpl {

namespace {

constexpr int PG_NT = 1024;             // the plan's workgroup
constexpr uint32_t PG_BLOCK = 2048;     // pages a block of the free set holds: 64 words
constexpr int PG_TAKE_NT = 256;
constexpr uint32_t PG_TOKENS = 2048;    // tokens a workgroup of the slot map writes
constexpr int PG_FILL_NT = 256;

__device__ __forceinline__ uint64_t wave_incl_scan_u64(uint64_t v)
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t x = __shfl_up(v, o, 64);
        if (static_cast<int>(__lane_id()) >= o) v += x;
    }
    return v;
}

// Block-wide exclusive scan in 64 bits (lengths are the caller's: their sums
// need not fit 32); `lds` holds one slot per wave.
template <int NT>
__device__ __forceinline__ uint64_t block_excl_scan_u64(uint64_t v, uint64_t* lds, uint64_t& total)
{
    const uint64_t incl = wave_incl_scan_u64(v);
    const uint32_t w = threadIdx.x >> 6;
    if (__lane_id() == 63) lds[w] = incl;
    __syncthreads();
    uint64_t base = 0, t = 0;
#pragma unroll
    for (uint32_t i = 0; i < NT / 64; ++i) {
        const uint64_t x = lds[i];
        base += i < w ? x : 0ull;
        t += x;
    }
    __syncthreads();
    total = t;
    return base + incl - v;
}

struct PlanArgs {
    const uint32_t* words;  // the free set's bits, (n_pages + 31) / 32 words
    uint32_t n_pages;
    uint32_t n_blocks;
    uint32_t page_lg;
    const int32_t* cached;
    const int32_t* fresh;
    uint32_t n_requests;
    int32_t* table;
    uint32_t cols;
    uint64_t table_stride;
    int64_t* slots;
    uint32_t slots_cap;
    int32_t* starts;
    int32_t* kv_len;
    int32_t* taken;
    uint32_t taken_cap;
    int32_t* counts;
    uint32_t* upto;       // [n_requests + 1] pages that the requests before take, in order
    uint32_t* block_pre;  // [n_blocks] free pages before each block
    uint32_t* n_taken;
};

// Word w of the free set, without the bits past the last page.
__device__ __forceinline__ uint32_t free_word(const PlanArgs& a, uint32_t w)
{
    uint32_t x = a.words[w];
    if (w == a.n_pages / 32u) x &= (1u << (a.n_pages % 32u)) - 1u;
    return x;
}

struct Request {
    uint64_t tokens, held, most;
    bool fits;  // lengths are not negative and the row holds the pages
};

__device__ __forceinline__ Request request_of(const PlanArgs& a, uint32_t r)
{
    const int32_t c = a.cached[r], n = a.fresh[r];
    const uint64_t page = 1ull << a.page_lg;
    Request q;
    q.tokens = n > 0 ? static_cast<uint64_t>(n) : 0ull;
    const uint64_t before = c > 0 ? static_cast<uint64_t>(c) : 0ull;
    q.held = (before + page - 1) >> a.page_lg;
    q.most = (before + q.tokens + page - 1) >> a.page_lg;
    q.fits = c >= 0 && n >= 0 && q.most <= a.cols && before + q.tokens <= 0x7FFFFFFFull;
    return q;
}

// The last entry of a[0, n) that is at most v (a[0] <= v, ascending).
template <class T>
__device__ __forceinline__ uint32_t last_at_most(const T* a, uint32_t lo, uint32_t hi, T v)
{
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (a[mid] <= v)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// One workgroup: the free pages before each block, then the requests' token
// offsets, the pages that they take and which of them get theirs.
__global__ __launch_bounds__(PG_NT) void pg_scan(PlanArgs a)
{
    __shared__ uint64_t s_scan[PG_NT / 64];
    __shared__ uint64_t s_taken, s_missing;
    const uint32_t t = threadIdx.x;
    if (t == 0) s_taken = s_missing = 0;
    uint64_t n_free = 0;
    for (uint32_t b0 = 0; b0 < a.n_blocks; b0 += PG_NT) {
        const uint32_t b = b0 + t;
        uint32_t n = 0;
        if (b < a.n_blocks) {
            const uint32_t last = (a.n_pages + 31u) / 32u;
            for (uint32_t w = b * (PG_BLOCK / 32u); w < min(last, (b + 1) * (PG_BLOCK / 32u)); ++w)
                n += __popc(free_word(a, w));
        }
        uint64_t all;
        const uint64_t pre = block_excl_scan_u64<PG_NT>(n, s_scan, all);
        if (b < a.n_blocks) a.block_pre[b] = static_cast<uint32_t>(n_free + pre);
        n_free += all;
    }
    uint64_t tokens = 0, pages = 0;
    for (uint32_t r0 = 0; r0 < a.n_requests; r0 += PG_NT) {
        const uint32_t r = r0 + t;
        Request q{0, 0, 0, false};
        if (r < a.n_requests) q = request_of(a, r);
        const uint64_t need = q.fits ? q.most - q.held : 0ull;
        uint64_t all_tokens, all_pages;
        const uint64_t at = tokens + block_excl_scan_u64<PG_NT>(q.tokens, s_scan, all_tokens);
        const uint64_t before = pages + block_excl_scan_u64<PG_NT>(need, s_scan, all_pages);
        if (r < a.n_requests) {
            const bool granted = q.fits && (need == 0 || before + need <= n_free);
            a.starts[r] = static_cast<int32_t>(min(at, static_cast<uint64_t>(0x7FFFFFFF)));
            a.kv_len[r] = granted ? a.cached[r] + a.fresh[r] : 0;
            a.upto[r] = static_cast<uint32_t>(min(before, static_cast<uint64_t>(0xFFFFFFFF)));
            if (granted && need) atomicMax(reinterpret_cast<unsigned long long*>(&s_taken),
                                           static_cast<unsigned long long>(before + need));
            if (!granted && q.most > q.held) atomicAdd(reinterpret_cast<unsigned long long*>(&s_missing),
                                                       static_cast<unsigned long long>(q.most - q.held));
        }
        tokens += all_tokens;
        pages += all_pages;
    }
    __syncthreads();
    if (t == 0) {
        const uint64_t most = 0x7FFFFFFF;
        a.starts[a.n_requests] = static_cast<int32_t>(min(tokens, most));
        a.upto[a.n_requests] = static_cast<uint32_t>(min(pages, static_cast<uint64_t>(0xFFFFFFFF)));
        *a.n_taken = static_cast<uint32_t>(s_taken);
        a.counts[0] = static_cast<int32_t>(min(tokens, most));
        a.counts[1] = static_cast<int32_t>(min(s_taken, most));
        a.counts[2] = static_cast<int32_t>(min(s_missing, most));
    }
}

// A workgroup per block of the free set: its pages that are taken, into the
// list of them and into the tables of the requests that take them.
__global__ __launch_bounds__(PG_TAKE_NT) void pg_take(PlanArgs a)
{
    constexpr uint32_t PER = PG_BLOCK / PG_TAKE_NT;  // pages a thread looks at
    __shared__ uint32_t s_scan[PG_TAKE_NT / 64];
    __shared__ uint16_t s_id[PG_BLOCK];
    const uint32_t n_taken = *a.n_taken, base = a.block_pre[blockIdx.x], t = threadIdx.x;
    if (base >= n_taken) return;
    const uint32_t first = blockIdx.x * PG_BLOCK + t * PER;
    uint32_t bits = 0;
    if (first < a.n_pages) bits = (free_word(a, first / 32u) >> (first % 32u)) & ((1u << PER) - 1u);
    uint32_t total;
    uint32_t at = block_excl_scan<PG_TAKE_NT>(__popc(bits), s_scan, total);
    for (; bits; bits &= bits - 1u) s_id[at++] = static_cast<uint16_t>(t * PER + __ffs(bits) - 1);
    __syncthreads();
    const uint32_t n = min(total, n_taken - base);
    const uint32_t lo = last_at_most(a.upto, 0u, a.n_requests, base);
    const uint32_t hi = n ? last_at_most(a.upto, lo, a.n_requests, base + n - 1) + 1 : lo + 1;
    for (uint32_t i = t; i < n; i += PG_TAKE_NT) {
        const uint32_t rank = base + i, id = blockIdx.x * PG_BLOCK + s_id[i];
        if (rank < a.taken_cap) a.taken[rank] = static_cast<int32_t>(id);
        const uint32_t r = last_at_most(a.upto, lo, hi, rank);
        const uint64_t col = request_of(a, r).held + (rank - a.upto[r]);
        if (col < a.cols) a.table[r * a.table_stride + col] = static_cast<int32_t>(id);
    }
}

// The slot of each new token, from the tables as pg_take left them.
__global__ __launch_bounds__(PG_FILL_NT) void pg_slots(PlanArgs a)
{
    const uint32_t total = min(a.slots_cap, static_cast<uint32_t>(a.starts[a.n_requests]));
    const uint32_t first = blockIdx.x * PG_TOKENS;
    if (first >= total) return;
    const uint32_t n = min(PG_TOKENS, total - first);
    const uint32_t lo = last_at_most(a.starts, 0u, a.n_requests, static_cast<int32_t>(first));
    const uint32_t hi = last_at_most(a.starts, lo, a.n_requests, static_cast<int32_t>(first + n - 1)) + 1;
    for (uint32_t i = threadIdx.x; i < n; i += PG_FILL_NT) {
        const uint32_t token = first + i;
        const uint32_t r = last_at_most(a.starts, lo, hi, static_cast<int32_t>(token));
        int64_t slot = -1;
        if (a.kv_len[r] > 0) {
            const uint32_t pos = static_cast<uint32_t>(a.cached[r]) + (token - static_cast<uint32_t>(a.starts[r]));
            const uint32_t col = pos >> a.page_lg;
            if (col < a.cols)
                slot = (static_cast<int64_t>(a.table[r * a.table_stride + col]) << a.page_lg) +
                       (pos & ((1u << a.page_lg) - 1u));
        }
        a.slots[token] = slot;
    }
}

// ---- append --------------------------------------------------------------------
struct AppendArgs {
    const char* src[2];
    char* dst[2];
    uint64_t src_token[2], src_head[2];            // strides in bytes
    uint64_t dst_page[2], dst_slot[2], dst_head[2];
    const int64_t* slots;
    uint32_t n_tokens, heads, units;  // units: pieces of sizeof(U) bytes in a head's row
    uint64_t n_slots;
    uint32_t page_lg;
};

constexpr int AP_NT = 256;
constexpr uint32_t AP_PER = 4;

// Each thread moves AP_PER pieces of keys and of values, all loads before the stores.
template <class U>
__global__ __launch_bounds__(AP_NT) void pg_append(AppendArgs a)
{
    const uint32_t row = a.heads * a.units;
    const uint64_t all = static_cast<uint64_t>(a.n_tokens) * row;
    U x[2][AP_PER];
    uint64_t to[2][AP_PER];
    bool on[AP_PER];
#pragma unroll
    for (uint32_t j = 0; j < AP_PER; ++j) {
        const uint64_t i = (static_cast<uint64_t>(blockIdx.x) * AP_PER + j) * AP_NT + threadIdx.x;
        on[j] = i < all;
        if (!on[j]) continue;
        const uint32_t token = static_cast<uint32_t>(i / row), in = static_cast<uint32_t>(i % row);
        const uint32_t head = in / a.units, unit = in % a.units;
        const int64_t slot = a.slots[token];
        on[j] = slot >= 0 && static_cast<uint64_t>(slot) < a.n_slots;
        if (!on[j]) continue;
        const uint64_t page = static_cast<uint64_t>(slot) >> a.page_lg, off = slot & ((1u << a.page_lg) - 1u);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            x[c][j] = *reinterpret_cast<const U*>(a.src[c] + token * a.src_token[c] + head * a.src_head[c] +
                                                  unit * sizeof(U));
            to[c][j] = page * a.dst_page[c] + off * a.dst_slot[c] + head * a.dst_head[c] + unit * sizeof(U);
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < AP_PER; ++j) {
        if (!on[j]) continue;
#pragma unroll
        for (int c = 0; c < 2; ++c) *reinterpret_cast<U*>(a.dst[c] + to[c][j]) = x[c][j];
    }
}

// ---- select --------------------------------------------------------------------
constexpr int SL_NT = 256;
constexpr uint32_t SL_POS = 32 * SL_NT;  // positions a workgroup looks at

struct SelectArgs {
    const uint32_t* words;  // visible slots, n_words of them
    uint32_t n_words;
    const int32_t* table;
    uint32_t cols;
    uint64_t table_stride;
    const int32_t* starts;
    const int32_t* kv_len;
    uint32_t n_requests;
    uint32_t page_lg;
    uint32_t n_pages;
    uint32_t n_tokens;
    int32_t* sel;
    uint64_t sel_stride;
    int32_t* sel_len;
    int32_t* limits;
    uint32_t chunks;
    uint32_t* counts;  // [n_requests][chunks] visible positions, where there is more than one chunk
};

__device__ __forceinline__ uint32_t select_len(const SelectArgs& a, uint32_t r)
{
    const int32_t n = a.kv_len[r];
    const uint64_t most = static_cast<uint64_t>(a.cols) << a.page_lg;
    return n <= 0 ? 0u : static_cast<uint32_t>(min(most, static_cast<uint64_t>(n)));
}

// Which of the 32 positions from p0 (a multiple of 32) are visible.
__device__ __forceinline__ uint32_t visible_word(const SelectArgs& a, uint32_t r, uint32_t p0, uint32_t len)
{
    if (p0 >= len) return 0u;
    const int32_t* row = a.table + r * a.table_stride;
    const uint32_t lg = min(a.page_lg, 5u), part = 1u << lg;
    uint32_t vis = 0;
    for (uint32_t k = 0; k < 32u && p0 + k < len; k += part) {
        const uint32_t pos = p0 + k, page = static_cast<uint32_t>(row[pos >> a.page_lg]);
        if (page >= a.n_pages) continue;
        const uint64_t slot = (static_cast<uint64_t>(page) << a.page_lg) + (pos & ((1u << a.page_lg) - 1u));
        uint32_t bits = a.words[slot >> 5] >> (slot & 31u);
        if (lg < 5u) bits &= (1u << part) - 1u;
        vis |= bits << k;
    }
    return len - p0 < 32u ? vis & ((1u << (len - p0)) - 1u) : vis;
}

__global__ __launch_bounds__(SL_NT) void sl_count(SelectArgs a)
{
    __shared__ uint32_t s[SL_NT / 64];
    const uint32_t r = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const uint32_t vis = visible_word(a, r, chunk * SL_POS + threadIdx.x * 32u, select_len(a, r));
    const uint32_t n = block_sum<SL_NT>(__popc(vis), s);
    if (threadIdx.x == 0) a.counts[blockIdx.x] = n;
}

__global__ __launch_bounds__(SL_NT) void sl_write(SelectArgs a)
{
    __shared__ uint32_t s[SL_NT / 64];
    __shared__ int32_t s_slot[SL_POS];
    const uint32_t r = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, t = threadIdx.x;
    const uint32_t len = select_len(a, r), p0 = chunk * SL_POS + t * 32u;
    // positions of the new tokens: the last `fresh` of the request's
    const int32_t t0 = min(max(a.starts[r], 0), static_cast<int32_t>(a.n_tokens));
    const int32_t t1 = min(max(a.starts[r + 1], t0), static_cast<int32_t>(a.n_tokens));
    const int64_t shift = static_cast<int64_t>(t1) - len;  // position p is new token p + shift
    if (chunk == 0) {  // tokens before the first position see nothing
        for (int64_t i = t0 + t; i < min(static_cast<int64_t>(t1), shift); i += SL_NT) a.limits[i] = 0;
    }
    if (chunk * SL_POS >= len && chunk > 0) return;
    uint32_t base = 0;
    for (uint32_t i = t; i < chunk; i += SL_NT) base += a.counts[r * a.chunks + i];
    if (a.chunks > 1) base = block_sum<SL_NT>(base, s);
    const uint32_t vis = visible_word(a, r, p0, len);
    uint32_t total;
    const uint32_t before = block_excl_scan<SL_NT>(__popc(vis), s, total);
    const int32_t* row = a.table + r * a.table_stride;
    uint32_t at = before;
    for (uint32_t b = vis; b; b &= b - 1u) {
        const uint32_t pos = p0 + __ffs(b) - 1;
        s_slot[at++] = (row[pos >> a.page_lg] << a.page_lg) + static_cast<int32_t>(pos & ((1u << a.page_lg) - 1u));
    }
    for (uint32_t k = 0; k < 32u && p0 + k < len; ++k) {
        const int64_t token = static_cast<int64_t>(p0 + k) + shift;
        if (token >= t0 && token < t1)
            a.limits[token] = static_cast<int32_t>(base + before + __popc(vis & (0xFFFFFFFFu >> (31u - k))));
    }
    __syncthreads();
    for (uint32_t i = t; i < total; i += SL_NT) a.sel[r * a.sel_stride + base + i] = s_slot[i];
    if (t == 0 && (len <= SL_POS || chunk == (len - 1) / SL_POS)) a.sel_len[r] = static_cast<int32_t>(base + total);
}

bool power_of_two(uint32_t x) { return x && (x & (x - 1)) == 0; }

}  // namespace

}  // namespace crimpl

using namespace crimpl;

extern "C" int cr_paged_plan(const cr_gpu_roaring* free_pages, uint32_t n_pages, uint32_t page_size,
                             const int32_t* d_cached, const int32_t* d_new, uint32_t n_requests, int32_t* d_table,
                             uint32_t table_cols, uint64_t table_stride, int64_t* d_slots, uint32_t slots_cap,
                             int32_t* d_starts, int32_t* d_kv_len, int32_t* d_taken, uint32_t taken_cap,
                             int32_t* d_counts, cr_stream_t stream)
{
    if (!free_pages || !d_starts || !d_counts || !power_of_two(page_size) ||
        (n_requests && (!d_cached || !d_new || !d_kv_len)) || (n_requests && table_cols && !d_table) ||
        table_stride < table_cols || (slots_cap && !d_slots) || (taken_cap && !d_taken)) {
        set_error("cr_paged_plan: invalid argument (page size %u)", page_size);
        return CR_ERR_INVALID;
    }
    if ((static_cast<uint64_t>(n_pages) * page_size) >> 31 || slots_cap >> 31 || n_requests >> 24) {
        set_error("cr_paged_plan: supported up to 2^31 - 1 slots and tokens and 2^24 - 1 requests");
        return CR_ERR_UNSUPPORTED;
    }
    hipStream_t s = as_stream(stream);
    PlanArgs a{};
    const uint32_t n_words = (n_pages + 31u) / 32u;
    a.n_pages = n_pages;
    a.n_blocks = (n_pages + PG_BLOCK - 1) / PG_BLOCK;
    a.page_lg = static_cast<uint32_t>(__builtin_ctz(page_size));
    a.cached = d_cached;
    a.fresh = d_new;
    a.n_requests = n_requests;
    a.table = d_table;
    a.cols = table_cols;
    a.table_stride = table_stride;
    a.slots = d_slots;
    a.slots_cap = slots_cap;
    a.starts = d_starts;
    a.kv_len = d_kv_len;
    a.taken = d_taken;
    a.taken_cap = taken_cap;
    a.counts = d_counts;
    Carver cv;
    const size_t o_words = cv.add(n_words * 4ull), o_upto = cv.add((n_requests + 1ull) * 4);
    const size_t o_pre = cv.add(a.n_blocks * 4ull), o_taken = cv.add(4);
    Scratch sc;
    CR_RET(sc.alloc(cv.total, s));
    a.words = sc.at<uint32_t>(o_words);
    a.upto = sc.at<uint32_t>(o_upto);
    a.block_pre = sc.at<uint32_t>(o_pre);
    a.n_taken = sc.at<uint32_t>(o_taken);
    CR_RET(cr_decompress_to_bitset(free_pages, sc.at<uint32_t>(o_words), n_words, stream));
    CR_TIMED("pg_plan", s);
    pg_scan<<<1, PG_NT, 0, s>>>(a);
    if (a.n_blocks && n_requests) pg_take<<<a.n_blocks, PG_TAKE_NT, 0, s>>>(a);
    if (slots_cap && n_requests) pg_slots<<<(slots_cap + PG_TOKENS - 1) / PG_TOKENS, PG_FILL_NT, 0, s>>>(a);
    CR_LAUNCH_CHECK();
    return CR_OK;
}

extern "C" int cr_paged_append(const void* d_k, const void* d_v, uint64_t k_token_stride, uint64_t k_head_stride,
                               uint64_t v_token_stride, uint64_t v_head_stride, uint32_t n_tokens,
                               const int64_t* d_slots, const cr_paged_cache* cache, cr_stream_t stream)
{
    if (!cache || !cache->k || !cache->v || !power_of_two(cache->page_size) || cache->dtype > CR_BF16 ||
        (n_tokens && (!d_k || !d_v || !d_slots))) {
        set_error("cr_paged_append: invalid argument");
        return CR_ERR_INVALID;
    }
    const uint64_t es = cache->dtype == CR_F32 ? 4 : 2;
    AppendArgs a{};
    a.src[0] = static_cast<const char*>(d_k);
    a.src[1] = static_cast<const char*>(d_v);
    a.dst[0] = static_cast<char*>(cache->k);
    a.dst[1] = static_cast<char*>(cache->v);
    a.src_token[0] = k_token_stride * es;
    a.src_token[1] = v_token_stride * es;
    a.src_head[0] = k_head_stride * es;
    a.src_head[1] = v_head_stride * es;
    a.dst_page[0] = cache->k_page_stride * es;
    a.dst_page[1] = cache->v_page_stride * es;
    a.dst_slot[0] = cache->k_slot_stride * es;
    a.dst_slot[1] = cache->v_slot_stride * es;
    a.dst_head[0] = cache->k_head_stride * es;
    a.dst_head[1] = cache->v_head_stride * es;
    a.slots = d_slots;
    a.n_tokens = n_tokens;
    a.heads = cache->n_heads;
    a.n_slots = static_cast<uint64_t>(cache->n_pages) * cache->page_size;
    a.page_lg = static_cast<uint32_t>(__builtin_ctz(cache->page_size));
    uint64_t all = cache->head_dim * es;
    for (int c = 0; c < 2; ++c)
        all |= reinterpret_cast<uintptr_t>(a.src[c]) | reinterpret_cast<uintptr_t>(a.dst[c]) | a.src_token[c] |
               a.src_head[c] | a.dst_page[c] | a.dst_slot[c] | a.dst_head[c];
    const uint32_t unit = all % 16 == 0 ? 16 : static_cast<uint32_t>(es);
    a.units = static_cast<uint32_t>(cache->head_dim * es / unit);
    const uint64_t pieces = static_cast<uint64_t>(n_tokens) * a.heads * a.units;
    if (pieces == 0) return CR_OK;
    const uint64_t grid = (pieces + AP_NT * AP_PER - 1) / (AP_NT * AP_PER);
    if (grid >> 31) {
        set_error("cr_paged_append: too many elements for one call");
        return CR_ERR_UNSUPPORTED;
    }
    hipStream_t s = as_stream(stream);
    CR_TIMED("pg_append", s);
    if (unit == 16)
        pg_append<uint4><<<static_cast<unsigned>(grid), AP_NT, 0, s>>>(a);
    else if (es == 4)
        pg_append<uint32_t><<<static_cast<unsigned>(grid), AP_NT, 0, s>>>(a);
    else
        pg_append<uint16_t><<<static_cast<unsigned>(grid), AP_NT, 0, s>>>(a);
    CR_LAUNCH_CHECK();
    return CR_OK;
}

extern "C" int cr_paged_select(const cr_gpu_roaring* visible, uint32_t n_pages, uint32_t page_size,
                               const int32_t* d_table, uint32_t table_cols, uint64_t table_stride,
                               const int32_t* d_starts, const int32_t* d_kv_len, uint32_t n_requests,
                               uint32_t n_tokens, int32_t* d_sel, uint64_t sel_stride, int32_t* d_sel_len,
                               int32_t* d_limits, cr_stream_t stream)
{
    if (n_requests == 0) return CR_OK;
    const uint64_t room = static_cast<uint64_t>(table_cols) * page_size;
    if (!visible || !power_of_two(page_size) || !d_starts || !d_kv_len || !d_sel_len || table_stride < table_cols ||
        (n_tokens && !d_limits) || (room && (!d_table || !d_sel)) || sel_stride < room) {
        set_error("cr_paged_select: invalid argument (a row of the selection holds table_cols * page_size slots)");
        return CR_ERR_INVALID;
    }
    const uint64_t n_slots = static_cast<uint64_t>(n_pages) * page_size;
    SelectArgs a{};
    a.chunks = static_cast<uint32_t>(std::max<uint64_t>(1, (room + SL_POS - 1) / SL_POS));
    if (n_slots >> 31 || room >> 31 || n_tokens >> 31 || (static_cast<uint64_t>(a.chunks) * n_requests) >> 31) {
        set_error("cr_paged_select: supported up to 2^31 - 1 slots, positions and tokens");
        return CR_ERR_UNSUPPORTED;
    }
    hipStream_t s = as_stream(stream);
    a.n_words = static_cast<uint32_t>((n_slots + 31) / 32);
    a.table = d_table;
    a.cols = table_cols;
    a.table_stride = table_stride;
    a.starts = d_starts;
    a.kv_len = d_kv_len;
    a.n_requests = n_requests;
    a.page_lg = static_cast<uint32_t>(__builtin_ctz(page_size));
    a.n_pages = n_pages;
    a.n_tokens = n_tokens;
    a.sel = d_sel;
    a.sel_stride = sel_stride;
    a.sel_len = d_sel_len;
    a.limits = d_limits;
    Carver cv;
    const size_t o_words = cv.add(a.n_words * 4ull);
    const size_t o_counts = cv.add(a.chunks > 1 ? 4ull * a.chunks * n_requests : 0);
    Scratch sc;
    CR_RET(sc.alloc(cv.total, s));
    a.words = sc.at<uint32_t>(o_words);
    a.counts = sc.at<uint32_t>(o_counts);
    CR_RET(cr_decompress_to_bitset(visible, sc.at<uint32_t>(o_words), a.n_words, stream));
    const uint32_t grid = a.chunks * n_requests;
    CR_TIMED("pg_select", s);
    if (a.chunks > 1) sl_count<<<grid, SL_NT, 0, s>>>(a);
    sl_write<<<grid, SL_NT, 0, s>>>(a);
    CR_LAUNCH_CHECK();
    return CR_OK;
}

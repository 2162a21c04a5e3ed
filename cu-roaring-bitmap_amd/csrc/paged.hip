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
#include "set_bits.hpp"

namespace crimpl {

namespace {

constexpr int PG_NT = 1024;             // the plan's workgroup
constexpr uint32_t PG_BLOCK = 2048;     // pages a block of the free set holds: 64 words
constexpr uint32_t PG_GROUP = 64;       // blocks that a workgroup of pg_count counts
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
    SetBits free;
    uint32_t n_quads;   // pieces of 128 pages
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
    uint32_t* upto;      // [n_requests + 1] pages that the requests before want
    uint32_t* block_n;   // [n_blocks] free pages of each block
    uint32_t* group_n;   // [n_groups] and of PG_GROUP blocks
    uint32_t n_groups;
    uint64_t* wanted;    // the pages that all requests want; those of requests that can not be
};

// Pages [128 q, 128 q + 128) of the free set for N values of q, without bits
// past the last page.  No load depends on a branch, so that those of all N are
// in flight together.
template <uint32_t N>
__device__ __forceinline__ void free_quads(const SetBits& f, const uint32_t (&q)[N], uint32_t n_quads, uint4 (&x)[N])
{
    if (f.flat) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) x[i] = reinterpret_cast<const uint4*>(f.flat)[min(q[i], n_quads - 1)];
    } else {
        uint32_t c[N], at[N];
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) c[i] = f.key_index[min(q[i] / 512u, f.max_key)];
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            c[i] = q[i] / 512u <= f.max_key ? c[i] : 0xFFFFu;
            at[i] = f.offsets[c[i] != 0xFFFFu ? c[i] : 0u] / 8u;
        }
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) x[i] = reinterpret_cast<const uint4*>(f.bitmaps + at[i])[q[i] % 512u];
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            const uint32_t keep = c[i] != 0xFFFFu ? 0xFFFFFFFFu : 0u;
            x[i] = make_uint4((x[i].x & keep) ^ f.flip, (x[i].y & keep) ^ f.flip, (x[i].z & keep) ^ f.flip,
                              (x[i].w & keep) ^ f.flip);
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        if (q[i] < f.end / 128u) continue;
        const uint32_t left = q[i] > f.end / 128u ? 0u : f.end % 128u;  // of these
        auto cut = [&](uint32_t w, uint32_t k) {
            return left >= 32u * k + 32u ? w : left <= 32u * k ? 0u : w & ((1u << (left - 32u * k)) - 1u);
        };
        x[i] = make_uint4(cut(x[i].x, 0), cut(x[i].y, 1), cut(x[i].z, 2), cut(x[i].w, 3));
    }
}

__device__ __forceinline__ uint4 free_quad(const SetBits& f, uint32_t q, uint32_t n_quads)
{
    const uint32_t at[1] = {q};
    uint4 x[1];
    free_quads(f, at, n_quads, x);
    return x[0];
}

__device__ __forceinline__ uint32_t count_quad(uint4 x)
{
    return __popc(x.x) + __popc(x.y) + __popc(x.z) + __popc(x.w);
}

// The place of the n-th set bit of w (it has more than n).
__device__ __forceinline__ uint32_t nth_bit(uint32_t w, uint32_t n)
{
    uint32_t at = 0;
#pragma unroll
    for (uint32_t half = 16; half > 0; half >>= 1) {
        const uint32_t low = __popc(w & ((1u << half) - 1u));
        const bool up = n >= low;
        n -= up ? low : 0u;
        at += up ? half : 0u;
        w = up ? w >> half : w & ((1u << half) - 1u);
    }
    return at;
}

__device__ __forceinline__ uint32_t nth_of_quad(uint4 x, uint32_t n)
{
    uint32_t at = 0, w = x.x;
    if (const uint32_t c = __popc(w); n >= c) { n -= c; w = x.y; at = 32;
        if (const uint32_t d = __popc(w); n >= d) { n -= d; w = x.z; at = 64;
            if (const uint32_t e = __popc(w); n >= e) { n -= e; w = x.w; at = 96; } } }
    return at + nth_bit(w, n);
}

struct Request {
    uint64_t tokens, held, most;
    bool fits;  // lengths are not negative and the row holds the pages
};

__device__ __forceinline__ uint64_t pages_held(const PlanArgs& a, int32_t cached)
{
    return (static_cast<uint64_t>(max(cached, 0)) + ((1ull << a.page_lg) - 1)) >> a.page_lg;
}

__device__ __forceinline__ Request request_of(const PlanArgs& a, int32_t c, int32_t n)
{
    const uint64_t page = 1ull << a.page_lg;
    Request q;
    q.tokens = n > 0 ? static_cast<uint64_t>(n) : 0ull;
    const uint64_t before = c > 0 ? static_cast<uint64_t>(c) : 0ull;
    q.held = pages_held(a, c);
    q.most = (before + q.tokens + page - 1) >> a.page_lg;
    q.fits = c >= 0 && n >= 0 && q.most <= a.cols && before + q.tokens <= 0x7FFFFFFFull;
    return q;
}

// The pages that a request wants.
__device__ __forceinline__ uint64_t pages_of(const Request& q) { return q.fits ? q.most - q.held : 0ull; }

// The last entry of a[lo, hi) that is at most v (a[lo] <= v, ascending).
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

// The entries [lo, hi) among which the last one at most v lies, for every v of
// [v0, v1]; a wave searches 64 entries at a time, for both ends at once.
template <class T>
__device__ __forceinline__ void wave_range(const T* a, uint32_t n, T v0, T v1, uint32_t& lo, uint32_t& hi)
{
    const uint32_t lane = __lane_id();
    uint32_t l0 = 0, l1 = 0;
    for (uint32_t len = n; len > 1;) {
        const uint32_t step = (len + 63) / 64, i = lane * step;
        const T x = a[min(l0 + i, n - 1)], y = a[min(l1 + i, n - 1)];
        const uint32_t c0 = static_cast<uint32_t>(__popcll(__ballot(i < len && l0 + i < n && x <= v0)));
        const uint32_t c1 = static_cast<uint32_t>(__popcll(__ballot(i < len && l1 + i < n && y <= v1)));
        l0 += (max(c0, 1u) - 1) * step;
        l1 += (max(c1, 1u) - 1) * step;
        len = step;
    }
    lo = l0;
    hi = l1 + 1;
}

// The requests' token offsets and the pages wanted before each of them, a
// workgroup's work; `upto` may lie in LDS.  c, n: the lengths of request
// threadIdx.x, loaded before.  Returns the pages wanted in all; *s_unfit receives
// those of requests that can not be, whatever is free.  The offsets go to
// a.starts, or to s_start if it is there.  ONCE: there are at most PG_NT requests
// (without a loop around it, a decoding step's plan takes 8.4 instead of 9.9 us).
template <bool ONCE>
__device__ __forceinline__ uint64_t scan_requests(const PlanArgs& a, int32_t c, int32_t n, uint32_t* upto,
                                                  uint64_t* s_scan, uint64_t* s_unfit, int32_t* s_start)
{
    const uint32_t t = threadIdx.x;
    uint64_t tokens = 0, pages = 0;
    if (t == 0) *s_unfit = 0;
    for (uint32_t r0 = 0; r0 < (ONCE ? 1u : a.n_requests); r0 += PG_NT) {
        const uint32_t r = r0 + t;
        Request q{0, 0, 0, true};
        if (r < a.n_requests) {
            if (r0) {
                c = a.cached[r];
                n = a.fresh[r];
            }
            q = request_of(a, c, n);
        }
        uint64_t all_tokens, all_pages;
        const uint64_t at = tokens + block_excl_scan_u64<PG_NT>(q.tokens, s_scan, all_tokens);
        const uint64_t before = pages + block_excl_scan_u64<PG_NT>(pages_of(q), s_scan, all_pages);
        if (r < a.n_requests) {
            const int32_t start = static_cast<int32_t>(min(at, static_cast<uint64_t>(0x7FFFFFFF)));
            if (s_start)
                s_start[r] = start;
            else
                a.starts[r] = start;
            upto[r] = static_cast<uint32_t>(min(before, static_cast<uint64_t>(0xFFFFFFFF)));
        }
        if (!q.fits)
            atomicAdd(reinterpret_cast<unsigned long long*>(s_unfit), static_cast<unsigned long long>(q.most - q.held));
        tokens += all_tokens;
        pages += all_pages;
    }
    if (t == 0) {
        upto[a.n_requests] = static_cast<uint32_t>(min(pages, static_cast<uint64_t>(0xFFFFFFFF)));
        const int32_t all = static_cast<int32_t>(min(tokens, static_cast<uint64_t>(0x7FFFFFFF)));
        if (s_start)
            s_start[a.n_requests] = all;
        else
            a.starts[a.n_requests] = a.counts[0] = all;
    }
    __syncthreads();
    return pages;
}

// Of n_free pages, those that are taken: what the requests want up to the first
// whose pages are not all there.  (Later ones want no fewer before them, so that
// only those that want none still get theirs.)
__device__ __forceinline__ uint32_t pages_taken(const uint32_t* upto, uint32_t n_requests, uint32_t n_free)
{
    const uint32_t all = upto[n_requests];
    return all <= n_free ? all : upto[last_at_most(upto, 0u, n_requests + 1, n_free)];
}

// The length of a request's cache after its new tokens, 0 where it is refused.
__device__ __forceinline__ int32_t planned_len(const PlanArgs& a, int32_t c, int32_t n, uint32_t before,
                                               uint32_t n_taken)
{
    const Request q = request_of(a, c, n);
    const uint64_t need = pages_of(q);
    return q.fits && (need == 0 || before + need <= n_taken) ? c + n : 0;
}

__device__ __forceinline__ void set_counts(const PlanArgs& a, uint32_t n_taken, uint64_t wanted, uint64_t unfit)
{
    a.counts[1] = static_cast<int32_t>(n_taken);
    a.counts[2] = static_cast<int32_t>(min(wanted - n_taken + unfit, static_cast<uint64_t>(0x7FFFFFFF)));
}

// Page `id` is the rank-th taken: into the list, and into the table of request
// r, which holds `cached` tokens and before which `before` pages are taken.
__device__ __forceinline__ void place_page(const PlanArgs& a, uint32_t rank, uint32_t id, uint32_t r, int32_t cached,
                                           uint32_t before)
{
    const uint64_t col = pages_held(a, cached) + (rank - before);
    if (rank < a.taken_cap) a.taken[rank] = static_cast<int32_t>(id);
    if (col < a.cols) a.table[r * a.table_stride + col] = static_cast<int32_t>(id);
}

// The slot of the token that is `in` places into request r's new ones.
__device__ __forceinline__ int64_t slot_at(const PlanArgs& a, uint32_t r, int32_t kv_len, int32_t cached, uint32_t in)
{
    const uint32_t pos = static_cast<uint32_t>(cached) + in, col = pos >> a.page_lg;
    if (kv_len <= 0 || col >= a.cols) return -1;
    return (static_cast<int64_t>(a.table[r * a.table_stride + col]) << a.page_lg) + (pos & ((1u << a.page_lg) - 1u));
}

// A large plan, in three launches: the first two are bound by the latency of a few
// dependent loads, the last writes 8 bytes a token (1024 requests, 4.2 million
// tokens, 2^20 pages: 4.5 + 8.3 + 12 us; the writing alone takes 7.1 at the card's
// copy rate; one workgroup for all the counting and the scan took 10.6).
//
// The first workgroup scans the requests, the others count the free pages of
// PG_GROUP blocks each, a row of 16 lanes a block.
__global__ __launch_bounds__(PG_NT) void pg_count(PlanArgs a)
{
    constexpr uint32_t QPB = PG_BLOCK / 128u;  // pieces of a block
    static_assert(QPB == 16 && PG_GROUP * QPB == PG_NT, "a row of 16 lanes per block");
    __shared__ uint64_t s_scan[PG_NT / 64], s_unfit;
    __shared__ uint32_t s_sum[PG_NT / 64];
    const uint32_t t = threadIdx.x;
    if (blockIdx.x == 0) {
        const int32_t c = t < a.n_requests ? a.cached[t] : 0, n = t < a.n_requests ? a.fresh[t] : 0;
        const uint64_t wanted = scan_requests<false>(a, c, n, a.upto, s_scan, &s_unfit, nullptr);
        if (t == 0) {
            a.wanted[0] = wanted;
            a.wanted[1] = s_unfit;
        }
        return;
    }
    const uint32_t group = blockIdx.x - 1, q = group * PG_NT + t, block = q / QPB;
    uint32_t k = count_quad(free_quad(a.free, q, a.n_quads));
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) k += static_cast<uint32_t>(__shfl_xor(static_cast<int>(k), o, 64));
    if (t % QPB == 0 && block < a.n_blocks) a.block_n[block] = k;
    k += static_cast<uint32_t>(__shfl_xor(static_cast<int>(k), 16, 64));
    k += static_cast<uint32_t>(__shfl_xor(static_cast<int>(k), 32, 64));
    if (__lane_id() == 0) s_sum[t / 64] = k;
    __syncthreads();
    if (t == 0) {
        uint32_t all = 0;
#pragma unroll
        for (uint32_t i = 0; i < PG_NT / 64; ++i) all += s_sum[i];
        a.group_n[group] = all;
    }
}

// A workgroup per block of the free set: its pages that are taken, into the
// list of them and into the tables of the requests that take them.  The
// workgroups behind those tell which requests got their pages.
__global__ __launch_bounds__(PG_TAKE_NT) void pg_take(PlanArgs a)
{
    constexpr uint32_t PER = PG_BLOCK / PG_TAKE_NT;  // pages a thread looks at
    __shared__ uint32_t s_scan[PG_TAKE_NT / 64];
    __shared__ uint16_t s_id[PG_BLOCK];
    const uint32_t t = threadIdx.x, group = blockIdx.x / PG_GROUP;
    const uint32_t first = blockIdx.x * PG_BLOCK + t * PER;
    uint32_t bits = 0, before = 0, in_all = 0;
    if (first / 128u < a.n_quads) {
        const uint4 x = free_quad(a.free, first / 128u, a.n_quads);
        const uint32_t w = first / 32u % 4u;
        bits = ((w == 0 ? x.x : w == 1 ? x.y : w == 2 ? x.z : x.w) >> (first % 32u)) & ((1u << PER) - 1u);
    }
    for (uint32_t i = t; i < a.n_groups; i += PG_TAKE_NT) {
        const uint32_t n = a.group_n[i];
        in_all += n;
        before += i < group ? n : 0u;
    }
    if (t < blockIdx.x % PG_GROUP && blockIdx.x < a.n_blocks) before += a.block_n[group * PG_GROUP + t];
    uint32_t base, n_free;
    block_excl_scan<PG_TAKE_NT>(before, s_scan, base);
    block_excl_scan<PG_TAKE_NT>(in_all, s_scan, n_free);
    const uint32_t n_taken = pages_taken(a.upto, a.n_requests, n_free);
    if (blockIdx.x >= a.n_blocks) {
        const uint32_t r = (blockIdx.x - a.n_blocks) * PG_TAKE_NT + t;
        if (r < a.n_requests) a.kv_len[r] = planned_len(a, a.cached[r], a.fresh[r], a.upto[r], n_taken);
        if (r == 0) set_counts(a, n_taken, a.wanted[0], a.wanted[1]);
        return;
    }
    if (base >= n_taken) return;
    uint32_t total;
    uint32_t at = block_excl_scan<PG_TAKE_NT>(__popc(bits), s_scan, total);
    for (; bits; bits &= bits - 1u) s_id[at++] = static_cast<uint16_t>(t * PER + __ffs(bits) - 1);
    __syncthreads();
    const uint32_t n = min(total, n_taken - base);
    if (n == 0) return;
    uint32_t lo, hi;
    wave_range(a.upto, a.n_requests, base, base + n - 1, lo, hi);
    for (uint32_t i = t; i < n; i += PG_TAKE_NT) {
        const uint32_t rank = base + i, r = last_at_most(a.upto, lo, hi, rank);
        place_page(a, rank, blockIdx.x * PG_BLOCK + s_id[i], r, a.cached[r], a.upto[r]);
    }
}

// The slot of each new token, from the tables as pg_take left them, two tokens a
// thread at a time, past the caches (12 us; through them 13.5).  The requests of
// the workgroup's tokens are kept in LDS (searched in memory, 15.9 us).  Each token
// still looks for its request and reads its page's entry by itself.
__global__ __launch_bounds__(PG_FILL_NT) void pg_slots(PlanArgs a, bool pairs)
{
    __shared__ int32_t s_start[PG_FILL_NT], s_kv[PG_FILL_NT], s_cached[PG_FILL_NT];
    const uint32_t first = blockIdx.x * PG_TOKENS, t = threadIdx.x;
    const uint32_t total = min(a.slots_cap, static_cast<uint32_t>(a.starts[a.n_requests]));
    uint32_t lo, hi;
    wave_range(a.starts, a.n_requests, static_cast<int32_t>(first),
               static_cast<int32_t>(min(first + PG_TOKENS, a.slots_cap) - 1), lo, hi);
    if (first >= total) return;
    const uint32_t n = min(PG_TOKENS, total - first);
    const bool held = hi - lo <= PG_FILL_NT;
    if (held && t < hi - lo) {
        s_start[t] = a.starts[lo + t];
        s_kv[t] = a.kv_len[lo + t];
        s_cached[t] = a.cached[lo + t];
    }
    __syncthreads();
    auto slot_of = [&](uint32_t i) {
        const int32_t token = static_cast<int32_t>(first + i);
        if (held) {
            const uint32_t r = last_at_most(s_start, 0u, hi - lo, token);
            return slot_at(a, lo + r, s_kv[r], s_cached[r], static_cast<uint32_t>(token - s_start[r]));
        }
        const uint32_t r = last_at_most(a.starts, lo, hi, token);
        return slot_at(a, r, a.kv_len[r], a.cached[r], static_cast<uint32_t>(token - a.starts[r]));
    };
    typedef int64_t pair __attribute__((ext_vector_type(2)));
    if (pairs && n == PG_TOKENS) {
#pragma unroll
        for (uint32_t j = 0; j < PG_TOKENS / (2 * PG_FILL_NT); ++j) {
            const uint32_t i = 2 * (j * PG_FILL_NT + t);
            pair z;
            z[0] = slot_of(i);
            z[1] = slot_of(i + 1);
            __builtin_nontemporal_store(z, reinterpret_cast<pair*>(a.slots + first + i));
        }
    } else {
        for (uint32_t i = t; i < n; i += PG_FILL_NT) a.slots[first + i] = slot_of(i);
    }
}

// The whole plan in one workgroup, for a decoding step: the free pages before
// each piece of 128, the offsets and the takers' ranks stay in LDS.  Bound by
// latency: 64 requests of 8192 pages 8.4 us (with the offsets in memory 9.7).
constexpr uint32_t PS_QUADS = 2048, PS_REQUESTS = 1024, PS_TOKENS = 8192;

__global__ __launch_bounds__(PG_NT) void pg_small(PlanArgs a)
{
    constexpr uint32_t PER = PS_QUADS / PG_NT;
    __shared__ uint64_t s_scan[PG_NT / 64];
    __shared__ uint64_t s_unfit;
    __shared__ uint32_t s_sum[PG_NT / 64];
    __shared__ uint32_t s_pre[PS_QUADS], s_upto[PS_REQUESTS + 1];
    __shared__ int32_t s_start[PS_REQUESTS + 1], s_kv[PS_REQUESTS], s_cached[PS_REQUESTS];
    static_assert(PS_REQUESTS <= PG_NT, "a thread per request");
    const uint32_t t = threadIdx.x;
    const int32_t c = t < a.n_requests ? a.cached[t] : 0, fresh = t < a.n_requests ? a.fresh[t] : 0;
    uint4 x[PER];
    uint32_t q[PER], n[PER], mine = 0, n_free;
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) q[i] = t * PER + i;
    if (a.n_quads) free_quads(a.free, q, a.n_quads, x);
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        n[i] = a.n_quads ? count_quad(x[i]) : 0u;
        mine += n[i];
    }
    uint32_t before = block_excl_scan<PG_NT>(mine, s_sum, n_free);
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        s_pre[t * PER + i] = before;
        before += n[i];
    }
    if (t < a.n_requests) s_cached[t] = c;
    const uint64_t wanted = scan_requests<true>(a, c, fresh, s_upto, s_scan, &s_unfit, s_start);
    const uint32_t n_taken = pages_taken(s_upto, a.n_requests, n_free);
    for (uint32_t rank = t; rank < n_taken; rank += PG_NT) {
        // pieces without a free page start where the next one does
        const uint32_t q = last_at_most(s_pre, 0u, PS_QUADS, rank);
        const uint32_t r = last_at_most(s_upto, 0u, a.n_requests, rank);
        const uint32_t id = q * 128u + nth_of_quad(free_quad(a.free, q, a.n_quads), rank - s_pre[q]);
        place_page(a, rank, id, r, s_cached[r], s_upto[r]);
    }
    if (t < a.n_requests) s_kv[t] = planned_len(a, c, fresh, s_upto[t], n_taken);
    __syncthreads();
    const uint32_t total = min(a.slots_cap, static_cast<uint32_t>(s_start[a.n_requests]));
    for (uint32_t i = t; i < total; i += PG_NT) {
        const uint32_t r = last_at_most(s_start, 0u, a.n_requests, static_cast<int32_t>(i));
        a.slots[i] = slot_at(a, r, s_kv[r], s_cached[r], i - static_cast<uint32_t>(s_start[r]));
    }
    // (Before a barrier, or a load, these stores would be waited for.)
    for (uint32_t r = t; r <= a.n_requests; r += PG_NT) a.starts[r] = s_start[r];
    if (t < a.n_requests) a.kv_len[t] = s_kv[t];
    if (t == 0) {
        a.counts[0] = s_start[a.n_requests];
        set_counts(a, n_taken, wanted, s_unfit);
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

// Bound by memory: a thread moves one piece of the keys and of the values, both
// past the caches (30011 tokens of 8 x 128: 43.9 us, 5.6 TB/s read and written;
// with ordinary stores 47.5; four pieces a thread 45.4 and 49.1; the card copies
// 1 GiB at 4.75).
template <class U>
__global__ __launch_bounds__(AP_NT) void pg_append(AppendArgs a)
{
    const uint32_t row = a.heads * a.units, i = blockIdx.x * AP_NT + threadIdx.x;
    if (i >= a.n_tokens * row) return;
    const uint32_t token = i / row, in = i % row, head = in / a.units, unit = in % a.units;
    const int64_t slot = a.slots[token];
    if (slot < 0 || static_cast<uint64_t>(slot) >= a.n_slots) return;
    const uint64_t page = static_cast<uint64_t>(slot) >> a.page_lg, off = slot & ((1u << a.page_lg) - 1u);
    U x[2];
#pragma unroll
    for (int c = 0; c < 2; ++c)
        x[c] = __builtin_nontemporal_load(
            reinterpret_cast<const U*>(a.src[c] + token * a.src_token[c] + head * a.src_head[c] + unit * sizeof(U)));
#pragma unroll
    for (int c = 0; c < 2; ++c)
        __builtin_nontemporal_store(x[c], reinterpret_cast<U*>(a.dst[c] + page * a.dst_page[c] + off * a.dst_slot[c] +
                                                               head * a.dst_head[c] + unit * sizeof(U)));
}

// ---- select --------------------------------------------------------------------
// A wave looks at 32 positions a lane: the bits of the pages that hold them are
// the positions' own, in words (or parts of one, where a page is shorter).
// Bound by the latency of its look-ups, so that many workgroups of one wave do it
// (4 requests of 131072 positions: 10 us; 17.4 with the bitmap written out as
// flat words first, 8192 positions a workgroup and a table look-up for each slot).
constexpr int SL_NT = 64;
constexpr uint32_t SL_POS = 32 * SL_NT;
// Up to this many look-ups a lane, a workgroup counts what lies before its chunk by
// itself; above, a launch of its own counts every chunk.  (8 requests, us counted and
// alone: 16 look-ups 9.5 and 8.1 in pages of 64, 9.5 and 7.9 in pages of 16; 32 of
// them 8.9 and 12.3, 8.9 and 12.4; 4 of them, 8192 positions in pages of 64, 8.8 and 6.5.)
constexpr uint32_t SL_ALONE = 16;

struct SelectArgs {
    SetBits visible;  // slots
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
    uint32_t* counts;  // [n_requests][chunks] visible positions, or nullptr: each workgroup counts those before it
};

__device__ __forceinline__ uint32_t select_len(const SelectArgs& a, uint32_t r)
{
    // (Not `n <= 0 ? 0 : min(most, n)`: the compiler moves the min before the test and then takes n for positive.)
    const uint64_t n = static_cast<uint64_t>(max(a.kv_len[r], 0));
    return static_cast<uint32_t>(min(static_cast<uint64_t>(a.cols) << a.page_lg, n));
}

// Calls f(first position, first slot, visible bits) for each page, or 32
// positions of one, among the 32 positions from p0 (a multiple of 32).
template <class F>
__device__ __forceinline__ void visible_parts(const SelectArgs& a, uint32_t r, uint32_t p0, uint32_t len, F f)
{
    const int32_t* row = a.table + r * a.table_stride;
    const uint32_t lg = min(a.page_lg, 5u), part = 1u << lg;
    for (uint32_t p = p0; p < min(len, p0 + 32u); p += part) {
        const uint32_t page = static_cast<uint32_t>(row[p >> a.page_lg]);
        if (page >= a.n_pages) continue;
        const uint32_t slot = (page << a.page_lg) + (p & ((1u << a.page_lg) - 1u));
        if (slot >= a.visible.end) continue;
        uint32_t bits = a.visible.word(slot >> 5) >> (slot & 31u);
        const uint32_t n = min(part, len - p);
        if (n < 32u) bits &= (1u << n) - 1u;
        f(p, slot, bits);
    }
}

__device__ __forceinline__ uint32_t wave_total(uint32_t v)
{
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(wave_incl_scan(v)), 63));
}

__global__ __launch_bounds__(SL_NT) void sl_count(SelectArgs a)
{
    const uint32_t r = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    uint32_t n = 0;
    visible_parts(a, r, chunk * SL_POS + threadIdx.x * 32u, select_len(a, r),
                  [&](uint32_t, uint32_t, uint32_t bits) { n += __popc(bits); });
    n = wave_total(n);
    if (threadIdx.x == 0) a.counts[blockIdx.x] = n;
}

// The visible ones among this lane's positions of the chunks before `chunk`, all of
// which are the request's.
__device__ __forceinline__ uint32_t visible_before(const SelectArgs& a, uint32_t r, uint32_t chunk)
{
    constexpr uint32_t N = 8;  // look-ups side by side
    if (a.visible.end == 0) return 0;
    const int32_t* row = a.table + r * a.table_stride;
    const uint32_t lg = min(a.page_lg, 5u), parts_lg = 5u - lg, items = chunk << parts_lg;
    const uint32_t keep = 0xFFFFFFFFu >> (32u - (1u << lg));
    uint32_t n = 0;
    for (uint32_t i = 0; i < items; i += N) {
        uint32_t slot[N], w[N], x[N];
        bool in[N];
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) {
            const uint32_t u = min(i + j, items - 1u);
            const uint32_t p = (u >> parts_lg) * SL_POS + threadIdx.x * 32u + ((u & ((1u << parts_lg) - 1u)) << lg);
            const uint32_t page = static_cast<uint32_t>(row[p >> a.page_lg]);
            slot[j] = (page << a.page_lg) + (p & ((1u << a.page_lg) - 1u));
            in[j] = i + j < items && page < a.n_pages && slot[j] < a.visible.end;
            w[j] = in[j] ? slot[j] >> 5 : 0u;
        }
        a.visible.words(w, x);
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) n += in[j] ? __popc((x[j] >> (slot[j] & 31u)) & keep) : 0u;
    }
    return n;
}

// visible_parts for pages of 8 or more, looked up once and side by side: slot[j] and
// bits[j] of the lane's part j, of at most SL_PARTS.
constexpr uint32_t SL_PARTS = 4;
__device__ __forceinline__ void visible_own(const SelectArgs& a, uint32_t r, uint32_t p0, uint32_t len,
                                            uint32_t (&slot)[SL_PARTS], uint32_t (&bits)[SL_PARTS])
{
    const int32_t* row = a.table + r * a.table_stride;
    const uint32_t lg = min(a.page_lg, 5u), part = 1u << lg;
    uint32_t w[SL_PARTS];
    bool in[SL_PARTS];
#pragma unroll
    for (uint32_t j = 0; j < SL_PARTS; ++j) {
        const uint32_t p = min(p0 + (j << lg), len - 1u);
        const uint32_t page = static_cast<uint32_t>(row[p >> a.page_lg]);
        slot[j] = (page << a.page_lg) + (p & ((1u << a.page_lg) - 1u));
        in[j] = j << lg < 32u && p0 + (j << lg) < len && page < a.n_pages && slot[j] < a.visible.end;
        w[j] = in[j] ? slot[j] >> 5 : 0u;
    }
    a.visible.words(w, bits);
#pragma unroll
    for (uint32_t j = 0; j < SL_PARTS; ++j) {
        const uint32_t n = in[j] ? min(part, len - p0 - (j << lg)) : 0u;  // positions there are
        bits[j] = n ? (bits[j] >> (slot[j] & 31u)) & (0xFFFFFFFFu >> (32u - n)) : 0u;
    }
}

__global__ __launch_bounds__(SL_NT) void sl_write(SelectArgs a)
{
    __shared__ int32_t s_slot[SL_POS];
    __shared__ uint32_t s_vis[SL_NT], s_before[SL_NT];
    const uint32_t r = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, t = threadIdx.x;
    const uint32_t len = select_len(a, r), p0 = chunk * SL_POS + t * 32u;
    // positions of the new tokens: the last of the request's
    const int32_t t0 = min(max(a.starts[r], 0), static_cast<int32_t>(a.n_tokens));
    const int32_t t1 = min(max(a.starts[r + 1], t0), static_cast<int32_t>(a.n_tokens));
    // position p is new token p + shift: by the request's own length, of which the table may not hold all
    const int64_t shift = static_cast<int64_t>(t1) - a.kv_len[r];
    if (chunk == 0) {  // tokens before the first position see nothing
        for (int64_t i = t0 + t; i < min(static_cast<int64_t>(t1), shift); i += SL_NT) a.limits[i] = 0;
    }
    if (chunk * SL_POS >= len && chunk > 0) return;
    uint32_t base = 0;
    if (a.counts) {
        for (uint32_t i = t; i < chunk; i += SL_NT) base += a.counts[r * a.chunks + i];
    } else {
        base = visible_before(a, r, chunk);
    }
    uint32_t vis = 0, own_slot[SL_PARTS] = {}, own[SL_PARTS] = {};
    if (a.page_lg >= 3) {
        if (len && a.visible.end) visible_own(a, r, p0, len, own_slot, own);
#pragma unroll
        for (uint32_t j = 0; j < SL_PARTS; ++j) vis |= own[j] << ((j << a.page_lg) & 31u);  // (0 from the last part on)
    } else {
        visible_parts(a, r, p0, len, [&](uint32_t p, uint32_t, uint32_t bits) { vis |= bits << (p - p0); });
    }
    base = wave_total(base);
    const uint32_t n = __popc(vis), upto = wave_incl_scan(n), before = upto - n;
    const uint32_t total = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), 63));
    uint32_t at = before;
    auto list = [&](uint32_t, uint32_t slot, uint32_t bits) {
        for (; bits; bits &= bits - 1u) s_slot[at++] = static_cast<int32_t>(slot + __ffs(bits) - 1);
    };
    if (a.page_lg >= 3) {
#pragma unroll
        for (uint32_t j = 0; j < SL_PARTS; ++j) list(0, own_slot[j], own[j]);
    } else {
        visible_parts(a, r, p0, len, list);
    }
    s_vis[t] = vis;
    s_before[t] = base + before;
    __syncthreads();
    // the new tokens' positions in this chunk
    const uint32_t c0 = chunk * SL_POS;
    const uint32_t from = static_cast<uint32_t>(max(static_cast<int64_t>(t0) - shift, static_cast<int64_t>(c0)));
    for (uint32_t p = from + t; p < min(len, c0 + SL_POS); p += SL_NT) {
        const uint32_t k = p - c0;
        a.limits[p + shift] =
            static_cast<int32_t>(s_before[k / 32u] + __popc(s_vis[k / 32u] & (0xFFFFFFFFu >> (31u - k % 32u))));
    }
    for (uint32_t i = t; i < total; i += SL_NT) a.sel[r * a.sel_stride + base + i] = s_slot[i];
    if (len <= SL_POS || chunk == (len - 1) / SL_POS) {
        if (t == 0) a.sel_len[r] = static_cast<int32_t>(base + total);
        // tokens behind the table's last position see all that it holds
        for (int64_t i = max(static_cast<int64_t>(t0), len + shift) + t; i < t1; i += SL_NT)
            a.limits[i] = static_cast<int32_t>(base + total);
    }
}

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
    a.n_quads = (n_pages + 127u) / 128u;
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
    const bool direct = is_direct(free_pages);
    // One workgroup for a decoding step (64 requests, 8192 pages: 19.4 us in several launches, 8.4 in one).
    const bool small = a.n_quads <= PS_QUADS && n_requests <= PS_REQUESTS && slots_cap <= PS_TOKENS;
    Carver cv;
    const size_t o_words = cv.add(direct ? 0 : a.n_quads * 16ull);
    a.n_groups = (a.n_blocks + PG_GROUP - 1) / PG_GROUP;
    const size_t o_upto = cv.add(small ? 0 : (n_requests + 1ull) * 4), o_wanted = cv.add(small ? 0 : 16);
    const size_t o_block = cv.add(small ? 0 : a.n_blocks * 4ull), o_group = cv.add(small ? 0 : a.n_groups * 4ull);
    Scratch sc;
    if (cv.total) CR_RET(sc.alloc(cv.total, s));
    a.upto = sc.at<uint32_t>(o_upto);
    a.wanted = sc.at<uint64_t>(o_wanted);
    a.block_n = sc.at<uint32_t>(o_block);
    a.group_n = sc.at<uint32_t>(o_group);
    CR_RET(set_bits(free_pages, direct, sc.at<uint32_t>(o_words), a.n_quads * 4u, n_pages, stream, &a.free));
    CR_TIMED("pg_plan", s);
    if (small) {
        pg_small<<<1, PG_NT, 0, s>>>(a);
    } else {
        const uint32_t request_blocks = std::max<uint32_t>(1, (n_requests + PG_TAKE_NT - 1) / PG_TAKE_NT);
        pg_count<<<1 + a.n_groups, PG_NT, 0, s>>>(a);
        pg_take<<<a.n_blocks + request_blocks, PG_TAKE_NT, 0, s>>>(a);
        const bool pairs = reinterpret_cast<uintptr_t>(d_slots) % 16 == 0;
        if (slots_cap && n_requests) pg_slots<<<(slots_cap + PG_TOKENS - 1) / PG_TOKENS, PG_FILL_NT, 0, s>>>(a, pairs);
    }
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
    const uint64_t grid = (pieces + AP_NT - 1) / AP_NT;
    if (grid >> 24) {  // a launch holds fewer than 2^32 threads
        set_error("cr_paged_append: too many elements for one call");
        return CR_ERR_UNSUPPORTED;
    }
    hipStream_t s = as_stream(stream);
    CR_TIMED("pg_append", s);
    if (unit == 16)
        pg_append<cr_v4u><<<static_cast<unsigned>(grid), AP_NT, 0, s>>>(a);
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
    if (n_slots >> 31 || room >> 31 || n_tokens >> 31 || (static_cast<uint64_t>(a.chunks) * n_requests) >> 25) {
        set_error("cr_paged_select: supported up to 2^31 - 1 slots, positions and tokens");
        return CR_ERR_UNSUPPORTED;
    }
    hipStream_t s = as_stream(stream);
    const uint32_t n_words = static_cast<uint32_t>((n_slots + 31) / 32);
    const bool direct = is_direct(visible);
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
    const size_t o_words = cv.add(direct ? 0 : n_words * 4ull);
    const bool counted = a.chunks * std::max(1u, 32u / page_size) > SL_ALONE;
    const size_t o_counts = cv.add(counted ? 4ull * a.chunks * n_requests : 0);
    Scratch sc;
    if (cv.total) CR_RET(sc.alloc(cv.total, s));
    if (counted) a.counts = sc.at<uint32_t>(o_counts);
    CR_RET(set_bits(visible, direct, sc.at<uint32_t>(o_words), n_words, static_cast<uint32_t>(n_slots), stream,
                    &a.visible));
    const uint32_t grid = a.chunks * n_requests;
    CR_TIMED("pg_select", s);
    if (counted) sl_count<<<grid, SL_NT, 0, s>>>(a);
    sl_write<<<grid, SL_NT, 0, s>>>(a);
    CR_LAUNCH_CHECK();
    return CR_OK;
}

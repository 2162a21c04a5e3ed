// Rotary positions, for serving language models (no reference implementation):
// queries and keys turned by the angles of their positions, and keys and values
// into their slots of the paged cache.
//
//   a = position * freq_i,  (x, y) -> m (x cos a - y sin a, y cos a + x sin a)
//
// for the pairs (x, y) of a row's first `rotated` dimensions: dimensions i and
// i + rotated / 2, or 2 i and 2 i + 1.  The rest of a row stays as it is.
#include <algorithm>

#include "internal.hpp"
#include "elements.hpp"
#include "rows.hpp"
#include "set_bits.hpp"

namespace crimpl {

namespace {

constexpr int RO_NT = 256;
constexpr uint32_t RO_PAIRS = 2048;  // cosines and sines that a workgroup keeps
constexpr uint32_t RO_AHEAD = 2;     // tokens whose pieces a thread asks for at a time

struct Plane {  // rows of one of the tensors; strides in elements
    const void* src;
    uint64_t src_token, src_head;
    void* dst;
    uint64_t dst_token, dst_head;  // queries
};

struct RotaryArgs {
    Plane q, k, v;
    uint64_t k_page, k_slot, k_head, v_page, v_slot, v_head;  // of the cache
    uint32_t n_tokens, heads, kv_heads, dim, half, magnitude_bits;
    const int32_t* positions;
    const double* freqs;
    const int64_t* slots;
    uint64_t n_slots;
    uint32_t page_lg;
    uint32_t per_row, per_token;   // pairs of pieces
    uint32_t tokens, rounds, side;  // tokens of a workgroup; workgroups that share them; tokens side by side
};

// Cosine and sine of position * freq, in 64 bits until whole turns are taken
// away: a position of 2^20 at one radian each has 17 bits before the point, which
// would leave 32 bits 2^-8 of a radian.  Within an eighth of a turn the first five terms
// of either series are off by less than 2^-29.
__device__ __forceinline__ float2 cos_sin(int32_t position, double freq, float m)
{
    const double turns = static_cast<double>(position) * (freq * 0.15915494309189533577);
    const double part = turns - rint(turns), quarter = rint(part * 4.0);  // [-1/2, 1/2], [-2, 2]
    const float x = static_cast<float>((part - quarter * 0.25) * 6.28318530717958647692), z = x * x;
    float s = __builtin_fmaf(z, 2.7557319224e-6f, -1.9841269841e-4f);
    s = __builtin_fmaf(z, s, 8.3333333333e-3f);
    s = __builtin_fmaf(z, s, -1.6666666667e-1f);
    s = __builtin_fmaf(z * x, s, x);
    float c = __builtin_fmaf(z, -2.7557319224e-7f, 2.4801587302e-5f);
    c = __builtin_fmaf(z, c, -1.3888888889e-3f);
    c = __builtin_fmaf(z, c, 4.1666666667e-2f);
    c = __builtin_fmaf(z, c, -0.5f);
    c = __builtin_fmaf(z, c, 1.0f);
    const int n = static_cast<int>(quarter) & 3;
    const float cn = n & 1 ? s : c, sn = n & 1 ? c : s;
    return make_float2((n == 1 || n == 2 ? -cn : cn) * m, (n >= 2 ? -sn : sn) * m);
}

// Bound by memory: every row once in, once out.  A thread looks after one pair of pieces that
// turn together (or of any two of a row), of all tokens of its workgroup (or of every side-th,
// where a token has few pieces): it works out where they lie once, and asks for those of
// RO_AHEAD tokens at a time, the first ones before the workgroup's cosines are there.
// 30011 tokens of 32 + 2 x 8 heads of 128 in f16: 127 us, 5.8 TB/s (192 where a thread took
// the pieces that came next, wherever they lay); 64 tokens in bf16: 3.5 to 4 us.
template <class E, uint32_t N, bool NEXT>
__global__ __launch_bounds__(RO_NT) void ro_turn(RotaryArgs a)
{
    typedef typename E::Bits Bits;
    typedef Piece<E, N> P;
    __shared__ float2 s_turn[RO_PAIRS];
    const uint32_t t = threadIdx.x, token0 = blockIdx.x / a.rounds * a.tokens;
    const uint32_t end = min(token0 + a.tokens, a.n_tokens), turned = NEXT ? a.half * 2 : a.half;
    const uint32_t first = token0 + (a.side > 1 ? t / a.per_token : 0u);
    const uint32_t item = a.side > 1 ? t % a.per_token : blockIdx.x % a.rounds * blockDim.x + t;
    const bool there = a.side > 1 ? t < a.side * a.per_token : item < a.per_token;
    const uint32_t row = item / a.per_row, c = item % a.per_row * N;
    // The pieces' first dimensions.  Neighbouring threads' pieces lie side by side.
    uint32_t at = c, two = c + (NEXT ? a.per_row * N : a.half);
    if (NEXT && N == 1) {
        at = 2 * c;
        two = at + 1;
    } else if (!NEXT && c >= turned) {
        at = a.half + c;
        two = at + a.per_row * N - a.half;
    }
    const bool both = two < a.dim, query = row < a.heads, key = !query && row < a.heads + a.kv_heads;
    const bool turn = (query || key) && at < turned;
    const uint32_t head = query ? row : key ? row - a.heads : row - a.heads - a.kv_heads;
    const Plane& plane = query ? a.q : key ? a.k : a.v;
    const Bits* from = static_cast<const Bits*>(plane.src) + head * plane.src_head;
    Bits* to = static_cast<Bits*>(plane.dst) + head * (query ? plane.dst_head : key ? a.k_head : a.v_head);
    const uint64_t page_stride = key ? a.k_page : a.v_page, slot_stride = key ? a.k_slot : a.v_slot;
    P x[RO_AHEAD], y[RO_AHEAD];
    int64_t slot[RO_AHEAD];
    auto load = [&](uint32_t token) {
#pragma unroll
        for (uint32_t j = 0; j < RO_AHEAD; ++j) {
            const uint32_t i = token + j * a.side;
            if (i >= end) continue;
            slot[j] = query ? 0 : a.slots[i];
            x[j] = P::load(from + i * plane.src_token + at);
            y[j] = P::load(from + i * plane.src_token + (both ? two : at));
        }
    };
    auto pair = [](float2 w, float u, float v) {
        return make_float2(__builtin_fmaf(u, w.x, -(v * w.y)), __builtin_fmaf(v, w.x, u * w.y));
    };
    auto finish = [&](uint32_t token) {
#pragma unroll
        for (uint32_t j = 0; j < RO_AHEAD; ++j) {
            const uint32_t i = token + j * a.side;
            if (i >= end) continue;
            const float2* w = s_turn + (i - token0) * a.half;
            if (turn) {
                if constexpr (NEXT && N > 1) {
#pragma unroll
                    for (uint32_t e = 0; e < N; e += 2) {
                        if (at + e < turned) {
                            const float2 z = pair(w[(at + e) / 2], x[j].get(e), x[j].get(e + 1));
                            x[j].set(e, z.x);
                            x[j].set(e + 1, z.y);
                        }
                        if (two + e < turned) {
                            const float2 z = pair(w[(two + e) / 2], y[j].get(e), y[j].get(e + 1));
                            y[j].set(e, z.x);
                            y[j].set(e + 1, z.y);
                        }
                    }
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < N; ++e) {
                        const float2 z = pair(w[NEXT ? at / 2 : at + e], x[j].get(e), y[j].get(e));
                        x[j].set(e, z.x);
                        y[j].set(e, z.y);
                    }
                }
            }
            Bits* out = to;
            if (query) {
                out += i * plane.dst_token;
            } else {
                if (slot[j] < 0 || static_cast<uint64_t>(slot[j]) >= a.n_slots) continue;
                out += (static_cast<uint64_t>(slot[j]) >> a.page_lg) * page_stride +
                       (slot[j] & ((1u << a.page_lg) - 1u)) * slot_stride;
            }
            x[j].store(out + at);
            if (both) y[j].store(out + two);
        }
    };
    if (there) load(first);
    const float m = __uint_as_float(a.magnitude_bits);
    for (uint32_t k = t; k < (end - token0) * a.half; k += blockDim.x)
        s_turn[k] = cos_sin(a.positions[token0 + k / a.half], a.freqs[k % a.half], m);
    __syncthreads();
    if (!there) return;
    for (uint32_t i = first; i < end; i += RO_AHEAD * a.side) {
        finish(i);
        load(i + RO_AHEAD * a.side);
    }
}

template <class E, uint32_t N>
void launch_rotary(const RotaryArgs& a, bool next, uint32_t grid, uint32_t threads, hipStream_t s)
{
    if (next)
        ro_turn<E, N, true><<<grid, threads, 0, s>>>(a);
    else
        ro_turn<E, N, false><<<grid, threads, 0, s>>>(a);
}

}  // namespace

}  // namespace crimpl

using namespace crimpl;

extern "C" int cr_paged_rotary(const cr_paged_rotary_args* args, const cr_paged_cache* cache, cr_stream_t stream)
{
    if (!args || !cache) {
        set_error("cr_paged_rotary: invalid argument");
        return CR_ERR_INVALID;
    }
    const cr_paged_rotary_args& p = *args;
    if (p.n_tokens == 0) return CR_OK;
    const uint32_t dim = cache->head_dim;
    if (!p.k || !p.v || !p.d_slots || !cache->k || !cache->v || !power_of_two(cache->page_size) ||
        cache->dtype > CR_BF16 || (p.n_heads && (!p.q || !p.q_out)) || dim == 0 || p.rotated % 2 || p.rotated > dim ||
        (p.rotated && (!p.d_positions || !p.d_freqs))) {
        set_error("cr_paged_rotary: invalid argument (%u of %u dimensions, page size %u)", p.rotated, dim,
                  cache->page_size);
        return CR_ERR_INVALID;
    }
    if (p.rotated / 2 > RO_PAIRS) {
        set_error("cr_paged_rotary: up to %u dimensions are turned (%u)", 2 * RO_PAIRS, p.rotated);
        return CR_ERR_UNSUPPORTED;
    }
    if ((p.n_heads > 1 && p.out_head_stride < dim) || (p.n_heads && p.n_tokens > 1 && p.out_token_stride < dim)) {
        set_error("cr_paged_rotary: invalid argument (rows of the turned queries lie over one another)");
        return CR_ERR_INVALID;
    }
    const uint32_t es = cache->dtype == CR_F32 ? 4 : 2;
    RotaryArgs a{};
    a.q = {p.q, p.q_token_stride, p.q_head_stride, p.q_out, p.out_token_stride, p.out_head_stride};
    a.k = {p.k, p.k_token_stride, p.k_head_stride, cache->k, 0, 0};
    a.v = {p.v, p.v_token_stride, p.v_head_stride, cache->v, 0, 0};
    a.k_page = cache->k_page_stride;
    a.k_slot = cache->k_slot_stride;
    a.k_head = cache->k_head_stride;
    a.v_page = cache->v_page_stride;
    a.v_slot = cache->v_slot_stride;
    a.v_head = cache->v_head_stride;
    a.n_tokens = p.n_tokens;
    a.heads = p.n_heads;
    a.kv_heads = cache->n_heads;
    a.dim = dim;
    a.half = p.rotated / 2;
    a.magnitude_bits = __builtin_bit_cast(uint32_t, p.magnitude);
    a.positions = p.d_positions;
    a.freqs = p.d_freqs;
    a.slots = p.d_slots;
    a.n_slots = static_cast<uint64_t>(cache->n_pages) * cache->page_size;
    a.page_lg = static_cast<uint32_t>(__builtin_ctz(cache->page_size));
    // Pieces of 16 bytes, of 8, or single values: what every row's pieces are aligned
    // to, and what does not reach over the end of the turned dimensions.
    auto over = [](uint32_t extent, uint64_t x, uint64_t y) { return extent > 1 ? x | y : 0; };
    uint64_t all = over(p.n_tokens, p.k_token_stride, p.v_token_stride) |
                   over(cache->n_heads, p.k_head_stride, p.v_head_stride) |
                   over(cache->n_pages, a.k_page, a.v_page) | over(cache->page_size, a.k_slot, a.v_slot) |
                   over(cache->n_heads, a.k_head, a.v_head) | dim;
    uintptr_t at = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
                   reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v);
    if (p.n_heads) {
        all |= over(p.n_tokens, p.q_token_stride, p.out_token_stride) | over(p.n_heads, p.q_head_stride, p.out_head_stride);
        at |= reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.q_out);
    }
    if (!p.interleaved) all |= a.half;
    const uint64_t bytes = all * es | at;
    const uint32_t n = bytes % 16 == 0 ? 16 / es : bytes % 8 == 0 ? 8 / es : 1;
    a.per_row = (dim + 2 * n - 1) / (2 * n);
    const uint64_t per_token = (static_cast<uint64_t>(p.n_heads) + 2ull * cache->n_heads) * a.per_row;
    if (per_token >> 24 || p.n_tokens >> 31) {
        set_error("cr_paged_rotary: too many elements for one call");
        return CR_ERR_UNSUPPORTED;
    }
    if (per_token == 0) return CR_OK;
    const uint64_t row = static_cast<uint64_t>(dim) * es;
    const Rows out(p.q_out, p.n_tokens, p.out_token_stride * es, p.n_heads, p.out_head_stride * es, row);
    const Rows in(p.q, p.n_tokens, p.q_token_stride * es, p.n_heads, p.q_head_stride * es, row);
    if (rows_overlap(out) || rows_overwrite(out, in)) {
        set_error("cr_paged_rotary: invalid argument (rows of the turned queries lie over one another, or over other rows of "
                  "those that are read)");
        return CR_ERR_INVALID;
    }
    a.per_token = static_cast<uint32_t>(per_token);
    // A workgroup's threads share a token's pieces, in several workgroups where there are more,
    // or take several tokens side by side.  Its cosines serve all of its tokens: as many as
    // still leave workgroups for the whole card, and no more than two rounds of loads (30011
    // tokens: 127 us, with four 143, with sixteen 155).
    a.side = std::max(1u, static_cast<uint32_t>(RO_NT) / a.per_token);
    a.rounds = a.side > 1 ? 1u : (a.per_token + RO_NT - 1) / RO_NT;
    const uint32_t threads = a.side > 1 ? RO_NT : ((a.per_token + a.rounds - 1) / a.rounds + 63) / 64 * 64;
    const uint32_t fit = a.half ? RO_PAIRS / a.half : 1u << 16;
    const uint64_t share = static_cast<uint64_t>(p.n_tokens) * a.rounds / (8ull * num_cus());
    a.tokens = static_cast<uint32_t>(std::min<uint64_t>(fit, std::max<uint64_t>(a.side, std::min<uint64_t>(2ull * RO_AHEAD * a.side, share))));
    const uint64_t grid = static_cast<uint64_t>((p.n_tokens + a.tokens - 1) / a.tokens) * a.rounds;
    if (grid >> 23) {  // a launch holds fewer than 2^32 threads
        set_error("cr_paged_rotary: too many tokens for one call");
        return CR_ERR_UNSUPPORTED;
    }
    hipStream_t s = as_stream(stream);
    CR_TIMED("ro_turn", s);
    const uint32_t g = static_cast<uint32_t>(grid);
    const bool next = p.interleaved != 0;
    if (cache->dtype == CR_F32) {
        if (n == 4)
            launch_rotary<F32, 4>(a, next, g, threads, s);
        else if (n == 2)
            launch_rotary<F32, 2>(a, next, g, threads, s);
        else
            launch_rotary<F32, 1>(a, next, g, threads, s);
    } else if (cache->dtype == CR_F16) {
        if (n == 8)
            launch_rotary<F16, 8>(a, next, g, threads, s);
        else if (n == 4)
            launch_rotary<F16, 4>(a, next, g, threads, s);
        else
            launch_rotary<F16, 1>(a, next, g, threads, s);
    } else {
        if (n == 8)
            launch_rotary<BF16, 8>(a, next, g, threads, s);
        else if (n == 4)
            launch_rotary<BF16, 4>(a, next, g, threads, s);
        else
            launch_rotary<BF16, 1>(a, next, g, threads, s);
    }
    CR_LAUNCH_CHECK();
    return CR_OK;
}

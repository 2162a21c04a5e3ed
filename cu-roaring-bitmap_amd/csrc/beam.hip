// Beam search's step (no reference implementation): the best continuations over
// beams and vocabulary, gated by a Roaring bitmap of allowed tokens, and the
// reordering of the beams' states by the parents chosen.
//
//   total(w, v) = cum(w) + (x(w, v) - lse(w))
//
// in fp32, each step rounded once, so that the choice is the same on every
// machine.  A total that is NaN or -inf is no candidate.  The k largest win;
// of equal ones the lowest place w * vocab + v.
//
//   1. bs_scan reads every score once: a wave per group of consecutive tokens
//      of a beam writes the group's largest total.
//   2. bs_pick, a workgroup per answer: the k-th largest of 256 disjoint sets'
//      maxima bounds the k-th total from below; the groups that reach it (about
//      k of them) are read again and their totals at or above it ranked.
// The scores pass by once; what is read again is k groups of an answer.
#include <algorithm>

#include "internal.hpp"

namespace crimpl {

namespace {

constexpr int BS_NT = 256;        // bs_scan: four waves
constexpr int BP_NT = 1024;       // bs_pick
constexpr uint32_t BP_SETS = 256;
constexpr uint32_t BP_CAP = 2048;  // candidates held
constexpr uint32_t BS_KMAX = 256;

struct BeamArgs {
    const void* x;
    uint64_t batch_stride, beam_stride;
    uint32_t batch, beams, vocab;
    const float* cum;
    const float* lse;
    const uint32_t* bits;  // allowed tokens (nullptr: all)
    uint64_t bits_stride;
    uint32_t k;
    uint32_t n_groups;  // of a beam
    float* gmax;        // [batch][beams][n_groups]
    float* out_scores;
    int32_t* out_tokens;
    int32_t* out_parents;
};

struct F16 {
    uint16_t v;
};
struct BF16 {
    uint16_t v;
};
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(BF16 x) { return __uint_as_float(static_cast<uint32_t>(x.v) << 16); }
__device__ __forceinline__ float to_f32(F16 x) { return static_cast<float>(__builtin_bit_cast(_Float16, x.v)); }

// Tokens of a group: what a wave reads with UNROLL 16-byte loads a lane.
template <class T>
struct Group {
    static constexpr uint32_t PER = 16 / sizeof(T);
    static constexpr uint32_t UNROLL = sizeof(T) == 4 ? 2 : 1;
    static constexpr uint32_t SIZE = 64 * PER * UNROLL;
};

// Whole numbers in the order of the totals; 0 for what is no candidate.
__device__ __forceinline__ uint32_t order_of(float total)
{
    if (!(total > -__builtin_inff())) return 0u;
    const uint32_t b = __float_as_uint(total + 0.0f);  // -0 counts as +0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float total_of(const BeamArgs& a, float x, float cum, float lse)
{
    return a.lse ? cum + (x - lse) : cum + x;
}

// A beam's row: its first token at a 16-byte boundary starts the vector loads;
// the tokens before it go with the first group.
template <class T>
struct Row {
    const T* p;
    const uint32_t* bits;
    uint32_t head;
    float cum, lse;
    __device__ __forceinline__ Row(const BeamArgs& a, uint32_t b, uint32_t w)
    {
        p = static_cast<const T*>(a.x) + b * a.batch_stride + w * a.beam_stride;
        head = static_cast<uint32_t>((16u - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / sizeof(T);
        bits = a.bits ? a.bits + (static_cast<uint64_t>(b) * a.beams + w) * a.bits_stride : nullptr;
        cum = a.cum[static_cast<uint64_t>(b) * a.beams + w];
        lse = a.lse ? a.lse[static_cast<uint64_t>(b) * a.beams + w] : 0.0f;
    }
    __device__ __forceinline__ bool allowed(uint32_t v) const { return !bits || ((bits[v >> 5] >> (v & 31u)) & 1u); }
};

// The lane's tokens [v, v + PER) of a row that lie below `vocab` and are
// allowed, as their order (0 for the others).
template <class T>
__device__ __forceinline__ void load_orders(const BeamArgs& a, const Row<T>& row, uint32_t v,
                                            uint32_t (&o)[Group<T>::PER])
{
    constexpr uint32_t PER = Group<T>::PER;
    uint32_t on = 0;
    if (v < a.vocab) {
        const uint32_t n = min(PER, a.vocab - v);
        on = (1u << n) - 1u;
        if (row.bits) {
            const uint32_t w = v >> 5, sh = v & 31u;
            uint64_t two = row.bits[w];
            if (sh + n > 32u) two |= static_cast<uint64_t>(row.bits[w + 1]) << 32;
            on &= static_cast<uint32_t>(two >> sh);
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) o[i] = 0u;
    if (on == 0) return;
    T x[PER];
    if (v + PER <= a.vocab) {
        *reinterpret_cast<uint4*>(x) = ld_stream(reinterpret_cast<const uint4*>(row.p + v));
    } else {
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) x[i] = row.p[min(v + i, a.vocab - 1)];
    }
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i)
        if ((on >> i) & 1u) o[i] = order_of(total_of(a, to_f32(x[i]), row.cum, row.lse));
}

template <class T>
__device__ __forceinline__ uint32_t head_order(const BeamArgs& a, const Row<T>& row, uint32_t v)
{
    if (v >= row.head || v >= a.vocab || !row.allowed(v)) return 0u;
    return order_of(total_of(a, to_f32(row.p[v]), row.cum, row.lse));
}

template <class T>
__global__ __launch_bounds__(BS_NT) void bs_scan(BeamArgs a, uint32_t* __restrict__ gmax)
{
    using G = Group<T>;
    const uint32_t lane = __lane_id();
    const uint64_t id = static_cast<uint64_t>(blockIdx.x) * (BS_NT / 64) + (threadIdx.x >> 6);
    const uint64_t all = static_cast<uint64_t>(a.batch) * a.beams * a.n_groups;
    if (id >= all) return;
    const uint32_t g = static_cast<uint32_t>(id % a.n_groups);
    const uint32_t r = static_cast<uint32_t>(id / a.n_groups);
    const Row<T> row(a, r / a.beams, r % a.beams);
    uint32_t best = g == 0 ? head_order(a, row, lane) : 0u;
#pragma unroll
    for (uint32_t u = 0; u < G::UNROLL; ++u) {
        uint32_t o[G::PER];
        load_orders(a, row, row.head + g * G::SIZE + (u * 64 + lane) * G::PER, o);
#pragma unroll
        for (uint32_t i = 0; i < G::PER; ++i) best = max(best, o[i]);
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) best = max(best, static_cast<uint32_t>(__shfl_xor(static_cast<int>(best), s, 64)));
    if (lane == 0) gmax[id] = best;
}

// Sorts the first n of `key` (n <= BP_CAP) in descending order.
__device__ __forceinline__ void sort_keys(uint64_t* key, uint32_t n)
{
    uint32_t p = 1;
    while (p < n) p <<= 1;
    for (uint32_t i = n + threadIdx.x; i < p; i += BP_NT) key[i] = 0;
    __syncthreads();
    for (uint32_t size = 2; size <= p; size <<= 1) {
        for (uint32_t step = size >> 1; step > 0; step >>= 1) {
            for (uint32_t i = threadIdx.x; i < p / 2; i += BP_NT) {
                const uint32_t lo = 2 * i - (i & (step - 1)), hi = lo + step;
                const bool down = (lo & size) == 0;
                const uint64_t x = key[lo], y = key[hi];
                if ((x < y) == down) {
                    key[lo] = y;
                    key[hi] = x;
                }
            }
            __syncthreads();
        }
    }
}

// Descending order of all keys by counting, for few of them: out[rank] = key.
__device__ __forceinline__ uint32_t rank_of(const uint64_t* key, uint32_t n, uint64_t mine)
{
    uint32_t r = 0;
    for (uint32_t i = 0; i < n; ++i) r += key[i] > mine ? 1u : 0u;
    return r;
}

template <class T>
__global__ __launch_bounds__(BP_NT) void bs_pick(BeamArgs a, const uint32_t* __restrict__ gmax)
{
    using G = Group<T>;
    constexpr uint32_t WAVES = BP_NT / 64;
    __shared__ uint64_t s_key[BP_CAP];
    __shared__ uint64_t s_set[BP_SETS];
    __shared__ uint32_t s_list[BP_NT];
    __shared__ uint32_t s_scan[WAVES];
    __shared__ uint32_t s_n;
    __shared__ uint64_t s_thr;
    const uint32_t t = threadIdx.x, lane = __lane_id(), wave = t >> 6, b = blockIdx.x;
    const uint32_t n_groups = a.beams * a.n_groups;
    const uint32_t* gm = gmax + static_cast<uint64_t>(b) * n_groups;

    // A lower bound of the k-th total: the k-th largest of the sets' maxima.
    for (uint32_t i = t; i < BP_SETS; i += BP_NT) s_set[i] = 0;
    if (t == 0) {
        s_n = 0;
        s_thr = 1;  // any candidate
    }
    __syncthreads();
    uint32_t best = 0;
    for (uint32_t i = t; i < n_groups; i += BP_NT) best = max(best, gm[i]);
    // one set is four threads' groups; the set's place makes the keys distinct
    best = max(best, static_cast<uint32_t>(__shfl_xor(static_cast<int>(best), 1, 64)));
    best = max(best, static_cast<uint32_t>(__shfl_xor(static_cast<int>(best), 2, 64)));
    if ((t & 3u) == 0) s_set[t >> 2] = (static_cast<uint64_t>(best) << 32) | (BP_SETS - (t >> 2));
    __syncthreads();
    if (t < BP_SETS) {
        const uint64_t mine = s_set[t];
        if (rank_of(s_set, BP_SETS, mine) + 1 == a.k && (mine >> 32)) s_thr = (mine >> 32) << 32;
    }
    __syncthreads();

    for (uint32_t g0 = 0; g0 < n_groups; g0 += BP_NT) {
        // the groups that can hold one of the k: in order, so that of equal totals the first are met first
        const uint32_t gi = g0 + t;
        bool in = false;
        if (gi < n_groups) {
            const uint32_t w = gi / a.n_groups, g = gi % a.n_groups;
            // no token of the group is placed before this one
            const uint32_t place = w * a.vocab + (g ? g * G::SIZE : 0u);
            in = gm[gi] != 0 && ((static_cast<uint64_t>(gm[gi]) << 32) | static_cast<uint32_t>(~place)) >= s_thr;
        }
        uint32_t listed;
        const uint32_t at = block_flag_rank<BP_NT>(in, s_scan, listed);
        if (in) s_list[at] = gi;
        __syncthreads();
        for (uint32_t l0 = 0; l0 < listed; l0 += WAVES) {
            const uint64_t thr = s_thr;
            uint64_t key[G::PER * G::UNROLL + 1];
            uint32_t mine = 0;
#pragma unroll
            for (uint32_t i = 0; i <= G::PER * G::UNROLL; ++i) key[i] = 0;
            if (l0 + wave < listed) {
                const uint32_t id = s_list[l0 + wave], w = id / a.n_groups, g = id % a.n_groups;
                const Row<T> row(a, b, w);
                const uint32_t first = w * a.vocab;
                if (g == 0) {
                    const uint32_t o = head_order(a, row, lane);
                    const uint64_t x = (static_cast<uint64_t>(o) << 32) | static_cast<uint32_t>(~(first + lane));
                    if (o && x >= thr) {
                        key[G::PER * G::UNROLL] = x;
                        ++mine;
                    }
                }
#pragma unroll
                for (uint32_t u = 0; u < G::UNROLL; ++u) {
                    const uint32_t v = row.head + g * G::SIZE + (u * 64 + lane) * G::PER;
                    uint32_t o[G::PER];
                    load_orders(a, row, v, o);
#pragma unroll
                    for (uint32_t i = 0; i < G::PER; ++i) {
                        const uint64_t x = (static_cast<uint64_t>(o[i]) << 32) | static_cast<uint32_t>(~(first + v + i));
                        if (o[i] && x >= thr) {
                            key[u * G::PER + i] = x;
                            ++mine;
                        }
                    }
                }
            }
            uint32_t more;
            uint32_t to = block_excl_scan<BP_NT>(mine, s_scan, more);
            const uint32_t held = s_n;  // the scan's barriers order it after the last round's update
            if (held + more <= BP_CAP) {
                to += held;
#pragma unroll
                for (uint32_t i = 0; i <= G::PER * G::UNROLL; ++i)
                    if (key[i]) s_key[to++] = key[i];
                __syncthreads();
                if (t == 0) s_n = held + more;
            } else {
                // too many at once: a token of each lane at a time, the best k kept in between
#pragma unroll
                for (uint32_t i = 0; i <= G::PER * G::UNROLL; ++i) {
                    __syncthreads();
                    uint32_t n = s_n;
                    if (n + BP_NT > BP_CAP) {
                        sort_keys(s_key, n);
                        n = min(n, a.k);
                        __syncthreads();
                        if (t == 0) {
                            s_n = n;
                            if (n == a.k) s_thr = max(s_thr, s_key[n - 1]);
                        }
                        __syncthreads();
                    }
                    uint32_t here;
                    const bool push = key[i] && key[i] >= s_thr;
                    const uint32_t slot = block_flag_rank<BP_NT>(push, s_scan, here);
                    if (push) s_key[n + slot] = key[i];
                    __syncthreads();
                    if (t == 0) s_n = n + here;
                }
            }
            __syncthreads();
        }
        __syncthreads();
    }

    uint32_t n = s_n;
    if (n > BP_SETS) {
        sort_keys(s_key, n);
        n = min(n, a.k);
    }
    const uint64_t out = static_cast<uint64_t>(b) * a.k;
    if (t < n) {
        const uint64_t mine = s_key[t];
        const uint32_t r = rank_of(s_key, n, mine);
        if (r < a.k) {
            const uint32_t place = ~static_cast<uint32_t>(mine), w = place / a.vocab, v = place % a.vocab;
            const Row<T> row(a, b, w);
            a.out_scores[out + r] = total_of(a, to_f32(row.p[v]), row.cum, row.lse);
            a.out_tokens[out + r] = static_cast<int32_t>(v);
            a.out_parents[out + r] = static_cast<int32_t>(w);
        }
    }
    for (uint32_t r = n + t; r < a.k; r += BP_NT) {
        a.out_scores[out + r] = -__builtin_inff();
        a.out_tokens[out + r] = -1;
        a.out_parents[out + r] = -1;
    }
}

// ---- reorder ---------------------------------------------------------------------
constexpr int BR_NT = 256;
constexpr uint32_t BR_PER = 4;

struct ReorderArgs {
    const char* src;
    char* dst;
    const int32_t* parents;
    const int32_t* len;
    uint32_t beams_in, beams_out;
    uint64_t row_bytes, unit_bytes, src_stride, dst_stride;
};

template <class U>
__global__ __launch_bounds__(BR_NT) void br_move(ReorderArgs a)
{
    const uint32_t row = blockIdx.y;
    const int32_t parent = a.parents[row];
    if (parent < 0 || static_cast<uint32_t>(parent) >= a.beams_in) return;
    const uint64_t from = static_cast<uint64_t>(row / a.beams_out) * a.beams_in + static_cast<uint32_t>(parent);
    uint64_t bytes = a.row_bytes;
    if (a.len) bytes = min(bytes, static_cast<uint64_t>(max(a.len[from], 0)) * a.unit_bytes);
    const char* src = a.src + from * a.src_stride;
    char* dst = a.dst + row * a.dst_stride;
    const uint64_t first = (static_cast<uint64_t>(blockIdx.x) * BR_PER * BR_NT + threadIdx.x) * sizeof(U);
    U x[BR_PER];
#pragma unroll
    for (uint32_t j = 0; j < BR_PER; ++j)
        if (first + (j * BR_NT + 1) * sizeof(U) <= bytes) x[j] = *reinterpret_cast<const U*>(src + first + j * BR_NT * sizeof(U));
#pragma unroll
    for (uint32_t j = 0; j < BR_PER; ++j)
        if (first + (j * BR_NT + 1) * sizeof(U) <= bytes) *reinterpret_cast<U*>(dst + first + j * BR_NT * sizeof(U)) = x[j];
}

template <class T>
int launch_select(const BeamArgs& a, uint32_t* gmax, hipStream_t s)
{
    const uint64_t groups = static_cast<uint64_t>(a.batch) * a.beams * a.n_groups;
    {
        CR_TIMED("bs_scan", s);
        bs_scan<T><<<static_cast<unsigned>((groups + BS_NT / 64 - 1) / (BS_NT / 64)), BS_NT, 0, s>>>(a, gmax);
    }
    CR_TIMED("bs_pick", s);
    bs_pick<T><<<a.batch, BP_NT, 0, s>>>(a, gmax);
    CR_LAUNCH_CHECK();
    return CR_OK;
}

template <class U>
int launch_reorder(const ReorderArgs& a, uint32_t rows, hipStream_t s)
{
    const uint64_t chunk = sizeof(U) * BR_PER * BR_NT;
    const uint64_t gx = (a.row_bytes + chunk - 1) / chunk;
    if (gx >> 31) {
        set_error("cr_beam_reorder: rows of %llu bytes are too long", static_cast<unsigned long long>(a.row_bytes));
        return CR_ERR_UNSUPPORTED;
    }
    CR_TIMED("br_move", s);
    const uint32_t most = 65535u / a.beams_out * a.beams_out;  // whole answers, within the grid's second extent
    for (uint32_t r = 0, n; r < rows; r += n) {
        n = std::min(rows - r, most);
        const uint64_t from = static_cast<uint64_t>(r / a.beams_out) * a.beams_in;
        ReorderArgs p = a;
        p.parents += r;
        p.dst += r * a.dst_stride;
        p.src += from * a.src_stride;
        if (p.len) p.len += from;
        br_move<U><<<dim3(static_cast<unsigned>(gx), n), BR_NT, 0, s>>>(p);
    }
    CR_LAUNCH_CHECK();
    return CR_OK;
}

}  // namespace

}  // namespace crimpl

using namespace crimpl;

extern "C" int cr_beam_select(const void* d_scores, uint32_t dtype, uint32_t batch, uint32_t beams, uint32_t vocab,
                              uint64_t batch_stride, uint64_t beam_stride, const float* d_cum, const float* d_lse,
                              const cr_gpu_roaring* allowed, const uint32_t* d_allowed_bits, uint64_t bits_stride,
                              uint32_t k, float* d_out_scores, int32_t* d_out_tokens, int32_t* d_out_parents,
                              cr_stream_t stream)
{
    if (batch == 0 || k == 0) return CR_OK;
    if (!d_scores || !d_cum || beams == 0 || vocab == 0 || dtype > CR_BF16 || !d_out_scores || !d_out_tokens ||
        !d_out_parents || (allowed && d_allowed_bits) || (beams > 1 && beam_stride < vocab) ||
        reinterpret_cast<uintptr_t>(d_scores) % (dtype == CR_F32 ? 4 : 2)) {
        set_error("cr_beam_select: invalid argument");
        return CR_ERR_INVALID;
    }
    if (k > BS_KMAX || (static_cast<uint64_t>(beams) * vocab) >> 31 || batch >> 20) {
        set_error("cr_beam_select: supported up to k %u, 2^31 - 1 continuations of an answer and 2^20 - 1 answers (k %u)",
                  BS_KMAX, k);
        return CR_ERR_UNSUPPORTED;
    }
    hipStream_t s = as_stream(stream);
    BeamArgs a{};
    a.x = d_scores;
    a.batch_stride = batch_stride;
    a.beam_stride = beam_stride;
    a.batch = batch;
    a.beams = beams;
    a.vocab = vocab;
    a.cum = d_cum;
    a.lse = d_lse;
    a.bits = d_allowed_bits;
    a.bits_stride = bits_stride;
    a.k = k;
    a.out_scores = d_out_scores;
    a.out_tokens = d_out_tokens;
    a.out_parents = d_out_parents;
    const uint32_t size = dtype == CR_F32 ? Group<float>::SIZE : Group<BF16>::SIZE;
    a.n_groups = (vocab + size - 1) / size;
    const uint64_t groups = static_cast<uint64_t>(batch) * beams * a.n_groups;
    if (groups >> 32) {
        set_error("cr_beam_select: too many scores for one call");
        return CR_ERR_UNSUPPORTED;
    }
    const uint32_t n_words = (vocab + 31) / 32;
    Carver cv;
    const size_t o_max = cv.add(groups * 4);
    const size_t o_bits = cv.add(allowed ? n_words * 4ull : 0);
    Scratch sc;
    CR_RET(sc.alloc(cv.total, s));
    if (allowed) {
        CR_RET(cr_decompress_to_bitset(allowed, sc.at<uint32_t>(o_bits), n_words, stream));
        a.bits = sc.at<uint32_t>(o_bits);
        a.bits_stride = 0;
    }
    if (dtype == CR_F32) return launch_select<float>(a, sc.at<uint32_t>(o_max), s);
    if (dtype == CR_F16) return launch_select<F16>(a, sc.at<uint32_t>(o_max), s);
    return launch_select<BF16>(a, sc.at<uint32_t>(o_max), s);
}

extern "C" int cr_beam_reorder(const void* d_src, const int32_t* d_parents, uint32_t batch, uint32_t beams_in,
                               uint32_t beams_out, uint64_t row_bytes, uint64_t src_stride, uint64_t dst_stride,
                               const int32_t* d_len, uint64_t unit_bytes, void* d_dst, cr_stream_t stream)
{
    const uint64_t rows = static_cast<uint64_t>(batch) * beams_out;
    if (rows == 0 || row_bytes == 0) return CR_OK;
    if (!d_src || !d_dst || !d_parents || beams_in == 0 || src_stride < row_bytes || dst_stride < row_bytes ||
        (d_len && unit_bytes == 0)) {
        set_error("cr_beam_reorder: invalid argument");
        return CR_ERR_INVALID;
    }
    if (rows >> 31 || beams_out > 65535) {
        set_error("cr_beam_reorder: supported up to 65535 beams and 2^31 - 1 rows");
        return CR_ERR_UNSUPPORTED;
    }
    const char* s0 = static_cast<const char*>(d_src);
    char* t0 = static_cast<char*>(d_dst);
    const uint64_t src_end = static_cast<uint64_t>(batch) * beams_in * src_stride;
    if (s0 < t0 + rows * dst_stride && t0 < s0 + src_end) {
        set_error("cr_beam_reorder: the states are reordered into another buffer");
        return CR_ERR_INVALID;
    }
    ReorderArgs a{s0, t0, d_parents, d_len, beams_in, beams_out, row_bytes, d_len ? unit_bytes : 1, src_stride, dst_stride};
    const uint64_t all = reinterpret_cast<uintptr_t>(d_src) | reinterpret_cast<uintptr_t>(d_dst) | row_bytes |
                         src_stride | dst_stride | (d_len ? unit_bytes : 0);
    hipStream_t s = as_stream(stream);
    if (all % 16 == 0) return launch_reorder<uint4>(a, static_cast<uint32_t>(rows), s);
    if (all % 4 == 0) return launch_reorder<uint32_t>(a, static_cast<uint32_t>(rows), s);
    return launch_reorder<uint8_t>(a, static_cast<uint32_t>(rows), s);
}

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
//   2. bs_pick, a workgroup per answer: the k-th largest of disjoint sets' maxima
//      bounds the k-th total from below; the groups that reach it (about
//      k of them) are read again and their totals at or above it ranked.
// The scores pass by once; what is read again is k groups of an answer.
#include <algorithm>

#include "internal.hpp"

namespace crimpl {

namespace {

constexpr int BS_NT = 256;        // bs_scan: four waves
constexpr uint32_t BP_CAP = 2048;  // candidates held
constexpr uint32_t BP_GROUPS = 1024;  // groups that a pass over them lists
constexpr uint32_t BS_KMAX = 256;

// Sets of allowed tokens: flat words, or the containers of a bitmap that has a
// bitmap container for each key (in key order, so that a key is its own index).
struct Allowed {
    const uint32_t* words;    // nullptr: every token is allowed
    const uint32_t* offsets;  // the containers' byte offsets, or nullptr: flat
    uint64_t stride;          // between rows
    uint32_t flip;            // all bits set where the containers hold the complement
};

struct BeamArgs {
    const void* x;
    uint64_t batch_stride, beam_stride;
    uint32_t batch, beams, vocab;
    const float* cum;
    const float* lse;
    Allowed allowed;
    uint32_t k;
    uint32_t n_groups;  // of a beam
    uint32_t parts, per_wave;  // workgroups that scan a beam, groups a wave of theirs takes
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
    static constexpr uint32_t UNROLL = sizeof(T) == 4 ? 4 : 2;
    static constexpr uint32_t SIZE = 64 * PER * UNROLL;
};

// Whole numbers in the order of the totals; 0 for what is no candidate.
__device__ __forceinline__ uint32_t order_of(float total)
{
    if (!(total > -__builtin_inff())) return 0u;
    const uint32_t b = __float_as_uint(total + 0.0f);  // -0 counts as +0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float total_from(uint32_t order)
{
    return __uint_as_float(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);
}

// Lane `lane`'s value.
__device__ __forceinline__ uint32_t lane_word(uint32_t x, uint32_t lane)
{
    return static_cast<uint32_t>(__shfl(static_cast<int>(x), static_cast<int>(lane), 64));
}

// A beam's row.  Tokens are read 16 bytes at a time from the row's first
// boundary on; the few before it go with the first group and those behind the
// last whole piece with the group they lie in, one by one.
template <class T>
struct Row {
    static constexpr uint32_t PER = Group<T>::PER, UNROLL = Group<T>::UNROLL, SIZE = Group<T>::SIZE;
    const T* p;
    const uint32_t* words;
    uint32_t head, pieces, vocab;
    float cum, lse;
    bool has_lse;
    __device__ __forceinline__ Row(const BeamArgs& a, uint32_t b, uint32_t w)
    {
        const uint64_t row = static_cast<uint64_t>(b) * a.beams + w;
        p = static_cast<const T*>(a.x) + b * a.batch_stride + w * a.beam_stride;
        vocab = a.vocab;
        const uint32_t past = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
        head = min(vocab, ((16u - past) & 15u) / static_cast<uint32_t>(sizeof(T)));
        pieces = (vocab - head) / PER;
        words = a.allowed.words ? a.allowed.words + row * a.allowed.stride : nullptr;
        cum = a.cum[row];
        has_lse = a.lse != nullptr;
        lse = has_lse ? a.lse[row] : 0.0f;
    }
    __device__ __forceinline__ float total(float x) const { return has_lse ? cum + (x - lse) : cum + x; }
    __device__ __forceinline__ uint32_t first(uint32_t g, uint32_t u) const
    {
        return (g * UNROLL + u) * 64u + __lane_id();
    }

    // The lane's pieces of group g; lanes past the last piece read it again.
    __device__ __forceinline__ void load(uint32_t g, cr_v4u (&x)[UNROLL]) const
    {
#pragma unroll
        for (uint32_t u = 0; u < UNROLL; ++u)
            x[u] = __builtin_nontemporal_load(reinterpret_cast<const cr_v4u*>(p + head) + min(first(g, u), pieces - 1));
    }
    // Lane l receives the set's word l of those that cover group g.  `at`: lane
    // c's is container c's first word.
    __device__ __forceinline__ uint32_t load_words(const Allowed& s, uint32_t at, uint32_t g) const
    {
        const uint32_t w = min((head + g * SIZE) / 32u + __lane_id(), (vocab - 1u) / 32u);
        if (!s.offsets) return words[w];
        return words[lane_word(at, w / 2048u) + w % 2048u] ^ s.flip;
    }
    // Which tokens of the lane's pieces there are and may follow.
    __device__ __forceinline__ void masks(uint32_t word, uint32_t g, uint32_t (&on)[UNROLL]) const
    {
#pragma unroll
        for (uint32_t u = 0; u < UNROLL; ++u) {
            const uint32_t all = first(g, u) < pieces ? (1u << PER) - 1u : 0u;
            if (words) {
                const uint32_t bit = (head + g * SIZE) % 32u + (u * 64u + __lane_id()) * PER;
                on[u] = all & __builtin_amdgcn_alignbit(lane_word(word, bit / 32u + 1u), lane_word(word, bit / 32u),
                                                        bit % 32u);
            } else {
                on[u] = all;
            }
        }
    }
    static __device__ __forceinline__ T value(const cr_v4u& x, uint32_t i)
    {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, static_cast<uint32_t>(x[i]));
        else return __builtin_bit_cast(T, static_cast<uint16_t>(x[i / 2] >> (i % 2 * 16u)));
    }
    // The lane's token of group g beside the pieces, or `vocab`.
    __device__ __forceinline__ uint32_t single(const Allowed& s, uint32_t g) const
    {
        const uint32_t lane = __lane_id(), tail = head + pieces * PER;
        uint32_t v = vocab;
        if (g == 0 && lane < head) v = lane;
        if (g == pieces * PER / SIZE && lane >= 32u) v = min(vocab, tail + lane - 32u);
        if (v < vocab && words) {
            const uint32_t w = v / 32u;
            const uint32_t at = s.offsets ? s.offsets[w / 2048u] / 4u + w % 2048u : w;
            const uint32_t bits = words[at] ^ (s.offsets ? s.flip : 0u);
            if (!((bits >> (v % 32u)) & 1u)) v = vocab;
        }
        return v;
    }
    __device__ __forceinline__ bool has_singles(uint32_t g) const { return g == 0 || g == pieces * PER / SIZE; }
};

__device__ __forceinline__ uint32_t container_starts(const Allowed& s, uint32_t vocab)
{
    return s.offsets ? s.offsets[min(__lane_id(), (vocab - 1u) / 65536u)] / 4u : 0u;
}

// The largest of the wave's values, in every lane (no value is NaN).
__device__ __forceinline__ float wave_max(float v)
{
    auto step = [](float x, int y) { return fmaxf(x, __int_as_float(y)); };
    const int low = __float_as_int(-__builtin_inff());
    v = step(v, __builtin_amdgcn_update_dpp(low, __float_as_int(v), 0x111, 0xF, 0xF, false));
    v = step(v, __builtin_amdgcn_update_dpp(low, __float_as_int(v), 0x112, 0xF, 0xF, false));
    v = step(v, __builtin_amdgcn_update_dpp(low, __float_as_int(v), 0x114, 0xF, 0xF, false));
    v = step(v, __builtin_amdgcn_update_dpp(low, __float_as_int(v), 0x118, 0xF, 0xF, false));
    v = step(v, __builtin_amdgcn_update_dpp(low, __float_as_int(v), 0x142, 0xA, 0xF, false));
    v = step(v, __builtin_amdgcn_update_dpp(low, __float_as_int(v), 0x143, 0xC, 0xF, false));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Totals rise with the scores (each rounding keeps their order), so that a
// group's largest total is its largest score's: one comparison a token, and the
// sum once a group.  Bound by reading the scores: 102 MB of bf16 in 21 us, 4.9
// TB/s (with a dependent load or a branch between a wave's loads 30 to 41).
// SPARSE: scores are read only where a token of theirs is allowed, once the masks
// are there; else both are on their way together.
template <class T, bool SPARSE>
__global__ __launch_bounds__(BS_NT) void bs_scan(BeamArgs a, uint32_t* __restrict__ gmax)
{
    using R = Row<T>;
    const uint32_t lane = __lane_id(), r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const R row(a, r / a.beams, r % a.beams);
    const uint32_t at = container_starts(a.allowed, a.vocab);
    const uint32_t g0 = (part * (BS_NT / 64) + (threadIdx.x >> 6)) * a.per_wave;
    for (uint32_t g = g0; g < min(a.n_groups, g0 + a.per_wave); ++g) {
        float best = -__builtin_inff();
        if (row.pieces) {
            uint32_t on[R::UNROLL], word = 0;
            cr_v4u x[R::UNROLL];
            if (!SPARSE) row.load(g, x);
            if (row.words) word = row.load_words(a.allowed, at, g);
            row.masks(word, g, on);
            if (SPARSE) {
                uint32_t any = 0;
#pragma unroll
                for (uint32_t u = 0; u < R::UNROLL; ++u) any |= on[u];
                if (any) row.load(g, x);
            }
#pragma unroll
            for (uint32_t u = 0; u < R::UNROLL; ++u)
#pragma unroll
                for (uint32_t i = 0; i < R::PER; ++i) {
                    const float y = to_f32(R::value(x[u], i));
                    best = ((on[u] >> i) & 1u) && y > best ? y : best;  // NaN is not larger
                }
        }
        if (row.has_singles(g)) {
            const uint32_t v = row.single(a.allowed, g);
            if (v < a.vocab) {
                const float y = to_f32(row.p[v]);
                best = y > best ? y : best;
            }
        }
        best = wave_max(best);
        if (lane == 0) gmax[static_cast<uint64_t>(r) * a.n_groups + g] = order_of(row.total(best));
    }
}

// Sorts the first n of `key` (n <= BP_CAP) in descending order.
template <uint32_t NT>
__device__ __forceinline__ void sort_keys(uint64_t* key, uint32_t n)
{
    uint32_t p = 1;
    while (p < n) p <<= 1;
    for (uint32_t i = n + threadIdx.x; i < p; i += NT) key[i] = 0;
    __syncthreads();
    for (uint32_t size = 2; size <= p; size <<= 1) {
        for (uint32_t step = size >> 1; step > 0; step >>= 1) {
            for (uint32_t i = threadIdx.x; i < p / 2; i += NT) {
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
#pragma unroll 8
    for (uint32_t i = 0; i < n; ++i) r += key[i] > mine ? 1u : 0u;
    return r;
}

// The largest score of the lane's allowed tokens of group g.
template <class T>
__device__ __forceinline__ float lane_best(const Row<T>& row, const Allowed& allowed, uint32_t at, uint32_t g)
{
    using R = Row<T>;
    float best = -__builtin_inff();
    if (row.pieces) {
        uint32_t on[R::UNROLL], word = 0;
        cr_v4u x[R::UNROLL];
        row.load(g, x);
        if (row.words) word = row.load_words(allowed, at, g);
        row.masks(word, g, on);
#pragma unroll
        for (uint32_t u = 0; u < R::UNROLL; ++u)
#pragma unroll
            for (uint32_t i = 0; i < R::PER; ++i) {
                const float y = to_f32(R::value(x[u], i));
                best = ((on[u] >> i) & 1u) && y > best ? y : best;
            }
    }
    if (row.has_singles(g)) {
        const uint32_t v = row.single(allowed, g);
        if (v < row.vocab) {
            const float y = to_f32(row.p[v]);
            best = y > best ? y : best;
        }
    }
    return best;
}

// A workgroup per answer, bound by the latency of its few dependent reads.  NT
// threads: 512 for few winners (k = 8 of 64 x 8 x 100003: 10.1 us, with 256 12.5,
// with 1024 10.6), 1024 for many, whose groups then take fewer rounds.  With the
// lanes' maxima where groups are few, 10 x 8 x 1507, k = 8, takes 19 us in all
// instead of 50, 4 x 4 x 30000, k = 64, 37 instead of 134.
template <class T, uint32_t NT>
__global__ __launch_bounds__(NT) void bs_pick(BeamArgs a, const uint32_t* __restrict__ gmax)
{
    using R = Row<T>;
    constexpr uint32_t WAVES = NT / 64, SETS = NT / 4, MINE = R::PER * R::UNROLL;
    constexpr uint32_t OWN = BP_GROUPS / NT;  // groups a thread looks at in a pass over them
    __shared__ uint64_t s_key[BP_CAP];
    __shared__ uint64_t s_set[SETS];
    __shared__ uint32_t s_list[BP_GROUPS];
    __shared__ uint32_t s_best[NT];
    __shared__ uint32_t s_scan[WAVES];
    __shared__ uint32_t s_n;
    __shared__ uint64_t s_thr;
    const uint32_t t = threadIdx.x, wave = t >> 6, b = blockIdx.x;
    const uint32_t n_groups = a.beams * a.n_groups;
    const uint32_t* gm = gmax + static_cast<uint64_t>(b) * n_groups;
    const uint32_t starts = container_starts(a.allowed, a.vocab);

    // A lower bound of the k-th total: the k-th largest of the sets' maxima.
    if (t == 0) {
        s_n = 0;
        s_thr = 1;  // any candidate
    }
    // `best`: the thread's, of totals that are no other thread's.  Returns how many
    // of the sets, four threads' totals each, have a candidate.
    auto bound = [&](uint32_t best) {
        s_best[t] = best;
        __syncthreads();
        if (t < SETS) {  // the set's place makes the keys distinct
            uint32_t most = s_best[t];
#pragma unroll
            for (uint32_t i = 1; i < 4; ++i) most = max(most, s_best[t + i * SETS]);
            s_set[t] = (static_cast<uint64_t>(most) << 32) | (SETS - t);
        }
        __syncthreads();
        // four threads count what lies above a set, a quarter of the sets each
        const uint64_t mine = s_set[t >> 2];
        uint32_t above = rank_of(s_set + (t & 3u) * (SETS / 4), SETS / 4, mine);
        above += static_cast<uint32_t>(__shfl_xor(static_cast<int>(above), 1, 64));
        above += static_cast<uint32_t>(__shfl_xor(static_cast<int>(above), 2, 64));
        const bool filled = (t & 3u) == 0 && (mine >> 32) != 0;
        if (filled && above + 1 == a.k) s_thr = max(s_thr, (mine >> 32) << 32);
        uint32_t all;
        block_excl_scan<NT>(filled ? 1u : 0u, s_scan, all);
        return all;
    };
    uint32_t best = 0;
    for (uint32_t i = t; i < n_groups; i += NT) best = max(best, gm[i]);
    // Few groups bound the answer badly (8 beams of 1507 tokens, k = 8: 16 maxima):
    // their lanes' own maxima are taken instead, below.
    const bool weak = bound(best) < min(2 * a.k, SETS);

    for (uint32_t g0 = 0; g0 < n_groups; g0 += BP_GROUPS) {
        // the groups that can hold one of the k: in order, so that of equal totals the first are met first
        uint32_t in = 0;
#pragma unroll
        for (uint32_t j = 0; j < OWN; ++j) {
            const uint32_t gi = g0 + t * OWN + j, most = gi < n_groups ? gm[gi] : 0u;
            const uint32_t w = gi / a.n_groups, g = gi % a.n_groups;
            // no token of the group is placed before this one
            const uint32_t place = w * a.vocab + (g ? g * R::SIZE : 0u);
            const uint64_t key = (static_cast<uint64_t>(most) << 32) | static_cast<uint32_t>(~place);
            if (most != 0 && key >= s_thr) in |= 1u << j;
        }
        uint32_t listed;
        uint32_t at = block_excl_scan<NT>(__popc(in), s_scan, listed);
#pragma unroll
        for (uint32_t j = 0; j < OWN; ++j)
            if ((in >> j) & 1u) s_list[at++] = g0 + t * OWN + j;
        __syncthreads();
        if (weak && g0 == 0 && listed > 1) {
            uint32_t most = 0;
            for (uint32_t l = wave; l < listed; l += WAVES) {
                const uint32_t id = s_list[l], g = id % a.n_groups;
                const R row(a, b, id / a.n_groups);
                most = max(most, order_of(row.total(lane_best(row, a.allowed, starts, g))));
            }
            bound(most);
        }
        for (uint32_t l0 = 0; l0 < listed; l0 += WAVES) {
            const uint64_t thr = s_thr;
            uint64_t key[MINE + 1];
            uint32_t mine = 0;
#pragma unroll
            for (uint32_t i = 0; i <= MINE; ++i) key[i] = 0;
            if (l0 + wave < listed) {
                const uint32_t id = s_list[l0 + wave], w = id / a.n_groups, g = id % a.n_groups;
                const R row(a, b, w);
                auto take = [&](uint32_t slot, uint32_t v, T y) {
                    const uint32_t o = order_of(row.total(to_f32(y)));
                    const uint64_t x = (static_cast<uint64_t>(o) << 32) | static_cast<uint32_t>(~(w * a.vocab + v));
                    if (o && x >= thr) {
                        key[slot] = x;
                        ++mine;
                    }
                };
                if (row.pieces) {
                    uint32_t on[R::UNROLL], word = 0;
                    cr_v4u x[R::UNROLL];
                    row.load(g, x);
                    if (row.words) word = row.load_words(a.allowed, starts, g);
                    row.masks(word, g, on);
#pragma unroll
                    for (uint32_t u = 0; u < R::UNROLL; ++u)
#pragma unroll
                        for (uint32_t i = 0; i < R::PER; ++i)
                            if ((on[u] >> i) & 1u)
                                take(u * R::PER + i, row.head + row.first(g, u) * R::PER + i, R::value(x[u], i));
                }
                if (row.has_singles(g)) {
                    const uint32_t v = row.single(a.allowed, g);
                    if (v < a.vocab) take(MINE, v, row.p[v]);
                }
            }
            uint32_t more;
            uint32_t to = block_excl_scan<NT>(mine, s_scan, more);
            const uint32_t held = s_n;  // the scan's barriers order it after the last round's update
            if (held + more <= BP_CAP) {
                to += held;
#pragma unroll
                for (uint32_t i = 0; i <= MINE; ++i)
                    if (key[i]) s_key[to++] = key[i];
                __syncthreads();
                if (t == 0) s_n = held + more;
            } else {
                // too many at once: a token of each lane at a time, the best k kept in between
#pragma unroll
                for (uint32_t i = 0; i <= MINE; ++i) {
                    __syncthreads();
                    uint32_t n = s_n;
                    if (n + NT > BP_CAP) {
                        sort_keys<NT>(s_key, n);
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
                    const uint32_t slot = block_flag_rank<NT>(push, s_scan, here);
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
    if (n > NT || n > 256) {
        sort_keys<NT>(s_key, n);
        n = min(n, a.k);
    }
    const uint64_t out = static_cast<uint64_t>(b) * a.k;
    if (t < n) {
        const uint64_t mine = s_key[t];
        const uint32_t r = rank_of(s_key, n, mine);
        if (r < a.k) {
            const uint32_t place = ~static_cast<uint32_t>(mine);
            a.out_scores[out + r] = total_from(static_cast<uint32_t>(mine >> 32));
            a.out_tokens[out + r] = static_cast<int32_t>(place % a.vocab);
            a.out_parents[out + r] = static_cast<int32_t>(place / a.vocab);
        }
    }
    for (uint32_t r = n + t; r < a.k; r += NT) {
        a.out_scores[out + r] = -__builtin_inff();
        a.out_tokens[out + r] = -1;
        a.out_parents[out + r] = -1;
    }
}

// ---- reorder ---------------------------------------------------------------------
// Bound by memory: a thread moves four pieces, past the caches (64 x 8 rows of 64
// KiB, half of them in use: 9.5 us, 3.5 TB/s read and written with the launch;
// through the caches 20).
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
        if (first + (j * BR_NT + 1) * sizeof(U) <= bytes)
            x[j] = __builtin_nontemporal_load(reinterpret_cast<const U*>(src + first + j * BR_NT * sizeof(U)));
#pragma unroll
    for (uint32_t j = 0; j < BR_PER; ++j)
        if (first + (j * BR_NT + 1) * sizeof(U) <= bytes)
            __builtin_nontemporal_store(x[j], reinterpret_cast<U*>(dst + first + j * BR_NT * sizeof(U)));
}

template <class T>
int launch_select(const BeamArgs& a, bool sparse, uint32_t* gmax, hipStream_t s)
{
    {
        CR_TIMED("bs_scan", s);
        const uint32_t grid = a.batch * a.beams * a.parts;
        if (sparse)
            bs_scan<T, true><<<grid, BS_NT, 0, s>>>(a, gmax);
        else
            bs_scan<T, false><<<grid, BS_NT, 0, s>>>(a, gmax);
    }
    CR_TIMED("bs_pick", s);
    if (a.k <= 32)
        bs_pick<T, 512><<<a.batch, 512, 0, s>>>(a, gmax);
    else
        bs_pick<T, 1024><<<a.batch, 1024, 0, s>>>(a, gmax);
    CR_LAUNCH_CHECK();
    return CR_OK;
}

template <class U>
int launch_reorder(const ReorderArgs& a, uint32_t rows, hipStream_t s)
{
    const uint64_t chunk = sizeof(U) * BR_PER * BR_NT;
    const uint64_t gx = (a.row_bytes + chunk - 1) / chunk;
    if (gx >> 24) {  // a launch holds fewer than 2^32 threads
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
        set_error("cr_beam_select: supported up to k %u, 2^31 - 1 continuations of an answer and 2^20 - 1 answers "
                  "(k %u)", BS_KMAX, k);
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
    a.allowed.words = d_allowed_bits;
    a.allowed.stride = bits_stride;
    a.k = k;
    a.out_scores = d_out_scores;
    a.out_tokens = d_out_tokens;
    a.out_parents = d_out_parents;
    const uint32_t size = dtype == CR_F32 ? Group<float>::SIZE : Group<BF16>::SIZE;
    a.n_groups = (vocab + size - 1) / size;
    const uint64_t rows = static_cast<uint64_t>(batch) * beams, groups = rows * a.n_groups;
    // A wave takes two groups of large batches, one of small ones (64 x 8 beams of
    // 100003 bf16 scores: one 52 us in all, two 48.9, four 49.3, eight 50.2).
    a.per_wave = static_cast<uint32_t>(std::min<uint64_t>(2, std::max<uint64_t>(1, groups / (16ull * num_cus()))));
    a.parts = (a.n_groups + a.per_wave * (BS_NT / 64) - 1) / (a.per_wave * (BS_NT / 64));
    if (groups >> 32 || (rows * a.parts) >> 24) {  // a launch holds fewer than 2^32 threads
        set_error("cr_beam_select: too many scores for one call");
        return CR_ERR_UNSUPPORTED;
    }
    // Bitmap containers for all keys are read where they lie; other layouts are
    // written out as flat words first.
    const uint32_t n_words = (vocab + 31) / 32;
    const uint32_t keys = (vocab + 65535) / 65536;
    const bool direct = allowed && keys <= 64 && allowed->n_containers == keys && allowed->max_key + 1 == keys &&
                        allowed->n_bitmap_containers == keys &&
                        (!allowed->negated || allowed->universe_size >= vocab);
    const bool flat = allowed && !direct;
    Carver cv;
    const size_t o_max = cv.add(groups * 4);
    const size_t o_bits = cv.add(flat ? n_words * 4ull : 0);
    Scratch sc;
    CR_RET(sc.alloc(cv.total, s));
    if (direct) {
        a.allowed = {reinterpret_cast<const uint32_t*>(allowed->bitmap_data), allowed->offsets, 0,
                     allowed->negated ? 0xFFFFFFFFu : 0u};
    } else if (flat) {
        CR_RET(cr_decompress_to_bitset(allowed, sc.at<uint32_t>(o_bits), n_words, stream));
        a.allowed.words = sc.at<uint32_t>(o_bits);
    }
    // Few of a cache line's 64 scores are allowed (its recorded cardinality is a
    // hint: it changes what is read, not the answer).
    const bool sparse = allowed && allowed->total_cardinality > 0 && allowed->total_cardinality < vocab / 64;
    if (dtype == CR_F32) return launch_select<float>(a, sparse, sc.at<uint32_t>(o_max), s);
    if (dtype == CR_F16) return launch_select<F16>(a, sparse, sc.at<uint32_t>(o_max), s);
    return launch_select<BF16>(a, sparse, sc.at<uint32_t>(o_max), s);
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
    ReorderArgs a{s0,        t0,        d_parents,              d_len,      beams_in,  beams_out,
                  row_bytes, d_len ? unit_bytes : 1, src_stride, dst_stride};
    const uint64_t all = reinterpret_cast<uintptr_t>(d_src) | reinterpret_cast<uintptr_t>(d_dst) | row_bytes |
                         src_stride | dst_stride | (d_len ? unit_bytes : 0);
    hipStream_t s = as_stream(stream);
    if (all % 16 == 0) return launch_reorder<cr_v4u>(a, static_cast<uint32_t>(rows), s);
    if (all % 4 == 0) return launch_reorder<uint32_t>(a, static_cast<uint32_t>(rows), s);
    return launch_reorder<uint8_t>(a, static_cast<uint32_t>(rows), s);
}

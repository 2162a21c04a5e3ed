// Verification of drafted tokens, for serving language models (no reference
// implementation).
//
// Row i of a request is what the model says after its i-th token, p = softmax(x / T)
// over the allowed tokens, and q what the drafting model said there.  Draft i, token
// d, is accepted while u_i q(d) < p(d); the token behind the accepted ones is drawn
// from max(p - q, 0), or from p where every draft was accepted: the first token at
// which the running sum exceeds u times the whole.  Tokens then follow the model's
// own distribution, whatever was drafted.
//
// Sums and exponentials are in 64 bits: a random number falls between two running
// sums that differ by 1e-5 and less, and which side it falls on is the answer.  That
// makes arithmetic the bound of long rows, not their bytes: some 20 instructions a
// token, nine of them on 64 bits, at 4 to 5 cycles a wave (32 bits: 2.4).  Shares below
// 2^-1000 of a row's largest are none.
//
//   1. dv_sums: every row once, a wave per piece of DV_PIECE tokens: largest score, and
//      the sum of e^((x - largest) / T).
//   2. dv_norms, where requests have many rows: each row's largest score and sum, and
//      whether its draft is accepted.  With fewer, the next launch finds that out.
//   3. dv_rest: the sums of max(p - q, 0), by pieces, of the row where the accepted ones
//      end.  Without a drafting model's scores q is 1 for the drafted token, and the
//      pieces of p do.
//   4. dv_pick: the piece in which the running sum passes the mark, and the token in it.
#include <algorithm>

#include "internal.hpp"
#include "elements.hpp"
#include "set_bits.hpp"

namespace crimpl {

namespace {

constexpr int DV_NT = 256;
constexpr uint32_t DV_WAVES = DV_NT / 64;
constexpr uint32_t DV_UNIT = 8;                  // neighbouring tokens of a lane
constexpr uint32_t DV_STEPS = 4;                 // times
constexpr uint32_t DV_PIECE = 64 * DV_UNIT * DV_STEPS;

// Requests of fewer rows on average are decided where the decision is asked for, four rows at a
// time up to the first draft that is not accepted, which saves a launch (4 drafts of 32000 tokens:
// 17 us, not 19; 128 requests of 3 looked-up ones: 24, not 27).  Where all drafts are accepted, 8
// rows take 17.5 us, not 18.2, but 12 take 18.8, not 17.6.
constexpr uint32_t DV_FOLD = 10;

struct Norm {  // of a row: p(v) = e^((x_v - top) / T) * part
    double part;
    float top;
};

struct RowState {
    Norm p, q;
    uint32_t accepted;  // whether the draft that follows the row is
};

struct Decision {
    uint32_t row, accepted;
    bool rejected;  // the draft that there was
    int32_t token;
    Norm p, q;
};

struct VerifyArgs {
    const void* x;
    const void* draft;  // or nullptr
    uint64_t x_row, draft_row;
    uint32_t n_rows, n_requests, vocab, pieces;
    const int32_t* tokens;
    const int32_t* starts;
    const float* uniform;
    double scale;        // 256 log2(e) / temperature
    double reach;        // scores so far below the largest have no share
    const uint32_t* flat;  // [rows of bits_stride words, or one for all (0)], or nullptr
    uint64_t bits_stride;
    SetBits allowed;
    bool masked;
    int32_t* accepted;
    int32_t* out;
    uint32_t most;         // columns of out
    uint64_t out_stride;
    // [2][n_rows][pieces]: the rows' pieces and the drafts'
    float* top;
    double* mass;
    RowState* state;       // [n_rows], or not needed: the rows' states are worked out where they are asked for
    bool folded;
    double* rest;          // [n_requests][pieces]
    Decision* decided;     // [n_requests], by dv_rest
};

// 2^(i / 256) for i = threadIdx.x: the series of e^y to y^11, y = (i / 256 - 1/2) log(2), which
// leaves 7e-15 of it, times 2^(1/2).
__device__ __forceinline__ double power_of(uint32_t i)
{
    const double y = (static_cast<double>(static_cast<int32_t>(i) - 128) / 256.0) * 0.693147180559945309417;
    double e = 2.505210838544171877505e-8;
    e = fma(e, y, 2.755731922398589065255e-7);
    e = fma(e, y, 2.755731922398589065255e-6);
    e = fma(e, y, 2.480158730158730158730e-5);
    e = fma(e, y, 1.984126984126984126984e-4);
    e = fma(e, y, 1.388888888888888888889e-3);
    e = fma(e, y, 8.333333333333333333333e-3);
    e = fma(e, y, 4.166666666666666666667e-2);
    e = fma(e, y, 1.666666666666666666667e-1);
    e = fma(e, y, 0.5);
    e = fma(e, y, 1.0);
    e = fma(e, y, 1.0);
    return e * 1.41421356237309504880;
}

constexpr uint32_t DV_POWERS = 256;

template <int NT>
__device__ __forceinline__ void make_powers(double* s_pow)
{
#pragma unroll
    for (uint32_t i = 0; i < DV_POWERS; i += NT) s_pow[i + threadIdx.x] = power_of(i + threadIdx.x);
    __syncthreads();
}

// e^((x - top) / T) of a row whose largest score is `top`: 2^(u / 256) with u rounded to a
// whole number n, which is added to an exponent and looked up, and the rest |f| <= 1/2 by
// the series of e^y to y^3, y = f log(2) / 256, which leaves 1.4e-13 of it.  Scores of +inf
// share the mass.
struct Shares {
    double scale, from, least;
    float top;
    __device__ __forceinline__ Shares(const VerifyArgs& a, float largest)
    {
        scale = a.scale;
        top = largest;
        from = static_cast<double>(largest);
        least = -a.reach;
    }
    // How far below a finite largest score x is, which is exact: at low temperatures its factors
    // are far above it.
    __device__ __forceinline__ double below(float x) const { return static_cast<double>(x) - from; }
    // The power and what it is multiplied by, of d from `least` to 0.
    __device__ __forceinline__ void parts(double d, const double* s_pow, double& power, double& more) const
    {
        constexpr double ROUND = 6755399441055744.0;  // 1.5 * 2^52
        const double r = fma(d, scale, ROUND), f = fma(d, scale, ROUND - r);
        const uint32_t n = static_cast<uint32_t>(__double_as_longlong(r));
        const uint64_t b = static_cast<uint64_t>(__double_as_longlong(s_pow[n % DV_POWERS]));
        const uint32_t hi = static_cast<uint32_t>(b >> 32) + (n / DV_POWERS << 20);  // (modulo 2^12: n may be negative)
        power = __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | static_cast<uint32_t>(b)));
        more = fma(f, fma(f, fma(f, 0x1.c6b08d704a0c0p-29, 0x1.ebfbdff82c58fp-19), 0x1.62e42fefa39efp-9), 1.0);
    }
    // Adds a share; those of NaN, -inf and scores below 2^-1000 of the largest as 2^-1000 of
    // it, which no sum notices.
    __device__ __forceinline__ void add(float x, const double* s_pow, double& sum) const
    {
        double power, more;
        parts(fmax(below(x), least), s_pow, power, more);
        sum = fma(power, more, sum);
    }
    // The share itself: of those none.
    __device__ __forceinline__ double finite(float x, const double* s_pow) const
    {
        double power, more;
        const double d = below(x);
        parts(fmax(d, least), s_pow, power, more);
        return d >= least ? power * more : 0.0;
    }
    __device__ __forceinline__ double operator()(float x, const double* s_pow) const
    {
        return top == __builtin_inff() ? (x == top ? 1.0 : 0.0) : finite(x, s_pow);
    }
    // A unit of them, worked out side by side.
    __device__ __forceinline__ void of(const float (&x)[DV_UNIT], const double* s_pow, double (&share)[DV_UNIT]) const
    {
        if (top == __builtin_inff()) {
#pragma unroll
            for (uint32_t e = 0; e < DV_UNIT; ++e) share[e] = x[e] == top ? 1.0 : 0.0;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < DV_UNIT; ++e) share[e] = finite(x[e], s_pow);
        }
    }
    template <uint32_t U>
    __device__ __forceinline__ double sum(const float (&x)[U][DV_UNIT], const double* s_pow) const
    {
        double mass = 0.0, more = 0.0;  // (two chains)
        if (top == __builtin_inff()) {
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
#pragma unroll
                for (uint32_t e = 0; e < DV_UNIT; ++e) mass += x[u][e] == top ? 1.0 : 0.0;
        } else {
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
#pragma unroll
                for (uint32_t e = 0; e < DV_UNIT; e += 2) {
                    add(x[u][e], s_pow, mass);
                    add(x[u][e + 1], s_pow, more);
                }
        }
        return mass + more;
    }
};

// Another lane's value within the rows of 16 lanes, then across them; 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double v)
{
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
    const uint32_t lo = static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(b)), CTRL, ROWS, 0xF, false));
    const uint32_t hi = static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(b >> 32)), CTRL, ROWS, 0xF, false));
    return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo));
}

// Inclusive scan over a wave.
__device__ __forceinline__ double wave_incl_scan_f64(double v)
{
    v += dpp_f64<0x111, 0xF>(v);
    v += dpp_f64<0x112, 0xF>(v);
    v += dpp_f64<0x114, 0xF>(v);
    v += dpp_f64<0x118, 0xF>(v);
    v += dpp_f64<0x142, 0xA>(v);
    v += dpp_f64<0x143, 0xC>(v);
    return v;
}

__device__ __forceinline__ double lane_f64(double v, int lane)
{
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(b)), lane));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(b >> 32)), lane));
    return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo));
}

__device__ __forceinline__ double wave_sum_f64(double v) { return lane_f64(wave_incl_scan_f64(v), 63); }

template <int CTRL, int ROWS>
__device__ __forceinline__ float max_dpp(float v)
{
    const int b = static_cast<int>(__float_as_uint(v));
    return fmaxf(v, __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(b, b, CTRL, ROWS, 0xF, false))));
}

__device__ __forceinline__ float wave_max(float v)
{
    v = max_dpp<0x111, 0xF>(v);
    v = max_dpp<0x112, 0xF>(v);
    v = max_dpp<0x114, 0xF>(v);
    v = max_dpp<0x118, 0xF>(v);
    v = max_dpp<0x142, 0xA>(v);
    v = max_dpp<0x143, 0xC>(v);
    return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(v)), 63)));
}

// The allowed tokens' bits where a piece lies, which is within one container: word w of them is
// (words[w] & keep) ^ flip, and tokens from `end` on may not be used.
struct Mask {
    const uint32_t* words;  // nullptr: every token may be used
    uint32_t keep, flip, end;
    __device__ __forceinline__ Mask(const VerifyArgs& a, uint32_t row, uint32_t first)
    {
        words = nullptr;
        keep = 0xFFFFFFFFu;
        flip = 0u;
        end = a.vocab;
        if (!a.masked) return;
        if (a.flat) {
            words = a.flat + row * a.bits_stride;
        } else if (a.allowed.flat) {
            words = a.allowed.flat;
        } else {
            const uint32_t key = __builtin_amdgcn_readfirstlane(first) / 65536u;
            uint32_t c = a.allowed.key_index[min(key, a.allowed.max_key)];
            if (key > a.allowed.max_key) c = 0xFFFFu;
            keep = c != 0xFFFFu ? 0xFFFFFFFFu : 0u;
            flip = a.allowed.flip;
            end = min(end, a.allowed.end);
            words = reinterpret_cast<const uint32_t*>(a.allowed.bitmaps) + a.allowed.offsets[c != 0xFFFFu ? c : 0u] / 4u -
                    static_cast<int64_t>(key) * 2048;
        }
    }
};

// A lane's tokens of a piece: DV_UNIT neighbours from first + u * 64 * DV_UNIT on, for U values
// of u, as they lie, and which of them are there and may be used.  No load waits for
// another, and none is waited for here.
template <class E, uint32_t U>
struct Tokens {
    typedef typename E::Bits Bits;
    // rows may begin anywhere
    typedef Bits Wide __attribute__((ext_vector_type(DV_UNIT), aligned(sizeof(Bits))));
    static constexpr uint32_t STEP = 64 * DV_UNIT;
    Wide raw[U];
    uint32_t on[U];
    bool all;  // every one is, in the whole wave

    __device__ __forceinline__ void load(const VerifyArgs& a, const Bits* p, const Mask& mask, uint32_t first)
    {
        const bool whole = __builtin_amdgcn_readfirstlane(first) + U * STEP <= a.vocab;  // (the first lane's are the first)
        all = whole && !mask.words;
        if (mask.words) {
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) on[u] = mask.words[min((first + u * STEP) / 32u, (a.vocab - 1) / 32u)];
        }
        if (whole) {
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
                raw[u] = __builtin_nontemporal_load(reinterpret_cast<const Wide*>(p + first + u * STEP));
        } else {
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
#pragma unroll
                for (uint32_t e = 0; e < DV_UNIT; ++e) raw[u][e] = p[min(first + u * STEP + e, a.vocab - 1)];
        }
    }
    // The scores of unit u: -inf for those that are not there or may not be used.
    __device__ __forceinline__ void scores(const Mask& mask, uint32_t first, uint32_t u, float (&x)[DV_UNIT]) const
    {
#pragma unroll
        for (uint32_t e = 0; e < DV_UNIT; ++e) x[e] = E::up(raw[u][e]);
        if (all) return;
        const uint32_t at = first + u * STEP, left = at < mask.end ? mask.end - at : 0u;
        const uint32_t bits = mask.words ? (on[u] & mask.keep) ^ mask.flip : 0xFFFFFFFFu;
        const uint32_t may = (bits >> (first % 32u)) & (left >= DV_UNIT ? 0xFFu : (1u << left) - 1u);
#pragma unroll
        for (uint32_t e = 0; e < DV_UNIT; ++e) {
            const uint32_t keep = static_cast<uint32_t>(static_cast<int32_t>(may << (31u - e)) >> 31);
            x[e] = __uint_as_float((__float_as_uint(x[e]) & keep) | (0xFF800000u & ~keep));
        }
    }
};

// Of a piece's tokens, where few may be used, those alone, by their numbers in LDS, in order: one
// unit a lane.  Exponentials are what a piece costs, and scores that nobody asks for need not be
// read: 64 requests of 4 drafts over 100003 bf16 tokens take 38 us with a fifth of them allowed and
// 27 with a thousandth, 48 to 52 either way where all are read.  Asking first costs where many are
// allowed after all, 55 us and not 52 with 45%, of which a list would make 64.
constexpr uint32_t DV_FEW = 64 * DV_UNIT;

struct Few {
    uint32_t total;
    bool is;  // few enough to be listed

    __device__ __forceinline__ Few(const VerifyArgs& a, const Mask& mask, uint32_t piece, uint16_t* s)
    {
        static_assert(DV_PIECE == 64 * 32, "a word a lane");
        const uint32_t lane = __lane_id(), first = piece * DV_PIECE + lane * 32u;
        const uint32_t left = first < mask.end ? mask.end - first : 0u;
        uint32_t bits = (mask.words[min(first, a.vocab - 1) / 32u] & mask.keep) ^ mask.flip;
        bits &= left >= 32u ? 0xFFFFFFFFu : (1u << left) - 1u;
        const uint32_t n = __popc(bits), upto = wave_incl_scan(n);
        total = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), 63));
        is = total <= DV_FEW;
        if (!is) return;
        for (uint32_t to = upto - n; bits; bits &= bits - 1) s[to++] = static_cast<uint16_t>(lane * 32u + __builtin_ctz(bits));
        wave_lds_fence();
    }
    // Their scores, DV_UNIT a lane, -inf behind the last; p: the piece's.
    template <class E>
    __device__ __forceinline__ void get(const typename E::Bits* p, const uint16_t* s, float (&x)[DV_UNIT]) const
    {
#pragma unroll
        for (uint32_t e = 0; e < DV_UNIT; ++e) {
            const uint32_t i = e * 64 + __lane_id();
            x[e] = i < total ? E::up(p[s[i]]) : -__builtin_inff();
        }
    }
};

__device__ __forceinline__ bool is_allowed(const VerifyArgs& a, uint64_t row, uint32_t token)
{
    if (!a.masked) return true;
    const uint32_t w = token / 32u;
    if (!a.flat && token >= a.allowed.end) return false;  // (a complement's words say nothing behind its universe)
    const uint32_t word = a.flat ? a.flat[row * a.bits_stride + w] : a.allowed.word(w);
    return (word >> (token % 32u)) & 1u;
}

struct RequestRows {
    uint32_t first, drafts;
    bool none;
};

__device__ __forceinline__ RequestRows rows_of(const VerifyArgs& a, uint32_t r)
{
    const int32_t n = static_cast<int32_t>(a.n_rows);
    const int32_t r0 = min(max(a.starts[r], 0), n), r1 = min(max(a.starts[r + 1], r0), n);
    const uint32_t rows = static_cast<uint32_t>(r1 - r0);
    return {static_cast<uint32_t>(r0), rows ? rows - 1 : 0u, rows == 0};
}

// Whether a request ends with this row, after which nothing is drafted: a wave looks at 64
// starts at a time.
__device__ __forceinline__ bool is_last(const VerifyArgs& a, uint32_t row)
{
    const int32_t next = static_cast<int32_t>(row) + 1;
    uint32_t lo = 0;
    for (uint32_t len = a.n_requests + 1; len > 1;) {  // the last start at or before the next row is among these
        const uint32_t step = (len + 63) / 64, i = lo + __lane_id() * step;
        const unsigned long long m = __ballot(__lane_id() * step < len && i <= a.n_requests && a.starts[min(i, a.n_requests)] <= next);
        lo += (max(static_cast<uint32_t>(__popcll(m)), 1u) - 1) * step;
        len = step;
    }
    return a.starts[min(lo, a.n_requests)] == next;
}

// Every row's pieces, a wave each; the drafting model's rows behind the model's.  A
// piece's 32 tokens a lane are asked for at once, and the table of powers is made while they
// come.  63 MB of bf16 scores take 28 us where all are asked for, 19 where a fifth may be
// used; longer loops over several pieces a wave gained nothing.
template <class E, bool MASKED>
__global__ __launch_bounds__(DV_NT) __attribute__((amdgpu_waves_per_eu(6))) void dv_sums(VerifyArgs a)
{
    __shared__ double s_pow[DV_POWERS];
    __shared__ uint16_t s_few[DV_WAVES][MASKED ? DV_FEW : 1];
    const uint32_t lane = __lane_id(), in_group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wave = blockIdx.x * DV_WAVES + in_group;
    const uint32_t at = wave / a.pieces, first = wave % a.pieces * DV_PIECE + lane * DV_UNIT;
    const bool there = at < (a.draft ? 2 : 1) * a.n_rows, drafted = at >= a.n_rows;
    const uint32_t row = drafted ? at - a.n_rows : at;
    const auto* p = static_cast<const typename E::Bits*>(drafted ? a.draft : a.x) +
                    row * (drafted ? a.draft_row : a.x_row);
    const Mask mask(a, there ? row : 0u, first);
    float top = -__builtin_inff();
    double mass = 0.0;
    Tokens<E, DV_STEPS> tokens;
    if constexpr (MASKED) {
        make_powers<DV_NT>(s_pow);
        if (!there || (drafted && is_last(a, row))) return;
        const Few few(a, mask, wave % a.pieces, s_few[in_group]);
        if (few.is) {
            float x[1][DV_UNIT];
            few.get<E>(p + wave % a.pieces * DV_PIECE, s_few[in_group], x[0]);
#pragma unroll
            for (uint32_t e = 0; e < DV_UNIT; ++e) top = fmaxf(top, x[0][e]);
            top = wave_max(top);
            if (top > -__builtin_inff()) mass = wave_sum_f64(Shares(a, top).sum(x, s_pow));
            if (lane == 0) {
                a.top[wave] = top;
                a.mass[wave] = mass;
            }
            return;
        }
        tokens.load(a, p, mask, first);
    } else {
        if (there) tokens.load(a, p, mask, first);
        make_powers<DV_NT>(s_pow);
        if (!there || (drafted && is_last(a, row))) return;
    }
    float x[DV_STEPS][DV_UNIT];
#pragma unroll
    for (uint32_t u = 0; u < DV_STEPS; ++u) {
        tokens.scores(mask, first, u, x[u]);
#pragma unroll
        for (uint32_t e = 0; e < DV_UNIT; ++e) top = fmaxf(top, x[u][e]);
    }
    top = wave_max(top);
    if (top > -__builtin_inff()) mass = wave_sum_f64(Shares(a, top).sum(x, s_pow));
    if (lane == 0) {
        a.top[wave] = top;
        a.mass[wave] = mass;
    }
}

// What the shares of a row are divided by: a wave's work, which joins the pieces in a fixed order.
struct Pieces {
    const float* top;
    const double* mass;
    float top0;  // the lane's first
    double mass0;
    __device__ __forceinline__ Pieces(const VerifyArgs& a, uint32_t at)
    {
        top = a.top + static_cast<uint64_t>(at) * a.pieces;
        mass = a.mass + static_cast<uint64_t>(at) * a.pieces;
        const uint32_t i = min(__lane_id(), a.pieces - 1);
        top0 = top[i];
        mass0 = mass[i];
    }
    __device__ __forceinline__ Norm norm(const VerifyArgs& a, const double* s_pow) const
    {
        float m = top0;
        for (uint32_t i = __lane_id() + 64; i < a.pieces; i += 64) m = fmaxf(m, top[i]);
        m = wave_max(m);
        double sum = 0.0;
        if (m > -__builtin_inff()) {
            const Shares share(a, m);
            if (__lane_id() < a.pieces) sum = mass0 * share(top0, s_pow);
            for (uint32_t i = __lane_id() + 64; i < a.pieces; i += 64) sum += mass[i] * share(top[i], s_pow);
        }
        sum = wave_sum_f64(sum);
        return {sum > 0.0 ? 1.0 / sum : 0.0, m};
    }
};

// The share of a token whose score is v.
__device__ __forceinline__ double share_of(const VerifyArgs& a, float v, Norm n, const double* s_pow)
{
    return v == v && n.part > 0.0 ? Shares(a, n.top)(v, s_pow) * n.part : 0.0;
}

template <class E>
__device__ __forceinline__ float score_of(const void* x, uint64_t row_stride, uint32_t row, uint32_t token)
{
    return E::up(static_cast<const typename E::Bits*>(x)[row * row_stride + token]);
}

// A wave's work: what a row's shares are divided by, and whether the draft behind it, which the
// last of a request's rows has none of, is accepted.  No load but the scores' waits for another.
template <class E>
__device__ __forceinline__ RowState row_state(const VerifyArgs& a, uint32_t row, bool last, const double* s_pow)
{
    RowState s{};
    const Pieces of_p(a, row), of_q(a, a.draft && !last ? a.n_rows + row : row);
    const int32_t token = last ? -1 : a.tokens[row + 1];
    const float u = a.uniform[row];
    const bool there = token >= 0 && static_cast<uint32_t>(token) < a.vocab && is_allowed(a, row, static_cast<uint32_t>(token));
    float x = 0.0f, y = 0.0f;
    if (there) {
        x = score_of<E>(a.x, a.x_row, row, static_cast<uint32_t>(token));
        if (a.draft) y = score_of<E>(a.draft, a.draft_row, row, static_cast<uint32_t>(token));
    }
    s.p = of_p.norm(a, s_pow);
    if (last) return s;
    double q = 1.0;
    if (a.draft) s.q = of_q.norm(a, s_pow);
    if (there) {
        const double p = share_of(a, x, s.p, s_pow);
        if (a.draft) q = share_of(a, y, s.q, s_pow);
        s.accepted = static_cast<double>(u) * q < p ? 1u : 0u;
    }
    return s;
}

// A wave a row.
template <class E>
__global__ __launch_bounds__(64) void dv_norms(VerifyArgs a)
{
    __shared__ double s_pow[DV_POWERS];
    const uint32_t row = blockIdx.x;
    make_powers<64>(s_pow);
    const RowState s = row_state<E>(a, row, row + 1 >= a.n_rows || is_last(a, row), s_pow);
    if (threadIdx.x == 0) a.state[row] = s;
}

// Where request r's accepted drafts end, by the rows' states, which dv_norms has left or the
// workgroup works out here, a wave a row.
template <class E>
__device__ __forceinline__ Decision decide(const VerifyArgs& a, const RequestRows& rows, const double* s_pow, RowState* s_state)
{
    Decision d;
    RowState s;
    if (a.folded) {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        for (uint32_t j0 = 0;; j0 += DV_WAVES) {
            const uint32_t j = j0 + wave;
            if (j <= rows.drafts) {
                const RowState mine = row_state<E>(a, rows.first + j, j == rows.drafts, s_pow);
                if (__lane_id() == 0) s_state[wave] = mine;
            }
            __syncthreads();
            uint32_t w = 0;
            while (w < DV_WAVES && j0 + w < rows.drafts && s_state[w].accepted) ++w;
            d.accepted = j0 + w;
            if (w < DV_WAVES) {  // (the last row's state says no)
                s = s_state[w];
                break;
            }
            __syncthreads();
        }
    } else {
        d.accepted = rows.drafts;
        for (uint32_t j0 = 0; j0 < rows.drafts; j0 += 64) {
            const uint32_t j = j0 + __lane_id();
            const unsigned long long no = __ballot(j < rows.drafts && !a.state[rows.first + min(j, rows.drafts - 1)].accepted);
            if (no) {
                d.accepted = j0 + static_cast<uint32_t>(__ffsll(no)) - 1;
                break;
            }
        }
        s = a.state[rows.first + d.accepted];
    }
    d.row = rows.first + d.accepted;
    d.rejected = d.accepted < rows.drafts;
    d.p = s.p;
    d.q = s.q;
    d.token = d.rejected ? a.tokens[d.row + 1] : -1;
    return d;
}

// max(p - q, 0) of shares and what they are multiplied by, each product rounded by itself, so that
// equal shares leave nothing.
__device__ __forceinline__ double left_of(double p, double p_part, double q, double q_part)
{
#pragma clang fp contract(off)
    return fmax(p * p_part - q * q_part, 0.0);
}

// max(p - q, 0), or p behind the last draft (or where `plain`), of a lane's tokens from
// `first` on: U units, f(u, those of unit u).
template <class E, uint32_t U, class F>
__device__ __forceinline__ void rest_of(const VerifyArgs& a, const Decision& d, uint32_t first, bool plain, const double* s_pow,
                                        F f)
{
    const bool both = a.draft && d.rejected && !plain && d.q.part > 0.0;
    const bool drop = !a.draft && d.rejected && !plain;
    const Mask mask(a, d.row, first);
    Tokens<E, U> of_model, of_draft;
    of_model.load(a, static_cast<const typename E::Bits*>(a.x) + d.row * a.x_row, mask, first);
    if (both) of_draft.load(a, static_cast<const typename E::Bits*>(a.draft) + d.row * a.draft_row, mask, first);
    const double p_part = d.p.part, q_part = d.q.part;
    const Shares p(a, d.p.top), q(a, d.q.top);
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        float x[DV_UNIT];
        double rest[DV_UNIT];
        of_model.scores(mask, first, u, x);
        p.of(x, s_pow, rest);  // (no share where the score is -inf)
        if (both) {
            double y[DV_UNIT];
            of_draft.scores(mask, first, u, x);
            q.of(x, s_pow, y);
#pragma unroll
            for (uint32_t e = 0; e < DV_UNIT; ++e) rest[e] = left_of(rest[e], p_part, y[e], q_part);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < DV_UNIT; ++e) {
                const bool is = drop && static_cast<int32_t>(first + u * 64 * DV_UNIT + e) == d.token;
                rest[e] = is ? 0.0 : rest[e] * p_part;
            }
        }
        f(u, rest);
    }
}

// The pieces' sums of what the next token is drawn from, a wave a piece: two exponentials a
// token.  64 requests over 100003 tokens: 13 us with a fifth of them allowed, of which the
// decision's chain of loads is about 4.
template <class E, bool MASKED>
__global__ __launch_bounds__(DV_NT) __attribute__((amdgpu_waves_per_eu(4))) void dv_rest(VerifyArgs a, uint32_t groups)
{
    __shared__ uint16_t s_few[DV_WAVES][MASKED ? DV_FEW : 1];
    __shared__ double s_pow[DV_POWERS];
    __shared__ RowState s_state[DV_WAVES];
    const uint32_t r = blockIdx.x / groups, lane = __lane_id();
    const uint32_t piece = __builtin_amdgcn_readfirstlane(blockIdx.x % groups * DV_WAVES + (threadIdx.x >> 6));
    const RequestRows rows = rows_of(a, r);
    if (rows.none) return;
    make_powers<DV_NT>(s_pow);
    const Decision d = decide<E>(a, rows, s_pow, s_state);
    if (piece == 0 && lane == 0) a.decided[r] = d;
    if (piece >= a.pieces) return;
    const uint32_t first = piece * DV_PIECE + lane * DV_UNIT;
    double sum = 0.0;
    if constexpr (MASKED) {
        const Mask mask(a, d.row, first);
        const uint16_t* listed = s_few[threadIdx.x >> 6];
        const Few few(a, mask, piece, s_few[threadIdx.x >> 6]);
        if (few.is) {
            const bool both = d.rejected && d.q.part > 0.0;
            const uint64_t from = static_cast<uint64_t>(piece) * DV_PIECE;
            const auto* px = static_cast<const typename E::Bits*>(a.x) + d.row * a.x_row + from;
            const auto* py = static_cast<const typename E::Bits*>(a.draft) + d.row * a.draft_row + from;
            const Shares p(a, d.p.top), q(a, d.q.top);
            float x[DV_UNIT];
            double rest[DV_UNIT], y[DV_UNIT] = {};
            few.get<E>(px, listed, x);
            p.of(x, s_pow, rest);
            if (both) {
                few.get<E>(py, listed, x);
                q.of(x, s_pow, y);
            }
#pragma unroll
            for (uint32_t e = 0; e < DV_UNIT; ++e) sum += left_of(rest[e], d.p.part, y[e], d.q.part);
            sum = wave_sum_f64(sum);
            if (lane == 0) a.rest[static_cast<uint64_t>(r) * a.pieces + piece] = sum;
            return;
        }
    }
    rest_of<E, DV_STEPS>(a, d, first, false, s_pow, [&](uint32_t, const double (&rest)[DV_UNIT]) {
#pragma unroll
        for (uint32_t e = 0; e < DV_UNIT; ++e) sum += rest[e];
    });
    sum = wave_sum_f64(sum);
    if (lane == 0) a.rest[static_cast<uint64_t>(r) * a.pieces + piece] = sum;
}

// A workgroup a request.  Its waves all find the piece; each then looks at a part of it.
// 5 to 6 us, a chain of dependent loads and scans.
template <class E>
__global__ __launch_bounds__(DV_NT) void dv_pick(VerifyArgs a)
{
    static_assert(DV_WAVES == DV_STEPS, "a wave a step of a piece");
    __shared__ double s_pow[DV_POWERS], s_sum[DV_WAVES];
    __shared__ int32_t s_hit[DV_WAVES], s_any[DV_WAVES];
    __shared__ RowState s_state[DV_WAVES];
    const uint32_t r = blockIdx.x, lane = __lane_id(), wave = threadIdx.x >> 6;
    const RequestRows rows = rows_of(a, r);
    int32_t* out = a.out + r * a.out_stride;
    if (rows.none) {
        if (threadIdx.x == 0) a.accepted[r] = 0;
        for (uint32_t j = threadIdx.x; j < a.most; j += DV_NT) out[j] = -1;
        return;
    }
    make_powers<DV_NT>(s_pow);
    const Decision d = a.draft ? a.decided[r] : decide<E>(a, rows, s_pow, s_state);
    for (uint32_t j = threadIdx.x; j < a.most; j += DV_NT)
        if (j != d.accepted) out[j] = j < d.accepted ? a.tokens[rows.first + j + 1] : -1;
    if (threadIdx.x == 0) a.accepted[r] = static_cast<int32_t>(d.accepted);
    // the pieces' sums: of what is left of p, or of p where nothing is
    const uint64_t row0 = static_cast<uint64_t>(d.row) * a.pieces;
    const Shares share(a, d.p.top);
    const bool looked_up = !a.draft && d.rejected && d.token >= 0 && static_cast<uint32_t>(d.token) < a.vocab &&
                           is_allowed(a, d.row, static_cast<uint32_t>(d.token));
    const uint32_t gone = looked_up ? static_cast<uint32_t>(d.token) / DV_PIECE : 0xFFFFFFFFu;
    const double gone_p =
        looked_up ? share_of(a, score_of<E>(a.x, a.x_row, d.row, static_cast<uint32_t>(d.token)), d.p, s_pow) : 0.0;
    bool plain = false, empty = false;  // p itself; the draft's piece holds nothing else
    auto piece_sum = [&](uint32_t i) {
        if (i >= a.pieces || !(d.p.part > 0.0)) return 0.0;
        if (a.draft && d.rejected && !plain) return a.rest[static_cast<uint64_t>(r) * a.pieces + i];
        const float top = a.top[row0 + i];
        const double p = top > -__builtin_inff() ? a.mass[row0 + i] * share(top, s_pow) * d.p.part : 0.0;
        return plain || i != gone ? p : empty ? 0.0 : fmax(p - gone_p, 0.0);
    };
    int32_t token = -1;
    for (;;) {
        double whole = 0.0;
        for (uint32_t i = lane; i < a.pieces; i += 64) whole += piece_sum(i);
        whole = wave_sum_f64(whole);
        if (!(whole > 0.0)) {
            if (plain) break;
            plain = true;
            continue;
        }
        const double mark = static_cast<double>(a.uniform[rows.first + rows.drafts]) * whole;
        // the first piece whose running sum passes the mark, or the last one that holds anything
        double base = 0.0, before = 0.0;
        uint32_t found = 0;
        for (uint32_t i0 = 0; i0 < a.pieces; i0 += 64) {
            const double mine = piece_sum(i0 + lane), upto = wave_incl_scan_f64(mine);
            const unsigned long long pass = __ballot(mine > 0.0 && base + upto > mark), any = __ballot(mine > 0.0);
            if (pass || any) {
                const int l = pass ? __ffsll(pass) - 1 : 63 - __clzll(static_cast<long long>(any));
                found = i0 + static_cast<uint32_t>(l);
                before = base + lane_f64(upto, __builtin_amdgcn_readfirstlane(l)) - lane_f64(mine, __builtin_amdgcn_readfirstlane(l));
            }
            if (pass) break;
            base += lane_f64(upto, 63);
        }
        // the first token of it that does, or its last one that can be drawn
        const uint32_t first = found * DV_PIECE + (wave * 64 + lane) * DV_UNIT;
        double x[DV_UNIT], sum = 0.0;
        rest_of<E, 1>(a, d, first, plain, s_pow, [&](uint32_t, const double (&rest)[DV_UNIT]) {
#pragma unroll
            for (uint32_t e = 0; e < DV_UNIT; ++e) {
                x[e] = rest[e];
                sum += rest[e];
            }
        });
        const double upto = wave_incl_scan_f64(sum);
        if (lane == 63) s_sum[wave] = upto;
        __syncthreads();
        double run = before + (upto - sum);
        for (uint32_t w = 0; w < wave; ++w) run += s_sum[w];
        int32_t hit = -1, any = -1;
#pragma unroll
        for (uint32_t e = 0; e < DV_UNIT; ++e) {
            run += x[e];
            if (x[e] > 0.0) {
                any = static_cast<int32_t>(first + e);
                if (hit < 0 && run > mark) hit = any;
            }
        }
        const unsigned long long hits = __ballot(hit >= 0), anys = __ballot(any >= 0);
        hit = hits ? __shfl(hit, __ffsll(hits) - 1, 64) : -1;
        any = anys ? __shfl(any, 63 - __clzll(static_cast<long long>(anys)), 64) : -1;
        if (lane == 0) {
            s_hit[wave] = hit;
            s_any[wave] = any;
        }
        __syncthreads();
        int32_t behind = -1;
        for (uint32_t w = 0; w < DV_WAVES; ++w) {
            if (token < 0) token = s_hit[w];
            behind = s_any[w] >= 0 ? s_any[w] : behind;
        }
        if (token < 0) token = behind;
        if (token >= 0 || empty || plain) break;
        empty = true;  // rounding had left something where the draft was all there is
        __syncthreads();
    }
    if (threadIdx.x == 0 && d.accepted < a.most) out[d.accepted] = token;
}

template <class E>
int launch_verify(const VerifyArgs& a, hipStream_t s)
{
    const uint64_t waves = static_cast<uint64_t>(a.draft ? 2 : 1) * a.n_rows * a.pieces;
    if (waves) {
        CR_TIMED("dv_sums", s);
        const unsigned grid = static_cast<unsigned>((waves + DV_WAVES - 1) / DV_WAVES);
        if (a.masked)
            dv_sums<E, true><<<grid, DV_NT, 0, s>>>(a);
        else
            dv_sums<E, false><<<grid, DV_NT, 0, s>>>(a);
    }
    if (a.n_rows && !a.folded) {
        CR_TIMED("dv_norms", s);
        dv_norms<E><<<a.n_rows, 64, 0, s>>>(a);
    }
    if (a.draft) {
        CR_TIMED("dv_rest", s);
        const uint32_t groups = (a.pieces + DV_WAVES - 1) / DV_WAVES;
        if (a.masked)
            dv_rest<E, true><<<a.n_requests * groups, DV_NT, 0, s>>>(a, groups);
        else
            dv_rest<E, false><<<a.n_requests * groups, DV_NT, 0, s>>>(a, groups);
    }
    CR_TIMED("dv_pick", s);
    dv_pick<E><<<a.n_requests, DV_NT, 0, s>>>(a);
    CR_LAUNCH_CHECK();
    return CR_OK;
}

}  // namespace

}  // namespace crimpl

using namespace crimpl;

extern "C" int cr_draft_verify(const cr_draft_verify_args* args, cr_stream_t stream)
{
    if (!args) {
        set_error("cr_draft_verify: invalid argument");
        return CR_ERR_INVALID;
    }
    const cr_draft_verify_args& p = *args;
    if (p.n_requests == 0) return CR_OK;
    const uint32_t es = p.dtype == CR_F32 ? 4 : 2;
    if (p.vocab == 0 || p.dtype > CR_BF16 || !p.d_starts || !p.d_accepted || (p.out_cols && !p.d_out) ||
        p.out_stride < p.out_cols || (p.n_rows && (!p.d_scores || !p.d_tokens || !p.d_uniform)) ||
        (p.n_rows > 1 && (p.row_stride < p.vocab || (p.d_draft && p.draft_row_stride < p.vocab))) ||
        (reinterpret_cast<uintptr_t>(p.d_scores) | reinterpret_cast<uintptr_t>(p.d_draft)) % es ||
        (p.allowed && p.d_allowed_bits) || !(p.temperature > 0.0f) || p.temperature > 3.0e38f) {
        set_error("cr_draft_verify: invalid argument (temperature %g)", static_cast<double>(p.temperature));
        return CR_ERR_INVALID;
    }
    VerifyArgs a{};
    a.pieces = (p.vocab + DV_PIECE - 1) / DV_PIECE;
    const uint64_t pieces = 2ull * std::max<uint32_t>(1, p.n_rows) * a.pieces;
    if (p.vocab >> 31 || p.n_rows >> 31 || pieces >> 24 || (static_cast<uint64_t>(p.n_requests) * a.pieces) >> 23 ||
        p.n_requests >> 20) {
        set_error("cr_draft_verify: too many scores for one call");
        return CR_ERR_UNSUPPORTED;
    }
    hipStream_t s = as_stream(stream);
    a.x = p.d_scores;
    a.draft = p.n_rows ? p.d_draft : nullptr;
    a.x_row = p.row_stride;
    a.draft_row = p.draft_row_stride;
    a.n_rows = p.n_rows;
    a.n_requests = p.n_requests;
    a.vocab = p.vocab;
    a.tokens = p.d_tokens;
    a.starts = p.d_starts;
    a.uniform = p.d_uniform;
    a.scale = 256.0 * 1.44269504088896340736 / static_cast<double>(p.temperature);
    a.reach = 693.0 * static_cast<double>(p.temperature);  // 2^-1000
    a.accepted = p.d_accepted;
    a.out = p.d_out;
    a.most = p.out_cols;
    a.out_stride = p.out_stride;
    a.folded = p.n_rows / p.n_requests < DV_FOLD;
    const uint32_t n_words = (p.vocab + 31) / 32;
    const bool direct = p.allowed && is_direct(p.allowed);
    Carver cv;
    const size_t o_mass = cv.add(pieces * 8), o_top = cv.add(pieces * 4);
    const size_t o_rest = cv.add(a.draft ? static_cast<size_t>(p.n_requests) * a.pieces * 8 : 0);
    const size_t o_decided = cv.add(a.draft ? p.n_requests * sizeof(Decision) : 0);
    const size_t o_state = cv.add(a.folded ? 0 : p.n_rows * sizeof(RowState));
    const size_t o_words = cv.add(p.allowed && !direct ? n_words * 4ull : 0);
    Scratch sc;
    CR_RET(sc.alloc(cv.total, s));
    a.mass = sc.at<double>(o_mass);
    a.top = sc.at<float>(o_top);
    a.rest = sc.at<double>(o_rest);
    a.decided = sc.at<Decision>(o_decided);
    a.state = sc.at<RowState>(o_state);
    a.masked = p.allowed || p.d_allowed_bits;
    a.flat = p.d_allowed_bits;
    a.bits_stride = p.bits_stride;
    if (p.allowed)
        CR_RET(set_bits(p.allowed, direct, sc.at<uint32_t>(o_words), n_words, p.vocab, stream, &a.allowed));
    if (p.dtype == CR_F32) return launch_verify<F32>(a, s);
    if (p.dtype == CR_F16) return launch_verify<F16>(a, s);
    return launch_verify<BF16>(a, s);
}

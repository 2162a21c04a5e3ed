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
// sums that differ by 1e-5 and less, and which side it falls on is the answer.
// (gfx950 multiplies and adds 64 bits at the rate of 32.)
//
//   1. dv_sums: every row once, a wave per piece of DV_PIECE tokens: largest score, and
//      the sum of e^((x - largest) / T).
//   2. dv_rest: which drafts are accepted, from the pieces' sums; then the sums of
//      max(p - q, 0) of the row where they end, again by pieces.  Without a drafting
//      model's scores q is 1 for the drafted token, and the pieces of p do.
//   3. dv_pick: the piece in which the running sum passes the mark, and the token in it.
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

struct VerifyArgs {
    const void* x;
    const void* draft;  // or nullptr
    uint64_t x_row, draft_row;
    uint32_t n_rows, n_requests, vocab, pieces;
    const int32_t* tokens;
    const int32_t* starts;
    const float* uniform;
    double scale;        // log2(e) / temperature
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
    double* rest;          // [n_requests][pieces]
    struct Decision* decided;  // [n_requests]
};

// 2^t for t <= 0: the power of two apart, and the series of e^y to y^11 for |y| <=
// log(2) / 2, which leaves 7e-15 of it.  Far below 2^-1022, and for -inf, 0.
__device__ __forceinline__ double exp2_64(double t)
{
    t = fmax(t, -1100.0);  // (-inf, whose fraction would be NaN; NaN is taken for it)
    const double n = rint(t), y = (t - n) * 0.693147180559945309417;
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
    return ldexp(e, static_cast<int>(n));
}

// e^((x - top) / T); of an infinite largest score, those that reach it share the mass.
__device__ __forceinline__ double part_of(float x, float top, double scale)
{
    return x == top ? (top == -__builtin_inff() ? 0.0 : 1.0)
                    : exp2_64((static_cast<double>(x) - static_cast<double>(top)) * scale);
}

__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ double wave_incl_scan_f64(double v)
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double x = __shfl_up(v, o, 64);
        if (static_cast<int>(__lane_id()) >= o) v += x;
    }
    return v;
}

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// Tokens [first, first + DV_UNIT) of a row: -inf for those that are not there, may not
// be used or are NaN.
template <class E>
__device__ __forceinline__ void load_scores(const typename E::Bits* row, uint32_t first, uint32_t vocab, uint32_t on,
                                            float (&x)[DV_UNIT])
{
    typedef typename E::Bits Bits;
    // rows may begin anywhere
    typedef Bits Wide __attribute__((ext_vector_type(DV_UNIT), aligned(sizeof(Bits))));
    if (first + DV_UNIT <= vocab) {
        const Wide w = __builtin_nontemporal_load(reinterpret_cast<const Wide*>(row + first));
#pragma unroll
        for (uint32_t e = 0; e < DV_UNIT; ++e) x[e] = E::up(w[e]);
    } else {
#pragma unroll
        for (uint32_t e = 0; e < DV_UNIT; ++e) x[e] = first + e < vocab ? E::up(row[first + e]) : 0.0f;
    }
#pragma unroll
    for (uint32_t e = 0; e < DV_UNIT; ++e) x[e] = (on >> e) & 1u && x[e] == x[e] ? x[e] : -__builtin_inff();
}

// Which of tokens [first, first + DV_UNIT) are there and may be used after row `row`.
__device__ __forceinline__ uint32_t allowed_unit(const VerifyArgs& a, uint64_t row, uint32_t first)
{
    if (first >= a.vocab) return 0u;
    uint32_t on = first + DV_UNIT <= a.vocab ? 0xFFu : (1u << (a.vocab - first)) - 1u;
    if (a.masked) {
        const uint32_t word = a.flat ? a.flat[row * a.bits_stride + first / 32u] : a.allowed.word(first / 32u);
        on &= word >> (first % 32u);
    }
    return on;
}

__device__ __forceinline__ bool is_allowed(const VerifyArgs& a, uint64_t row, uint32_t token)
{
    return (allowed_unit(a, row, token / DV_UNIT * DV_UNIT) >> (token % DV_UNIT)) & 1u;
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

// Every row's pieces; the drafting model's rows behind the model's.
template <class E>
__global__ __launch_bounds__(DV_NT) void dv_sums(VerifyArgs a)
{
    const uint32_t lane = __lane_id(), wave = blockIdx.x * DV_WAVES + (threadIdx.x >> 6);
    const uint32_t at = wave / a.pieces, piece = wave % a.pieces;
    if (at >= (a.draft ? 2 : 1) * a.n_rows) return;
    const bool drafted = at >= a.n_rows;
    const uint32_t row = drafted ? at - a.n_rows : at;
    const auto* p = static_cast<const typename E::Bits*>(drafted ? a.draft : a.x) +
                    row * (drafted ? a.draft_row : a.x_row);
    float x[DV_STEPS][DV_UNIT], top = -__builtin_inff();
    uint32_t on[DV_STEPS];
#pragma unroll
    for (uint32_t u = 0; u < DV_STEPS; ++u)
        on[u] = allowed_unit(a, row, piece * DV_PIECE + (u * 64 + lane) * DV_UNIT);
#pragma unroll
    for (uint32_t u = 0; u < DV_STEPS; ++u) {
        load_scores<E>(p, piece * DV_PIECE + (u * 64 + lane) * DV_UNIT, a.vocab, on[u], x[u]);
#pragma unroll
        for (uint32_t e = 0; e < DV_UNIT; ++e) top = fmaxf(top, x[u][e]);
    }
    top = wave_max(top);
    double mass = 0.0;
    if (top > -__builtin_inff()) {
#pragma unroll
        for (uint32_t u = 0; u < DV_STEPS; ++u)
#pragma unroll
            for (uint32_t e = 0; e < DV_UNIT; ++e) mass += part_of(x[u][e], top, a.scale);
    }
    mass = wave_sum_f64(mass);
    if (lane == 0) {
        a.top[wave] = top;
        a.mass[wave] = mass;
    }
}

struct Norm {  // of a row: p(v) = e^((x_v - top) / T) * part
    float top;
    double part;
};

// A wave's work: the pieces joined in a fixed order.
__device__ __forceinline__ Norm norm_of(const VerifyArgs& a, uint32_t at)
{
    const float* top = a.top + static_cast<uint64_t>(at) * a.pieces;
    const double* mass = a.mass + static_cast<uint64_t>(at) * a.pieces;
    float m = -__builtin_inff();
    for (uint32_t i = __lane_id(); i < a.pieces; i += 64) m = fmaxf(m, top[i]);
    m = wave_max(m);
    double sum = 0.0;
    for (uint32_t i = __lane_id(); i < a.pieces; i += 64)
        if (mass[i] > 0.0) sum += mass[i] * part_of(top[i], m, a.scale);
    sum = wave_sum_f64(sum);
    return {m, sum > 0.0 ? 1.0 / sum : 0.0};
}

struct Decision {
    uint32_t row, accepted;
    uint32_t rejected;  // whether the draft there was: its token
    int32_t token;
    Norm p, q;
};

// p and q of one token.
template <class E>
__device__ __forceinline__ double share_of(const VerifyArgs& a, const void* x, uint64_t row_stride, uint32_t row,
                                           uint32_t token, Norm n)
{
    const float v = E::up(static_cast<const typename E::Bits*>(x)[row * row_stride + token]);
    return v == v && n.part > 0.0 ? part_of(v, n.top, a.scale) * n.part : 0.0;
}

// How many drafts of request r are accepted.  A workgroup's work, a wave a draft at a time.
template <class E>
__device__ __forceinline__ Decision decide(const VerifyArgs& a, const RequestRows& rows, Decision* s_waves)
{
    const uint32_t wave = threadIdx.x >> 6;
    Decision d{};
    for (uint32_t j0 = 0;; j0 += DV_WAVES) {
        const uint32_t j = min(j0 + wave, rows.drafts), row = rows.first + j;
        d.row = row;
        d.accepted = j;
        d.rejected = 0;
        d.token = -1;
        d.p = norm_of(a, row);
        d.q = {0.0f, 0.0};
        if (j < rows.drafts) {
            d.token = a.tokens[row + 1];
            double p = 0.0, q = 1.0;
            if (a.draft) d.q = norm_of(a, a.n_rows + row);
            const bool there = d.token >= 0 && static_cast<uint32_t>(d.token) < a.vocab &&
                               is_allowed(a, row, static_cast<uint32_t>(d.token));
            if (there) {
                p = share_of<E>(a, a.x, a.x_row, row, static_cast<uint32_t>(d.token), d.p);
                if (a.draft) q = share_of<E>(a, a.draft, a.draft_row, row, static_cast<uint32_t>(d.token), d.q);
            }
            d.rejected = there && static_cast<double>(a.uniform[row]) * q < p ? 0u : 1u;
        }
        if (__lane_id() == 0) s_waves[wave] = d;
        __syncthreads();
        // the first that ends it
        uint32_t end = DV_WAVES;
        for (uint32_t w = 0; w < DV_WAVES; ++w)
            if (end == DV_WAVES && (s_waves[w].rejected || s_waves[w].accepted == rows.drafts)) end = w;
        if (end < DV_WAVES) d = s_waves[end];
        __syncthreads();
        if (end < DV_WAVES) return d;
    }
}

// max(p - q, 0), or p behind the last draft, of a lane's tokens from `first`.
template <class E>
__device__ __forceinline__ void rest_of(const VerifyArgs& a, const Decision& d, uint32_t first, bool plain,
                                        double (&rest)[DV_UNIT])
{
    // each product rounded by itself, so that equal shares leave nothing
#pragma clang fp contract(off)
    const uint32_t on = allowed_unit(a, d.row, first);
    float x[DV_UNIT], y[DV_UNIT];
    if (first < a.vocab) {
        load_scores<E>(static_cast<const typename E::Bits*>(a.x) + d.row * a.x_row, first, a.vocab, on, x);
        if (a.draft && d.rejected && !plain)
            load_scores<E>(static_cast<const typename E::Bits*>(a.draft) + d.row * a.draft_row, first, a.vocab, on, y);
    }
#pragma unroll
    for (uint32_t e = 0; e < DV_UNIT; ++e) {
        rest[e] = 0.0;
        if (first >= a.vocab || !((on >> e) & 1u) || d.p.part == 0.0) continue;
        rest[e] = part_of(x[e], d.p.top, a.scale) * d.p.part;
        if (!d.rejected || plain) continue;
        if (a.draft) {
            if (d.q.part > 0.0) rest[e] = fmax(rest[e] - part_of(y[e], d.q.top, a.scale) * d.q.part, 0.0);
        } else if (static_cast<int32_t>(first + e) == d.token) {
            rest[e] = 0.0;
        }
    }
}

// The pieces' sums of what the next token is drawn from, a wave a piece.
template <class E>
__global__ __launch_bounds__(DV_NT) void dv_rest(VerifyArgs a, uint32_t groups)
{
    __shared__ Decision s_waves[DV_WAVES];
    const uint32_t r = blockIdx.x / groups, part = blockIdx.x % groups, lane = __lane_id();
    const RequestRows rows = rows_of(a, r);
    if (rows.none) return;
    const Decision d = decide<E>(a, rows, s_waves);
    if (part == 0 && threadIdx.x == 0) a.decided[r] = d;
    const uint32_t piece = part * DV_WAVES + (threadIdx.x >> 6);
    if (piece >= a.pieces) return;
    double sum = 0.0;
#pragma unroll
    for (uint32_t u = 0; u < DV_STEPS; ++u) {
        double rest[DV_UNIT];
        rest_of<E>(a, d, piece * DV_PIECE + (u * 64 + lane) * DV_UNIT, false, rest);
#pragma unroll
        for (uint32_t e = 0; e < DV_UNIT; ++e) sum += rest[e];
    }
    sum = wave_sum_f64(sum);
    if (lane == 0) a.rest[static_cast<uint64_t>(r) * a.pieces + piece] = sum;
}

// The piece's own sum of p.
__device__ __forceinline__ double piece_of_p(const VerifyArgs& a, const Decision& d, uint32_t piece)
{
    const uint64_t at = static_cast<uint64_t>(d.row) * a.pieces + piece;
    const double mass = a.mass[at];
    return mass > 0.0 ? mass * part_of(a.top[at], d.p.top, a.scale) * d.p.part : 0.0;
}

// A workgroup a request; its first wave finds the token.
template <class E>
__global__ __launch_bounds__(DV_NT) void dv_pick(VerifyArgs a)
{
    __shared__ Decision s_waves[DV_WAVES];
    const uint32_t r = blockIdx.x, lane = __lane_id();
    const RequestRows rows = rows_of(a, r);
    int32_t* out = a.out + r * a.out_stride;
    if (rows.none) {
        if (threadIdx.x == 0) a.accepted[r] = 0;
        for (uint32_t j = threadIdx.x; j < a.most; j += DV_NT) out[j] = -1;
        return;
    }
    Decision d;
    if (a.draft)
        d = a.decided[r];
    else
        d = decide<E>(a, rows, s_waves);
    for (uint32_t j = threadIdx.x; j < a.most; j += DV_NT)
        if (j != d.accepted) out[j] = j < d.accepted ? a.tokens[rows.first + j + 1] : -1;
    if (threadIdx.x >= 64) return;
    if (lane == 0) a.accepted[r] = static_cast<int32_t>(d.accepted);
    // the pieces' sums: of what is left of p, or of p where nothing is
    const double* rest = a.draft ? a.rest + static_cast<uint64_t>(r) * a.pieces : nullptr;
    const uint32_t gone = !a.draft && d.rejected && d.token >= 0 && static_cast<uint32_t>(d.token) < a.vocab &&
                                  is_allowed(a, d.row, static_cast<uint32_t>(d.token))
                              ? static_cast<uint32_t>(d.token)
                              : 0xFFFFFFFFu;
    const double gone_p = gone != 0xFFFFFFFFu ? share_of<E>(a, a.x, a.x_row, d.row, gone, d.p) : 0.0;
    bool plain = false;
    auto piece_sum = [&](uint32_t i) {
        if (i >= a.pieces) return 0.0;
        if (plain || !rest) {
            const double p = piece_of_p(a, d, i);
            return !plain && gone / DV_PIECE == i ? fmax(p - gone_p, 0.0) : p;
        }
        return rest[i];
    };
    double whole = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        whole = 0.0;
        for (uint32_t i = lane; i < a.pieces; i += 64) whole += piece_sum(i);
        whole = wave_sum_f64(whole);
        if (whole > 0.0) break;
        plain = true;
    }
    int32_t token = -1;
    if (whole > 0.0) {
        const double mark = static_cast<double>(a.uniform[rows.first + rows.drafts]) * whole;
        // the first piece whose running sum passes the mark, or the last one that holds anything
        double base = 0.0, before = 0.0;
        uint32_t found = 0xFFFFFFFFu, last = 0;
        double last_before = 0.0;
        for (uint32_t i0 = 0; i0 < a.pieces && found == 0xFFFFFFFFu; i0 += 64) {
            const double mine = piece_sum(i0 + lane), upto = wave_incl_scan_f64(mine);
            const unsigned long long pass = __ballot(mine > 0.0 && base + upto > mark), any = __ballot(mine > 0.0);
            if (pass) {
                const int l = __ffsll(static_cast<unsigned long long>(pass)) - 1;
                found = i0 + static_cast<uint32_t>(l);
                before = base + __shfl(upto, l, 64) - __shfl(mine, l, 64);
            } else if (any) {
                const int l = 63 - __clzll(static_cast<long long>(any));
                last = i0 + static_cast<uint32_t>(l);
                last_before = base + __shfl(upto, l, 64) - __shfl(mine, l, 64);
            }
            base += __shfl(upto, 63, 64);
        }
        if (found == 0xFFFFFFFFu) {
            found = last;
            before = last_before;
        }
        // the first token of it that does, or its last one that can be drawn
        int32_t behind = -1;
        for (uint32_t u = 0; u < DV_STEPS && token < 0; ++u) {
            const uint32_t first = found * DV_PIECE + (u * 64 + lane) * DV_UNIT;
            double x[DV_UNIT], sum = 0.0;
            rest_of<E>(a, d, first, plain, x);
#pragma unroll
            for (uint32_t e = 0; e < DV_UNIT; ++e) sum += x[e];
            const double upto = wave_incl_scan_f64(sum);
            double run = before + upto - sum;
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
            if (hits) token = __shfl(hit, __ffsll(hits) - 1, 64);
            if (anys) behind = __shfl(any, 63 - __clzll(static_cast<long long>(anys)), 64);
            before += __shfl(upto, 63, 64);
        }
        if (token < 0) token = behind;
    }
    if (lane == 0 && d.accepted < a.most) out[d.accepted] = token;
}

template <class E>
int launch_verify(const VerifyArgs& a, hipStream_t s)
{
    const uint64_t waves = static_cast<uint64_t>(a.draft ? 2 : 1) * a.n_rows * a.pieces;
    if (waves) {
        CR_TIMED("dv_sums", s);
        dv_sums<E><<<static_cast<unsigned>((waves + DV_WAVES - 1) / DV_WAVES), DV_NT, 0, s>>>(a);
    }
    if (a.draft) {
        CR_TIMED("dv_rest", s);
        const uint32_t groups = (a.pieces + DV_WAVES - 1) / DV_WAVES;
        dv_rest<E><<<a.n_requests * groups, DV_NT, 0, s>>>(a, groups);
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
    a.scale = 1.44269504088896340736 / static_cast<double>(p.temperature);
    a.accepted = p.d_accepted;
    a.out = p.d_out;
    a.most = p.out_cols;
    a.out_stride = p.out_stride;
    const uint32_t n_words = (p.vocab + 31) / 32;
    const bool direct = p.allowed && is_direct(p.allowed);
    Carver cv;
    const size_t o_mass = cv.add(pieces * 8), o_top = cv.add(pieces * 4);
    const size_t o_rest = cv.add(a.draft ? static_cast<size_t>(p.n_requests) * a.pieces * 8 : 0);
    const size_t o_decided = cv.add(a.draft ? p.n_requests * sizeof(Decision) : 0);
    const size_t o_words = cv.add(p.allowed && !direct ? n_words * 4ull : 0);
    Scratch sc;
    CR_RET(sc.alloc(cv.total, s));
    a.mass = sc.at<double>(o_mass);
    a.top = sc.at<float>(o_top);
    a.rest = sc.at<double>(o_rest);
    a.decided = sc.at<Decision>(o_decided);
    a.masked = p.allowed || p.d_allowed_bits;
    a.flat = p.d_allowed_bits;
    a.bits_stride = p.bits_stride;
    if (p.allowed)
        CR_RET(set_bits(p.allowed, direct, sc.at<uint32_t>(o_words), n_words, p.vocab, stream, &a.allowed));
    if (p.dtype == CR_F32) return launch_verify<F32>(a, s);
    if (p.dtype == CR_F16) return launch_verify<F16>(a, s);
    return launch_verify<BF16>(a, s);
}

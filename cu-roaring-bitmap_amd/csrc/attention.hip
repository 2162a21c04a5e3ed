// Attention of new tokens over a paged key/value cache (no reference
// implementation).
//
// For token t and head h, over the keys j that the token sees:
//   s_j = scale * q_t . k_j,  o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),
//   lse = m + log(sum_j e^(s_j - m)),  m = max_j s_j.
#include <algorithm>

#include "internal.hpp"
#include "attention_work.hpp"

namespace crimpl {

namespace {

constexpr uint32_t AT_DIM_MAX = 256;

typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint16_t v2u16 __attribute__((ext_vector_type(2)));
typedef uint16_t v4u16 __attribute__((ext_vector_type(4)));
typedef uint16_t v8u16 __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// The two element types: rounding to nearest even, and the matrix products.
struct Half {
    static __device__ __forceinline__ float up(uint16_t x)
    {
        return static_cast<float>(__builtin_bit_cast(_Float16, x));
    }
    static __device__ __forceinline__ uint16_t down(float x)
    {
        return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
    }
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
    static constexpr uint32_t EXP = 0x7C00u;  // the exponent's bits: all set in infinities and NaN
    static constexpr float LIFT = 7.0f;
};
struct BHalf {
    static __device__ __forceinline__ float up(uint16_t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }
    static __device__ __forceinline__ uint16_t down(float x)
    {
        return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
    }
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
    static constexpr uint32_t EXP = 0x7F80u;
    static constexpr float LIFT = 0.0f;
};

constexpr float NEG_INF = -__builtin_inff();
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.693147180559945309417f;
// A row's running maximum may fall this far (in powers of two) behind its
// scores before the sums are scaled anew: a row is then scaled a few times in all
// instead of at each new maximum.
constexpr float LAG = 8.0f;

// What a row's scores, in powers of two, are lowered by before their exponentials.
// Those are summed in fp32, and rounded to the keys' type for the second product:
// the matrix units take that type, and products of an upper and a lower part would
// be twice as many.  bf16 has fp32's range.  f16 begins at 2^-24, so that its
// exponentials are lifted by 2^LIFT: with the lag they reach 2^15, which it holds,
// and a key counts down to 2^-32 of the row's largest (unlifted, 131072 keys at 2^-25
// of it were lost).  Sums are lifted alike; the log-sum is lowered again.
template <class E>
__device__ __forceinline__ float base_of(float m, float c)
{
    return __builtin_fmaf(m, c, -E::LIFT);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Four transposed pieces of LDS: of each 16 lanes, lane i names 8 bytes of row
// i / 4 and receives elements i of the four rows.
__device__ __forceinline__ v4s lds_tr(const uint16_t* p)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p);
}

__device__ __forceinline__ v8s join(v4s x, v4s y) { return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7); }

__device__ __forceinline__ v8s load8(const uint16_t* p) { return *reinterpret_cast<const v8s*>(p); }
// The same, for data that no other workgroup reads.
__device__ __forceinline__ v8s load8_once(const uint16_t* p)
{
    return __builtin_nontemporal_load(reinterpret_cast<const v8s*>(p));
}
__device__ __forceinline__ v4s load4(const uint16_t* p) { return *reinterpret_cast<const v4s*>(p); }

// Whether any of eight values is infinite or NaN, and the eight with zeros for those.
__device__ __forceinline__ bool has_special(v8s x, uint32_t exp)
{
    const v8u16 y = __builtin_bit_cast(v8u16, x) & static_cast<uint16_t>(0x7FFF);
    const v4u16 a = __builtin_elementwise_max(__builtin_shufflevector(y, y, 0, 1, 2, 3),
                                              __builtin_shufflevector(y, y, 4, 5, 6, 7));
    const v2u16 b = __builtin_elementwise_max(__builtin_shufflevector(a, a, 0, 1), __builtin_shufflevector(a, a, 2, 3));
    return max(b[0], b[1]) >= exp;
}

__device__ __forceinline__ v8s without_special(v8s x, uint32_t exp)
{
    v4u w = __builtin_bit_cast(v4u, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = (w[i] & exp) == exp ? 0u : 0xFFFFu;
        const uint32_t hi = (w[i] & (exp << 16)) == exp << 16 ? 0u : 0xFFFF0000u;
        w[i] &= lo | hi;
    }
    return __builtin_bit_cast(v8s, w);
}

__device__ __forceinline__ v8s zero_unless(bool keep, v8s x)
{
    const uint32_t mask = keep ? 0xFFFFFFFFu : 0u;
    return __builtin_bit_cast(v8s, __builtin_bit_cast(v4u, x) & mask);
}

// The lowest n bits, all for n >= 32 and none for n <= 0.
__device__ __forceinline__ uint32_t low_bits(int32_t n)
{
    return n >= 32 ? 0xFFFFFFFFu : (1u << max(n, 0)) - 1u;
}

// The score where bit i of `on` is set, else -inf.
__device__ __forceinline__ float score_if(uint32_t on, uint32_t i, float x)
{
    const uint32_t keep = static_cast<uint32_t>(static_cast<int32_t>(on << (31u - i)) >> 31);
    return __uint_as_float((__float_as_uint(x) & keep) | (0xFF800000u & ~keep));
}

// Adds the infinite and NaN ones of four values.
template <class E, class V>
__device__ __forceinline__ void add_special(V& o, uint32_t i, v4s x)
{
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e)
        if ((static_cast<uint16_t>(x[e]) & E::EXP) == E::EXP) o[i + e] += E::up(static_cast<uint16_t>(x[e]));
}

// 16 bytes a lane from memory to LDS, lane after lane from `to`, which is the
// same for the wave.
__device__ __forceinline__ void load_to_lds(const uint16_t* from, uint16_t* to)
{
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) const void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

__device__ __forceinline__ uint32_t limit_of(const AttnArgs& a, const Work& t, uint32_t token)
{
    if (!t.real || !a.causal) return t.keys;
    const int64_t at = a.sel ? static_cast<int64_t>(a.limits[t.token0 + token])
                             : static_cast<int64_t>(t.len) - t.tokens + token + 1;
    return static_cast<uint32_t>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(t.keys), at)));
}

// The cache slot of the request's key j < keys, -1 where its page is outside
// the cache.
// In two steps, so that nothing waits for the load before it has to: what the
// selection or the table holds for it, and what that says.
__device__ __forceinline__ int32_t look_up(const AttnArgs& a, uint32_t request, uint32_t j)
{
    return a.sel ? a.sel[request * a.sel_stride + j] : a.table[request * a.table_stride + (j >> a.page_lg)];
}

__device__ __forceinline__ int32_t slot_of(const AttnArgs& a, int32_t found, uint32_t j)
{
    const uint32_t page = a.sel ? static_cast<uint32_t>(found) >> a.page_lg : static_cast<uint32_t>(found);
    const uint32_t slot = a.sel ? static_cast<uint32_t>(found) : (page << a.page_lg) + (j & ((1u << a.page_lg) - 1u));
    return page < a.n_pages ? static_cast<int32_t>(slot) : -1;
}

__device__ __forceinline__ uint64_t offset_of(int32_t slot, uint32_t page_lg, uint64_t page_stride,
                                              uint64_t slot_stride)
{
    const uint32_t at = static_cast<uint32_t>(max(slot, 0));
    return (at >> page_lg) * page_stride + (at & ((1u << page_lg) - 1u)) * slot_stride;
}

// A row's queries come in with the sign of the scale, so that the largest product
// is the largest score.
struct Query {
    const uint16_t* p;
    uint32_t dim;  // 0: zeros
    __device__ __forceinline__ Query(const AttnArgs& a, const Work& t, uint32_t row, uint32_t kh)
    {
        const uint32_t group = a.heads / a.kv_heads, at = min(row, t.rows - 1);
        p = a.q + (static_cast<uint64_t>(t.token0) + at / group) * a.q_token + (kh * group + at % group) * a.q_head;
        dim = row < t.rows && a.scale != 0.0f ? a.dim : 0u;
    }
    // Dimensions [d, d + 8), in two steps: nothing waits for the load but the second.
    __device__ __forceinline__ v4u load(uint32_t d) const
    {
        return *reinterpret_cast<const v4u*>(p + (d < dim ? d : 0u));
    }
};

__device__ __forceinline__ v8s finish_query(const AttnArgs& a, uint32_t dim, uint32_t d, v4u x)
{
    return __builtin_bit_cast(v8s, (x & (d < dim ? 0xFFFFFFFFu : 0u)) ^ (a.scale < 0.0f ? 0x80008000u : 0u));
}

__device__ __forceinline__ float score_scale(const AttnArgs& a)
{
    return a.scale == 0.0f ? 1.0f : fabsf(a.scale) * LOG2E;  // queries are zero where the scale is
}

// A row's four dimensions from d: rounded into the output, or kept in fp32
// where another kernel joins the ranges of keys.  `place` numbers the rows of
// the ranges' results.
template <class E>
__device__ __forceinline__ void store_row(const AttnArgs& a, E, const Work& t, uint64_t place, uint32_t token,
                                          uint32_t head, uint32_t d, f32x4 x)
{
    if (!t.whole) {
        *reinterpret_cast<f32x4*>(a.part_o + place * a.dim + d) = x;
    } else {
        const v4s y = {static_cast<short>(E::down(x[0])), static_cast<short>(E::down(x[1])),
                       static_cast<short>(E::down(x[2])), static_cast<short>(E::down(x[3]))};
        *reinterpret_cast<v4s*>(a.out + token * a.out_token + head * a.out_head + d) = y;
    }
}

// lse2: base 2
__device__ __forceinline__ void store_lse(const AttnArgs& a, const Work& t, uint64_t place, uint32_t token,
                                          uint32_t head, float lse2)
{
    if (!t.whole)
        a.part_lse[place] = lse2;
    else if (a.lse)
        a.lse[static_cast<uint64_t>(token) * a.heads + head] = lse2 * LN2;
}

// ---- few rows: bound by reading keys and values ------------------------------------
// A workgroup answers up to 16 NB rows over a range of keys, each of its waves
// every fourth 32 of them on its own: scores are transposed products (keys x
// rows) of 16x16x32 matrix instructions, whose result has a row's probabilities
// in the lanes that the second product wants them in, if keys are taken in the
// order 4h..4h+3, 16+4h..16+4h+3 for lane group h.  Keys and values are loaded
// into registers a tile ahead, whole rows by neighbouring lanes and past the
// caches, and pass through the wave's own LDS, which hands keys out in operand
// order and transposes values; rows there are turned by pieces of 16 bytes
// against bank conflicts.  No wave waits for another before the end.
//
// 64 requests of up to 16384 keys, 32 heads over 8, 128 dimensions, bf16: 335 us
// with the join, 5.85 TB/s (the card copies 1 GiB at 4.75 and reads alone at up to
// 7).  On the way, each alone: keys loaded straight in operand order, which asks
// for half lines, 400, past the caches even 430; whole rows past them 376; a tile's
// offsets looked up once, through LDS, 361.  48 requests of 4 rows and up to 2048
// keys, 16 heads of 64 dimensions: 49 us, 4.5 TB/s; they are one workgroup a slot
// of the card and wait for the longest (64 keys a tile, with fewer waves, 59).

template <uint32_t DIM>
struct Rows {
    static constexpr uint32_t CHUNKS = DIM <= 64 ? 8 : DIM <= 128 ? 16 : 32;  // 16-byte pieces of a row in LDS
    static constexpr uint32_t STRIDE = CHUNKS * 8;                             // its elements
};

template <class E, uint32_t DIM, uint32_t NB>
__global__ __launch_bounds__(DC_NT) void at_rows(AttnArgs a)
{
    constexpr uint32_t STEPS = DIM / 32, BLOCKS = DIM / 16, CHUNKS = Rows<DIM>::CHUNKS, STRIDE = Rows<DIM>::STRIDE;
    constexpr uint32_t PER = 64 / CHUNKS, LOADS = DC_KEYS / PER;  // values: rows an instruction covers, instructions
    constexpr uint32_t RED = DIM + 4;
    // the values' tiles, and in the end the waves' sums
    constexpr uint32_t KTURN = CHUNKS < 16 ? CHUNKS - 1 : 15;
    constexpr uint32_t BYTES = DC_WAVES * (DC_KEYS * STRIDE * 4 > 16 * RED * 4 ? DC_KEYS * STRIDE * 4 : 16 * RED * 4);
    __shared__ alignas(16) char s_mem[BYTES];
    __shared__ uint64_t s_at[DC_WAVES][2][DC_KEYS];  // where a tile's keys and values are
    __shared__ float s_m[DC_WAVES][16 * NB], s_l[DC_WAVES][16 * NB];
    const uint32_t lane = __lane_id(), wave = threadIdx.x >> 6, c16 = lane & 15u, h = lane >> 4;
    const uint32_t kh = blockIdx.x % a.kv_heads, group = a.heads / a.kv_heads;
    const Work t = find_work<false, true>(a, blockIdx.x / a.kv_heads, 16 * NB);
    if (t.none) return;
    // Lane j < 32 (and j + 32) looks after key j of a tile.  The first look-up comes
    // before all that is not needed for it: what is loaded later is waited for later.
    auto find = [&](uint32_t j0, uint32_t end) { return look_up(a, t.request, min(j0 + (lane & 31u), end - 1)); };
    uint32_t j0 = t.k0 + wave * DC_KEYS;
    int32_t found = j0 < t.k1 ? find(j0, t.k1) : -1;
    uint32_t limit[NB], most = 0, least = 0xFFFFFFFFu;
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) {
        const uint32_t row = t.row0 + b * 16 + c16;
        limit[b] = row < t.rows ? limit_of(a, t, row / group) : 0u;
        most = max(most, limit[b]);
        if (row < t.rows) least = min(least, limit[b]);
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), o, 64)));
        least = min(least, static_cast<uint32_t>(__shfl_xor(static_cast<int>(least), o, 64)));
    }
    most = __builtin_amdgcn_readfirstlane(most);
    least = __builtin_amdgcn_readfirstlane(least);
    const uint32_t k0 = t.k0, k1 = min(most, t.k1);
    const uint64_t place0 = (static_cast<uint64_t>(t.range) * a.kv_heads + kh) * (16 * NB);  // of the tile's first row
    if (!t.whole && k0 >= k1) {
        if (threadIdx.x < 16 * NB) a.part_lse[place0 + threadIdx.x] = NEG_INF;
        return;
    }

    v4u q_raw[NB][STEPS];
    uint32_t q_dim[NB];
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) {
        const Query from(a, t, t.row0 + b * 16 + c16, kh);
        q_dim[b] = from.dim;
#pragma unroll
        for (uint32_t s = 0; s < STEPS; ++s) q_raw[b][s] = from.load(s * 32 + h * 8);
    }
    f32x4 o[NB][BLOCKS];
    float m[NB], l[NB];
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) {
        m[b] = NEG_INF;
        l[b] = 0.0f;
#pragma unroll
        for (uint32_t d = 0; d < BLOCKS; ++d) o[b][d] = f32x4{0, 0, 0, 0};
    }
    const float c = score_scale(a);
    uint16_t* lds_k = reinterpret_cast<uint16_t*>(s_mem) + wave * 2 * DC_KEYS * STRIDE;
    uint16_t* lds = lds_k + DC_KEYS * STRIDE;
    const uint32_t vrow = lane / CHUNKS, vchunk = lane % CHUNKS;
    const uint32_t vcol = vchunk * 8 < a.dim ? vchunk * 8 : 0u;
    const uint16_t* kp = a.k + kh * a.k_head + vcol;
    const uint16_t* vp = a.v + kh * a.v_head + vcol;

    v8s k[LOADS], v[LOADS];
    auto slots = [&](uint32_t j0, int32_t found) {
        const uint32_t j = j0 + (lane & 31u);
        return j < k1 ? slot_of(a, found, j) : -1;
    };
    auto note = [&](int32_t slot) {
        if (lane < DC_KEYS) {
            s_at[wave][0][lane] = offset_of(slot, a.page_lg, a.k_page, a.k_slot);
            s_at[wave][1][lane] = offset_of(slot, a.page_lg, a.v_page, a.v_slot);
        }
        wave_lds_fence();
    };
    auto load_keys = [&]() {
#pragma unroll
        for (uint32_t i = 0; i < LOADS; ++i) k[i] = load8_once(kp + s_at[wave][0][i * PER + vrow]);
    };
    auto load_values = [&]() {
#pragma unroll
        for (uint32_t i = 0; i < LOADS; ++i) v[i] = load8_once(vp + s_at[wave][1][i * PER + vrow]);
    };

    // Pieces behind the head dimension are loaded from the row's beginning.  Those of
    // keys become zeros, as the queries they meet; those of values reach only columns
    // that are not stored.
    const bool inside = vchunk * 8 < a.dim;
    auto put_key = [&](uint32_t i, v8s x) {
        const uint32_t r = i * PER + vrow;
        *reinterpret_cast<v8s*>(lds_k + r * STRIDE + (vchunk ^ (r & KTURN)) * 8) = zero_unless(inside, x);
    };

    int32_t slot = -1, next = -1;
    if (j0 < k1) {
        slot = slots(j0, found);
        note(slot);
        found = find(j0 + DC_WAVES * DC_KEYS, k1);
        load_keys();
        load_values();
    }
    v8s q[NB][STEPS];
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
        for (uint32_t s = 0; s < STEPS; ++s) q[b][s] = finish_query(a, q_dim[b], s * 32 + h * 8, q_raw[b][s]);
    for (; j0 < k1; j0 += DC_WAVES * DC_KEYS) {
        const uint64_t there = __ballot(slot >= 0);
        const bool more = j0 + DC_WAVES * DC_KEYS < k1;
        const bool whole = static_cast<uint32_t>(there) == 0xFFFFFFFFu && j0 + DC_KEYS <= least;
        f32x4 s[NB][2];
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
            for (uint32_t x = 0; x < 2; ++x) s[b][x] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (uint32_t i = 0; i < LOADS; ++i) put_key(i, k[i]);
        if (more) {
            next = slots(j0 + DC_WAVES * DC_KEYS, found);
            note(next);
            load_keys();
        }
        wave_lds_fence();
#pragma unroll
        for (uint32_t x = 0; x < 2; ++x)
#pragma unroll
            for (uint32_t st = 0; st < STEPS; ++st) {
                const v8s y = load8(lds_k + (x * 16 + c16) * STRIDE + ((st * 4 + h) ^ (c16 & KTURN)) * 8);
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) s[b][x] = E::mfma16(y, q[b][st], s[b][x]);
            }

        v8s p[NB];
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            if (!whole) {
                const int32_t left = static_cast<int32_t>(limit[b] - j0 - h * 4);
                const uint32_t on = (static_cast<uint32_t>(there) >> (h * 4)) & low_bits(left);
#pragma unroll
                for (uint32_t x = 0; x < 2; ++x)
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) s[b][x][i] = score_if(on, x * 16 + i, s[b][x][i]);
            }
            float top = NEG_INF;
#pragma unroll
            for (uint32_t x = 0; x < 2; ++x)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) top = fmaxf(top, s[b][x][i]);
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (__any((top - m[b]) * c > LAG)) {  // m starts at -inf; NaN where both are
                const float now = fmaxf(m[b], top);
                const float fix = now == NEG_INF ? 1.0f : exp2_fast((m[b] - now) * c);
                m[b] = now;
                l[b] *= fix;
#pragma unroll
                for (uint32_t d = 0; d < BLOCKS; ++d) o[b][d] *= fix;
            }
            const float mc = m[b] == NEG_INF ? 0.0f : base_of<E>(m[b], c);
#pragma unroll
            for (uint32_t x = 0; x < 2; ++x)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float e = exp2_fast(__builtin_fmaf(s[b][x][i], c, -mc));
                    l[b] += e;
                    p[b][x * 4 + i] = static_cast<short>(E::down(e));
                }
        }

        // The values of keys that no row sees count as zeros.
        uint64_t bad = 0;
#pragma unroll
        for (uint32_t i = 0; i < LOADS; ++i) {
            const uint32_t r = i * PER + vrow;
            v8s x = v[i];
            if (!whole) {
                x = zero_unless((there >> r) & 1u, x);
                bad |= __ballot(has_special(x, E::EXP));
                x = without_special(x, E::EXP);
            }
            const uint32_t turn = CHUNKS == 8 ? ((r >> 1) & 3u) << 1 : (r & 7u) << 1;
            *reinterpret_cast<v8s*>(lds + r * STRIDE + (vchunk ^ turn) * 8) = x;
        }
        const int32_t was = slot;
        slot = next;
        if (more) {
            found = find(j0 + 2 * DC_WAVES * DC_KEYS, k1);
            load_values();
        }
        wave_lds_fence();
#pragma unroll
        for (uint32_t d = 0; d < BLOCKS; ++d) {
            const uint32_t r = h * 4 + c16 / 4, chunk = d * 2 + (c16 & 3u) / 2;
            const uint32_t turn = CHUNKS == 8 ? ((r >> 1) & 3u) << 1 : (r & 7u) << 1;
            const uint16_t* at = lds + r * STRIDE + (chunk ^ turn) * 8 + (c16 & 1u) * 4;
            const v8s x = join(lds_tr(at), lds_tr(at + 16 * STRIDE));
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) o[b][d] = E::mfma16(x, p[b], o[b][d]);
        }
        wave_lds_fence();
        if (bad) {
            // Infinite and NaN values, left out above so that rows which do not
            // see their keys are spared, reach the rows that do.
            for (uint32_t j = 0; j < DC_KEYS; ++j) {
                const int32_t at = __shfl(was, static_cast<int>(j), 64);
                if (at < 0) continue;
                const uint16_t* from = a.v + kh * a.v_head + offset_of(at, a.page_lg, a.v_page, a.v_slot);
                uint32_t h4 = h * 4;
                asm volatile("" : "+v"(h4));  // the addresses are worked out here, not kept in registers
#pragma unroll
                for (uint32_t d = 0; d < BLOCKS; ++d) {
                    const uint32_t at_d = d * 16 + h4;
                    const v4s x = load4(from + (at_d < a.dim ? at_d : 0u));
#pragma unroll
                    for (uint32_t b = 0; b < NB; ++b)
                        if (j0 + j < limit[b]) add_special<E>(o[b][d], 0, x);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }

    // The waves' sums meet at their common maximum.
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) {
        l[b] += __shfl_xor(l[b], 16, 64);
        l[b] += __shfl_xor(l[b], 32, 64);
        if (h == 0) {
            s_m[wave][b * 16 + c16] = m[b];
            s_l[wave][b * 16 + c16] = l[b];
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) {
        const uint32_t r = b * 16 + c16;
        float top = NEG_INF;
#pragma unroll
        for (uint32_t w = 0; w < DC_WAVES; ++w) top = fmaxf(top, s_m[w][r]);
        const float fix = l[b] == 0.0f ? 0.0f : exp2_fast((m[b] - top) * c);  // NaN scores stay
        float* red = reinterpret_cast<float*>(s_mem) + (wave * 16 + c16) * RED;
#pragma unroll
        for (uint32_t d = 0; d < BLOCKS; ++d)
            *reinterpret_cast<f32x4*>(red + d * 16 + h * 4) = l[b] == 0.0f ? f32x4{0, 0, 0, 0} : o[b][d] * fix;
        __syncthreads();
        // 256 threads: 16 rows, 16 threads of a row, four dimensions at a time
        const uint32_t mine = threadIdx.x / 16, row = t.row0 + b * 16 + mine;
        float mt = NEG_INF, lt = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < DC_WAVES; ++w) mt = fmaxf(mt, s_m[w][b * 16 + mine]);
#pragma unroll
        for (uint32_t w = 0; w < DC_WAVES; ++w) {
            const float lw = s_l[w][b * 16 + mine];
            lt += lw == 0.0f ? 0.0f : lw * exp2_fast((s_m[w][b * 16 + mine] - mt) * c);
        }
        const bool none = lt == 0.0f;
        const float part = none ? 0.0f : 1.0f / lt;
        if (row < t.rows) {
            const uint32_t token = t.token0 + row / group, head = kh * group + row % group;
            const uint64_t place = place0 + b * 16 + mine;
            const float lse2 = none ? NEG_INF : base_of<E>(mt, c) + __builtin_amdgcn_logf(lt);
#pragma unroll
            for (uint32_t d = (threadIdx.x % 16) * 4; d < DIM; d += 64) {
                f32x4 x = {0, 0, 0, 0};
#pragma unroll
                for (uint32_t w = 0; w < DC_WAVES; ++w)
                    x += *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(s_mem) + (w * 16 + mine) * RED + d);
                if (d < a.dim) store_row(a, E{}, t, place, token, head, d, x * part);
            }
            if (threadIdx.x % 16 == 0) store_lse(a, t, place, token, head, lse2);
        }
        __syncthreads();
    }
}

// ---- many rows: bound by the matrix units --------------------------------------------
// A workgroup answers 128 rows, 32 of them a wave, over tiles of 64 keys that all
// its waves read from LDS, where the next keys and values arrive meanwhile
// without passing through registers.  Scores are transposed products (keys x
// rows) of 32x32x16 matrix instructions; a row's probabilities then lie in the
// lanes that the second product wants them in, if its 16 keys are taken in the
// order 4h..4h+3, 8+4h..8+4h+3 for lane half h, and values are transposed on
// their way out of LDS.  Rows of LDS are turned by pieces of 16 bytes so that
// neither the 32 rows of a key fragment nor the four of a value's share banks.
//
// The products run a tile ahead of the softmax: while the matrix units multiply
// tile i + 1's keys, the wave turns tile i's scores into probabilities, and while
// they multiply those with the values, it takes the maximum of the new scores.
// One workgroup and two waves a SIMD more or less keep the other busy too.
// Up to 192 dimensions (8 requests of 1000 tokens of up to 8192, 24 heads over 8:
// 588 us, 657 TFLOP/s, with one wave a SIMD 950); 256 leave registers for one
// (1540 us, 413).  Of ragged chunks the longest is waited for (8 of up to 1000 tokens
// of up to 8192 keys, of which 0.6 are visible, 96 dimensions: 872 workgroups on 512
// places, which the longest first keep busy 0.8 of the time: 140 us, 640 TFLOP/s).
// 16384 tokens, 32 heads over 8, 128 dimensions, bf16: 2.31 ms, 950 TFLOP/s (a
// large bf16 library product reaches 1206): the matrix units work 45% of the
// cycles, at 2.0 GHz, to which their power brings the clock down from 2.35.  On
// the way: keys and values through registers 2.72 ms; straight to LDS, without
// running ahead 2.36; 64 rows a wave with one wave a SIMD, which halves what is
// read from LDS, 3.2.
constexpr int TL_NT = 256;
// Keys of a tile: 64, or 32 of longer rows: the tile's keys and values and the next
// one's take 64 KB of LDS then, as 64 of up to 128 dimensions do (of up to 64, 32
// KB), and 128 KB would leave no room for a second workgroup.
constexpr uint32_t tile_keys(uint32_t dim) { return dim <= 128 ? 64 : 32; }

// Orders the products of the block before: READS fragments of LDS first, then
// after each product the next one's fragments and a few other
// instructions, which the matrix units cover.
template <uint32_t PRODUCTS, uint32_t READS, uint32_t PER_STEP, uint32_t OTHERS>
__device__ __forceinline__ void between_products()
{
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
    for (uint32_t i = 0; i < PRODUCTS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, PER_STEP, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, OTHERS, 0);
    }
}

template <class E, uint32_t DIM>
__global__ __launch_bounds__(TL_NT) __attribute__((amdgpu_waves_per_eu(DIM <= 192 ? 2 : 1))) void at_tiles(AttnArgs a)
{
    constexpr uint32_t STEPS = DIM / 16, BLOCKS = DIM / 32, CHUNKS = Rows<DIM>::CHUNKS, STRIDE = Rows<DIM>::STRIDE;
    constexpr uint32_t KEYS = tile_keys(DIM), HALVES = KEYS / 32;
    constexpr uint64_t ALL = ~0ull >> (64 - KEYS);
    constexpr uint32_t PER = TL_NT / CHUNKS, LOADS = KEYS / PER;  // rows that the workgroup loads at once, how often
    constexpr uint32_t KTURN = CHUNKS < 16 ? CHUNKS - 1 : 15;
    // separate arrays: what is read is not what is being loaded
    __shared__ alignas(16) uint16_t s_k0[KEYS * STRIDE], s_k1[KEYS * STRIDE];
    __shared__ alignas(16) uint16_t s_v0[KEYS * STRIDE], s_v1[KEYS * STRIDE];
    __shared__ uint64_t s_koff[4][KEYS], s_voff[4][KEYS], s_there[4];
    __shared__ uint32_t s_bad[4], s_most[TL_NT / 64], s_least[TL_NT / 64];
    const uint32_t lane = __lane_id(), wave = threadIdx.x >> 6, c32 = lane & 31u, h = lane >> 5;
    const uint32_t kh = blockIdx.x % a.kv_heads, id = blockIdx.x / a.kv_heads, group = a.heads / a.kv_heads;
    const Work t = find_work<(DIM <= 128), false>(a, id, 128);
    if (t.none) return;
    // The first wave looks up where tiles are: first of all, since what is loaded
    // later is waited for later.
    auto find = [&](uint32_t i, uint32_t end) {
        return look_up(a, t.request, min(t.k0 + i * KEYS + lane % KEYS, end - 1));
    };
    int32_t found[3] = {-1, -1, -1};
    if (wave == 0 && t.k0 < t.k1) {
#pragma unroll
        for (uint32_t i = 0; i < 3; ++i) found[i] = find(i, t.k1);
    }
    const uint32_t row = t.row0 + wave * 32 + c32;  // the lane's
    const uint32_t limit = row < t.rows ? limit_of(a, t, row / group) : 0u;
    uint32_t most, least, wave_most, wave_least;
    if (a.sel) {
        most = limit;
        least = row < t.rows ? limit : 0xFFFFFFFFu;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), o, 64)));
            least = min(least, static_cast<uint32_t>(__shfl_xor(static_cast<int>(least), o, 64)));
        }
        wave_most = __builtin_amdgcn_readfirstlane(most);
        wave_least = __builtin_amdgcn_readfirstlane(least);
        if (lane == 0) {
            s_most[wave] = wave_most;
            s_least[wave] = wave_least;
        }
        __syncthreads();
        most = 0;
        least = 0xFFFFFFFFu;
#pragma unroll
        for (uint32_t w = 0; w < TL_NT / 64; ++w) {
            most = max(most, s_most[w]);
            least = min(least, s_least[w]);
        }
        most = __builtin_amdgcn_readfirstlane(most);
        least = __builtin_amdgcn_readfirstlane(least);
    } else {
        // without a selection they rise with the rows
        const uint32_t w0 = __builtin_amdgcn_readfirstlane(t.row0 + wave * 32), last = t.rows - 1;
        auto at_row = [&](uint32_t r) { return limit_of(a, t, min(r, last) / group); };
        least = at_row(t.row0);
        most = at_row(t.row0 + 127);
        wave_least = w0 < t.rows ? at_row(w0) : 0xFFFFFFFFu;
        wave_most = w0 < t.rows ? at_row(w0 + 31) : 0u;
    }
    const uint32_t k0 = t.k0, k1 = min(most, t.k1);
    const uint64_t place0 = (static_cast<uint64_t>(t.range) * a.kv_heads + kh) * 128;  // of the tile's first row
    if (!t.whole && k0 >= k1) {
        if (threadIdx.x < 128) a.part_lse[place0 + threadIdx.x] = NEG_INF;
        return;
    }

    const Query from(a, t, row, kh);
    v4u q_raw[STEPS];
#pragma unroll
    for (uint32_t st = 0; st < STEPS; ++st) q_raw[st] = from.load(st * 16 + h * 8);
    f32x16 o[BLOCKS];
    float m = NEG_INF, l = 0.0f;
#pragma unroll
    for (uint32_t d = 0; d < BLOCKS; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    const float c = score_scale(a);
    const uint16_t* kp = a.k + kh * a.k_head;
    const uint16_t* vp = a.v + kh * a.v_head;
    const uint32_t lrow = threadIdx.x / CHUNKS, lpos = threadIdx.x % CHUNKS;
    const uint32_t wave_row = __builtin_amdgcn_readfirstlane(wave) * (64 / CHUNKS);

    // The first wave notes where tile i's keys and values are.
    auto note = [&](uint32_t i, int32_t found) {
        const uint32_t at = i % 4, j = k0 + i * KEYS + lane;
        const int32_t slot = lane < KEYS && j < k1 ? slot_of(a, found, j) : -1;
        if (lane < KEYS) {
            s_koff[at][lane] = offset_of(slot, a.page_lg, a.k_page, a.k_slot);
            s_voff[at][lane] = offset_of(slot, a.page_lg, a.v_page, a.v_slot);
        }
        const uint64_t there = __ballot(slot >= 0);
        if (lane == 0) {
            s_there[at] = there;
            s_bad[at] = 0;
        }
    };
    auto v_turn = [](uint32_t r) { return (CHUNKS == 8 ? (r >> 1) & 1u : r & 3u) << 2; };
    // Each lane's 16 bytes go straight to the wave's next 1 KiB of LDS; which of a
    // row's pieces a lane names turns the row.  Pieces behind the head dimension are
    // not loaded: those of keys are zeros, as the queries they meet, and what lies in
    // those of values reaches only columns that are not stored.
    auto load_keys = [&](uint32_t i, uint16_t* sk) {
#pragma unroll
        for (uint32_t x = 0; x < LOADS; ++x) {
            const uint32_t r = x * PER + lrow, d = (lpos ^ (r & KTURN)) * 8;
            if (d < a.dim) load_to_lds(kp + s_koff[i % 4][r] + d, sk + (x * PER + wave_row) * STRIDE);
        }
    };
    auto load_values = [&](uint32_t i, uint16_t* sv) {
#pragma unroll
        for (uint32_t x = 0; x < LOADS; ++x) {
            const uint32_t r = x * PER + lrow, d = (lpos ^ v_turn(r)) * 8;
            if (d < a.dim) load_to_lds(vp + s_voff[i % 4][r] + d, sv + (x * PER + wave_row) * STRIDE);
        }
    };
    // Values of keys that no row sees become zeros, and, in a tile that some rows
    // see and others do not, infinite and NaN ones too.
    auto mend_tile = [&](uint32_t i, uint64_t there, uint16_t* sv) {
        uint64_t bad = 0;
        v8s y[LOADS];
#pragma unroll
        for (uint32_t x = 0; x < LOADS; ++x) {
            const uint32_t r = x * PER + lrow;
            y[x] = zero_unless((there >> r) & 1u, load8(sv + r * STRIDE + lpos * 8));
            bad |= __ballot((lpos ^ v_turn(r)) * 8 < a.dim && has_special(y[x], E::EXP));
        }
        if (there == ALL && !bad) return;
#pragma unroll
        for (uint32_t x = 0; x < LOADS; ++x)
            *reinterpret_cast<v8s*>(sv + (x * PER + lrow) * STRIDE + lpos * 8) = without_special(y[x], E::EXP);
        if (bad && lane == 0) s_bad[i % 4] = 1;
    };

    // Where this lane's fragments begin: keys step by step, values by blocks of 32
    // dimensions (the turn of a row moves a block among four).
    uint32_t v_at[4];
    const uint32_t k_at = c32 * STRIDE + (h ^ (c32 & KTURN)) * 8;  // of step st: k_at ^ st * 16
    {
        const uint32_t i16 = lane & 15u, r = h * 4 + i16 / 4, turn = v_turn(r) / 4;
#pragma unroll
        for (uint32_t d = 0; d < 4; ++d)
            v_at[d] = r * STRIDE + (d ^ turn) * 32 + ((lane >> 4) & 1u) * 16 + (i16 & 3u) * 4;
    }

    if (a.dim < DIM) {
#pragma unroll
        for (uint32_t x = 0; x < LOADS; ++x) {
            const uint32_t r = x * PER + lrow, at = r * STRIDE + lpos * 8;
            if ((lpos ^ (r & KTURN)) * 8 >= a.dim) {
                *reinterpret_cast<v8s*>(s_k0 + at) = v8s{0, 0, 0, 0, 0, 0, 0, 0};
                *reinterpret_cast<v8s*>(s_k1 + at) = v8s{0, 0, 0, 0, 0, 0, 0, 0};
            }
        }
    }
    v8s q[STEPS];
    f32x16 s[HALVES];  // the scores of the tile to come
    float top;
    // Its products, as transposed blocks of 32 keys by 32 rows.
    auto multiply = [&](const uint16_t* sk, f32x16 (&x)[HALVES]) {
#pragma unroll
        for (uint32_t y = 0; y < HALVES; ++y)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[y][e] = 0.0f;
        uint32_t at = k_at;
        // Two waves a SIMD leave 192 dimensions no registers to keep all addresses in.
        if constexpr (DIM == 192) asm volatile("" : "+v"(at));
#pragma unroll
        for (uint32_t y = 0; y < HALVES; ++y)
#pragma unroll
            for (uint32_t st = 0; st < STEPS; ++st) {
                const v8s k = load8(sk + y * 32 * STRIDE + (at ^ (st * 16)));
                x[y] = E::mfma32(k, q[st], x[y]);
            }
    };
    auto hide = [&](uint32_t i) {
        const uint32_t j0 = k0 + i * KEYS;
        const uint64_t there = s_there[i % 4];
        if (there == ALL && j0 + KEYS <= wave_least) return;
        const int32_t left = static_cast<int32_t>(limit - j0 - h * 4);
#pragma unroll
        for (int32_t x = 0; x < static_cast<int32_t>(HALVES); ++x) {
            const uint32_t on = (static_cast<uint32_t>(there >> (x * 32)) >> (h * 4)) & low_bits(left - x * 32);
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e) s[x][e] = score_if(on, (e / 4) * 8 + e % 4, s[x][e]);
        }
    };
    auto highest = [&]() {
        top = NEG_INF;
#pragma unroll
        for (uint32_t x = 0; x < HALVES; ++x)
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e) top = fmaxf(top, s[x][e]);
    };
    auto follow = [&]() {
        const float all = fmaxf(top, __shfl_xor(top, 32, 64));
        if (__any((all - m) * c > LAG)) {  // m starts at -inf; NaN where both are
            const float now = fmaxf(m, all);
            const float fix = now == NEG_INF ? 1.0f : exp2_fast((m - now) * c);
            m = now;
            l *= fix;
#pragma unroll
            for (uint32_t d = 0; d < BLOCKS; ++d) o[d] *= fix;
        }
    };

    const uint32_t n_tiles = k1 > k0 ? (k1 - k0 + KEYS - 1) / KEYS : 0;
    const uint32_t mine = min(n_tiles, wave_most > k0 ? (wave_most - k0 + KEYS - 1) / KEYS : 0u);  // this wave's
    if (n_tiles) {
        if (wave == 0) {
#pragma unroll
            for (uint32_t i = 0; i < 3; ++i) note(i, found[i]);
        }
        __syncthreads();
        load_keys(0, s_k0);
        load_values(0, s_v0);
        if (n_tiles > 1) load_keys(1, s_k1);
#pragma unroll
        for (uint32_t st = 0; st < STEPS; ++st) q[st] = finish_query(a, from.dim, st * 16 + h * 8, q_raw[st]);
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        __syncthreads();
        if (mine) {
            multiply(s_k0, s);
            hide(0);
            highest();
            m = fmaxf(top, __shfl_xor(top, 32, 64));
        }
    }
    // The queries are waited for here, on every way to the loop, or each of its
    // turns would wait for all loads before its first product.
#pragma unroll
    for (uint32_t st = 0; st < STEPS; ++st) asm volatile("" : "+v"(q[st]));
    // Tile i's probabilities and values, while the matrix units turn the next
    // tile's keys into scores; the keys behind those and the next values come in.
    auto tile = [&](uint32_t i, uint16_t* sk, uint16_t* next_k, uint16_t* sv, uint16_t* next_v) {
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's loads to LDS have arrived
        __syncthreads();  // keys i + 1 and values i are there, and nobody reads those before any more
        int32_t ahead = -1;
        if (wave == 0) ahead = find(i + 3, k1);
        if (i + 1 < n_tiles) load_values(i + 1, next_v);
        if (i + 2 < n_tiles) load_keys(i + 2, sk);
        const uint32_t j0 = k0 + i * KEYS;
        const uint64_t there = s_there[i % 4];
        if (!(there == ALL && j0 + KEYS <= least)) {
            mend_tile(i, there, sv);
            __syncthreads();
        }
        if (i < mine) {
            __builtin_amdgcn_sched_barrier(0);
            f32x16 ahead_s[HALVES];
            v8s p[2 * HALVES];
            multiply(next_k, ahead_s);
            const float mc = m == NEG_INF ? 0.0f : base_of<E>(m, c);
#pragma unroll
            for (uint32_t x = 0; x < HALVES; ++x)
#pragma unroll
                for (uint32_t e = 0; e < 16; ++e) {
                    const float y = exp2_fast(__builtin_fmaf(s[x][e], c, -mc));
                    l += y;
                    p[x * 2 + e / 8][e % 8] = static_cast<short>(E::down(y));
                }
            // all of it before the branch, between the products
            asm volatile("" : "+v"(l));
#pragma unroll
            for (uint32_t x = 0; x < 2 * HALVES; ++x) asm volatile("" : "+v"(p[x]));
            between_products<STEPS * HALVES, 3, 1, 6>();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (uint32_t x = 0; x < HALVES; ++x) s[x] = ahead_s[x];
            if (i + 1 < mine) hide(i + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (uint32_t st = 0; st < 2 * HALVES; ++st)
#pragma unroll
                for (uint32_t d = 0; d < BLOCKS; ++d) {
                    const uint16_t* at = sv + st * 16 * STRIDE + d / 4 * 128 + v_at[d % 4];
                    const v8s x = join(lds_tr(at), lds_tr(at + 8 * STRIDE));
                    o[d] = E::mfma32(x, p[st], o[d]);
                }
            highest();
            asm volatile("" : "+v"(top));
            between_products<2 * HALVES * BLOCKS, 6, 2, 2>();
            __builtin_amdgcn_sched_barrier(0);
            if (s_bad[i % 4]) {
                // Infinite and NaN values, left out of LDS so that rows which do
                // not see their keys are spared, reach the rows that do.
                for (uint32_t j = 0; j < KEYS; ++j) {
                    if (!((there >> j) & 1ull)) continue;
                    const uint16_t* from = vp + s_voff[i % 4][j];
                    uint32_t h4 = h * 4;
                    asm volatile("" : "+v"(h4));  // the addresses are worked out here, not kept in registers
#pragma unroll
                    for (uint32_t d = 0; d < BLOCKS; ++d)
#pragma unroll
                        for (uint32_t e = 0; e < 16; e += 4) {
                            const uint32_t at_d = d * 32 + e * 2 + h4;
                            const v4s x = load4(from + (at_d < a.dim ? at_d : 0u));
                            if (j0 + j < limit) add_special<E>(o[d], e, x);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                }
            }
            if (i + 1 < mine) follow();
        }
        if (wave == 0) note(i + 3, ahead);
    };
    for (uint32_t i = 0; i < n_tiles; i += 2) {
        tile(i, s_k0, s_k1, s_v0, s_v1);
        if (i + 1 < n_tiles) tile(i + 1, s_k1, s_k0, s_v1, s_v0);
    }

    const float lt = l + __shfl_xor(l, 32, 64);
    const bool none = lt == 0.0f;
    const float part = none ? 0.0f : 1.0f / lt;
    if (row >= t.rows) return;
    const uint32_t token = t.token0 + row / group, head = kh * group + row % group;
    const uint64_t place = place0 + wave * 32 + c32;
#pragma unroll
    for (uint32_t d = 0; d < BLOCKS; ++d)
#pragma unroll
        for (uint32_t e = 0; e < 16; e += 4) {
            const uint32_t at_d = d * 32 + e * 2 + h * 4;
            const f32x4 x = {o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
            if (at_d < a.dim) store_row(a, E{}, t, place, token, head, at_d, none ? f32x4{0, 0, 0, 0} : x * part);
        }
    if (h == 0) store_lse(a, t, place, token, head, none ? NEG_INF : base_of<E>(m, c) + __builtin_amdgcn_logf(lt));
}

// ---- the ranges' results joined: a workgroup per row -----------------------------------
//   o = sum_r 2^(lse_r - top) o_r / sum_r 2^(lse_r - top),  lse = top + log2(...),
// in fp32, the ranges in a fixed order.  Bound by latency: 3.5 us for 32 rows of a
// context of 1003 keys, 4.6 for 128 rows of 31 ranges each.
constexpr int JN_NT = 256;

template <class E>
__device__ __forceinline__ void store_joined(const AttnArgs& a, E, uint32_t token, uint32_t head, uint32_t d, f32x4 x,
                                             float sum, float top)
{
    const bool none = sum == 0.0f;
    x *= none ? 0.0f : 1.0f / sum;
    if (d < a.dim) {
        const v4s y = {static_cast<short>(E::down(x[0])), static_cast<short>(E::down(x[1])),
                       static_cast<short>(E::down(x[2])), static_cast<short>(E::down(x[3]))};
        *reinterpret_cast<v4s*>(a.out + token * a.out_token + head * a.out_head + d) = y;
    }
    if (a.lse && d == 0)
        a.lse[static_cast<uint64_t>(token) * a.heads + head] =
            none ? NEG_INF : (top + __builtin_amdgcn_logf(sum)) * LN2;
}

// TPR threads take four dimensions each of a range's row, JN_NT / TPR ranges at a time.
template <class E, uint32_t TPR>
__global__ __launch_bounds__(JN_NT) void at_join(AttnArgs a, uint32_t most)
{
    constexpr uint32_t SLOTS = JN_NT / TPR;
    __shared__ float s_o[SLOTS][TPR * 4 + 4], s_sum[SLOTS];
    const uint32_t token = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
    const Joined j = find_joined(a, token, head, most);
    if (j.count == 0) return;  // written already
    float top = NEG_INF;
    for (uint32_t r = __lane_id(); r < j.count; r += 64) top = fmaxf(top, a.part_lse[part_place(a, j, head, most, r)]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const uint32_t slot = threadIdx.x / TPR, d = threadIdx.x % TPR * 4;
    float sum = 0.0f;
    f32x4 x = {0, 0, 0, 0};
#pragma unroll 4
    for (uint32_t r = slot; r < j.count; r += SLOTS) {
        const uint64_t at = part_place(a, j, head, most, r);
        const float lse = a.part_lse[at], w = lse == NEG_INF ? 0.0f : exp2_fast(lse - top);
        sum += w;
        // a range without a visible key has left nothing to read
        if (lse != NEG_INF && d < a.dim) x += w * *reinterpret_cast<const f32x4*>(a.part_o + at * a.dim + d);
    }
    *reinterpret_cast<f32x4*>(&s_o[slot][d]) = x;
    if (threadIdx.x % TPR == 0) s_sum[slot] = sum;
    __syncthreads();
    if (slot == 0) {
#pragma unroll
        for (uint32_t i = 1; i < SLOTS; ++i) {
            x += *reinterpret_cast<const f32x4*>(&s_o[i][d]);
            sum += s_sum[i];
        }
        store_joined(a, E{}, token, head, d, x, sum, top);
    }
}

// The same for many rows: TPR threads a row, one range after another.
template <class E, uint32_t TPR>
__global__ __launch_bounds__(JN_NT) void at_join_rows(AttnArgs a, uint32_t most)
{
    constexpr uint32_t ROWS = 64 / TPR;  // a wave's
    const uint32_t lane = __lane_id(), n = a.n_tokens * a.heads;
    const uint32_t row0 = __builtin_amdgcn_readfirstlane((blockIdx.x * JN_NT + threadIdx.x) / 64 * ROWS);
    if (row0 >= n) return;
    const uint32_t mine = min(row0 + lane / TPR, n - 1), token = mine / a.heads, head = mine % a.heads;
    const uint32_t d = lane % TPR * 4;
    Joined j = {0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < ROWS; ++i) {
        const uint32_t row = min(row0 + i, n - 1);
        const Joined found = find_joined(a, row / a.heads, row % a.heads, most);
        if (lane / TPR == i) j = found;
    }
    if (row0 + lane / TPR >= n || j.count == 0) return;
    float top = NEG_INF, sum = 0.0f;
    for (uint32_t r = 0; r < j.count; ++r) top = fmaxf(top, a.part_lse[part_place(a, j, head, most, r)]);
    f32x4 x = {0, 0, 0, 0};
#pragma unroll 4
    for (uint32_t r = 0; r < j.count; ++r) {
        const uint64_t at = part_place(a, j, head, most, r);
        const float lse = a.part_lse[at], w = lse == NEG_INF ? 0.0f : exp2_fast(lse - top);
        sum += w;
        if (lse != NEG_INF && d < a.dim) x += w * *reinterpret_cast<const f32x4*>(a.part_o + at * a.dim + d);
    }
    store_joined(a, E{}, token, head, d, x, sum, top);
}

template <class E, uint32_t DIM>
int launch_dim(const AttnArgs& a, uint32_t per_wave, uint32_t grid, hipStream_t s)
{
    if (per_wave == 0) {
        CR_TIMED("at_tiles", s);
        at_tiles<E, DIM><<<grid, TL_NT, 0, s>>>(a);
    } else {
        CR_TIMED("at_rows", s);
        if constexpr (DIM <= 128) {
            if (per_wave == 2) {
                at_rows<E, DIM, 2><<<grid, DC_NT, 0, s>>>(a);
                CR_LAUNCH_CHECK();
                return CR_OK;
            }
        }
        at_rows<E, DIM, 1><<<grid, DC_NT, 0, s>>>(a);
    }
    CR_LAUNCH_CHECK();
    return CR_OK;
}

// A workgroup a row where there are few (4 requests of 16 tokens, 2048 rows in
// about 16 ranges each: 24 us in all, 33 with the other; one of 32 rows 15.8 and
// 18.6), several rows a wave where there are many (64 of 8 tokens, 16384 rows: 156
// and 165; 1024 tokens, 32768 rows in two ranges: 48 and 84).
template <class E, uint32_t TPR>
void launch_join(const AttnArgs& a, uint32_t rows, uint32_t most, hipStream_t s)
{
    constexpr uint32_t PER = JN_NT / TPR;
    if (rows > 4096)
        at_join_rows<E, TPR><<<(rows + PER - 1) / PER, JN_NT, 0, s>>>(a, most);
    else
        at_join<E, TPR><<<rows, JN_NT, 0, s>>>(a, most);
}

template <class E>
int launch_attention(const AttnArgs& a, uint32_t per_wave, uint32_t grid, hipStream_t s)
{
    if (a.dim <= 64)
        CR_RET((launch_dim<E, 64>(a, per_wave, grid, s)));
    else if (a.dim <= 96)
        CR_RET((launch_dim<E, 96>(a, per_wave, grid, s)));
    else if (a.dim <= 128)
        CR_RET((launch_dim<E, 128>(a, per_wave, grid, s)));
    else if (a.dim <= 192)
        CR_RET((launch_dim<E, 192>(a, per_wave, grid, s)));
    else
        CR_RET((launch_dim<E, 256>(a, per_wave, grid, s)));
    if (a.share) {
        CR_TIMED("at_join", s);
        const uint32_t rows = a.n_tokens * a.heads, most = per_wave ? 16 * per_wave : 128;
        if (a.dim <= 64)
            launch_join<E, 16>(a, rows, most, s);
        else if (a.dim <= 128)
            launch_join<E, 32>(a, rows, most, s);
        else
            launch_join<E, 64>(a, rows, most, s);
        CR_LAUNCH_CHECK();
    }
    return CR_OK;
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
    // The strides that lead anywhere: that of an axis of one entry may be any number.
    auto over = [](uint32_t extent, uint64_t x, uint64_t y) { return extent > 1 ? x | y : 0; };
    const uint64_t strides = over(p.n_tokens, p.q_token_stride, p.out_token_stride) |
                             over(p.n_heads, p.q_head_stride, p.out_head_stride) |
                             over(cache->n_pages, cache->k_page_stride, cache->v_page_stride) |
                             over(cache->page_size, cache->k_slot_stride, cache->v_slot_stride) |
                             over(cache->n_heads, cache->k_head_stride, cache->v_head_stride) | cache->head_dim;
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
    a.cols = cache->n_pages ? p.table_cols : 0;  // without a page nothing is there to be seen
    a.table_stride = p.table_stride;
    a.sel = p.d_sel;
    a.sel_stride = p.sel_stride;
    a.sel_len = p.d_sel_len;
    a.limits = p.d_limits;
    a.scale = p.scale;
    a.causal = p.causal;
    hipStream_t s = as_stream(stream);

    uint32_t per_wave = 0;
    if (!size_launch(a, room, p.max_new, p.max_kv, num_cus(), &per_wave)) {
        set_error("cr_paged_attention: too many rows for one call");
        return CR_ERR_UNSUPPORTED;
    }
    Scratch sc;
    if (a.share) {
        const uint64_t part_rows = static_cast<uint64_t>(a.n_ranges) * a.kv_heads * (per_wave ? 16 * per_wave : 128);
        Carver cv;
        const size_t o_part = cv.add(part_rows * a.dim * 4), o_lse = cv.add(part_rows * 4);
        const size_t o_at = cv.add(a.n_tiles * 8ull);
        CR_RET(sc.alloc(cv.total, s));
        a.part_o = sc.at<float>(o_part);
        a.part_lse = sc.at<float>(o_lse);
        a.ranges = sc.at<uint2>(o_at);
    }
    const uint32_t grid = a.n_ranges * a.kv_heads;
    if (cache->dtype == CR_F16) return launch_attention<Half>(a, per_wave, grid, s);
    return launch_attention<BHalf>(a, per_wave, grid, s);
}

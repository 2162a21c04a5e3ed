// A Roaring bitmap as the set that a kernel of the serving operators looks ids up
// in.  Included behind internal.hpp.
#pragma once
#include <algorithm>
#include <cstdint>

namespace crimpl {

namespace {

// A set's bits: flat words, or the containers of a bitmap that holds nothing but
// bitmap containers.
struct SetBits {
    const uint32_t* flat;
    const uint16_t* key_index;
    const uint32_t* offsets;
    const uint64_t* bitmaps;
    uint32_t max_key;
    uint32_t flip;  // all bits set where the containers hold the complement
    uint32_t end;   // ids from here on are not in the set

    // Word w of the set (ids [32 w, 32 w + 32), w <= (end - 1) / 32).
    __device__ __forceinline__ uint32_t word(uint32_t w) const
    {
        uint32_t x;
        if (flat) {
            x = flat[w];
        } else {
            const uint32_t key = w / 2048u, c = key <= max_key ? key_index[key] : 0xFFFFu;
            x = c != 0xFFFFu ? reinterpret_cast<const uint32_t*>(bitmaps)[offsets[c] / 4u + w % 2048u] : 0u;
            x ^= flip;
        }
        return w == end / 32u ? x & ((1u << (end % 32u)) - 1u) : x;
    }

    // N words of a set with end > 0, their look-ups side by side.
    template <uint32_t N>
    __device__ __forceinline__ void words(const uint32_t (&w)[N], uint32_t (&x)[N]) const
    {
        if (flat) {
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) x[j] = flat[w[j]];
        } else {
            uint32_t c[N], at[N];
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) c[j] = key_index[min(w[j] / 2048u, max_key)];
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) {
                if (w[j] / 2048u > max_key) c[j] = 0xFFFFu;
                at[j] = offsets[c[j] != 0xFFFFu ? c[j] : 0u];
            }
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) x[j] = reinterpret_cast<const uint32_t*>(bitmaps)[at[j] / 4u + w[j] % 2048u];
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) x[j] = (c[j] != 0xFFFFu ? x[j] : 0u) ^ flip;
        }
#pragma unroll
        for (uint32_t j = 0; j < N; ++j)
            if (w[j] == end / 32u) x[j] &= (1u << (end % 32u)) - 1u;
    }
};

// Bitmap containers are read where they lie; other layouts are written out as
// flat words first.
inline bool is_direct(const cr_gpu_roaring* bm)
{
    return bm->key_index && bm->n_containers > 0 && bm->n_bitmap_containers == bm->n_containers &&
           reinterpret_cast<uintptr_t>(bm->bitmap_data) % 16 == 0;
}

// The bits of `bm` below `end`; `words` has room for n_words where they are written out.
inline int set_bits(const cr_gpu_roaring* bm, bool direct, uint32_t* words, uint32_t n_words, uint32_t end, cr_stream_t stream,
             SetBits* out)
{
    out->end = end;
    if (!direct) {
        out->flat = words;
        return cr_decompress_to_bitset(bm, words, n_words, stream);
    }
    out->key_index = bm->key_index;
    out->offsets = bm->offsets;
    out->bitmaps = bm->bitmap_data;
    out->max_key = bm->max_key;
    if (bm->negated) {
        out->flip = 0xFFFFFFFFu;
        out->end = std::min(end, bm->universe_size);
    }
    return CR_OK;
}

inline bool power_of_two(uint32_t x) { return x && (x & (x - 1)) == 0; }

}  // namespace

}  // namespace crimpl

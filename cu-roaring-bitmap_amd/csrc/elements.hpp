// The element types of the serving operators' tensors as floats, and the values that
// one load or store moves.
#pragma once
#include <cstdint>

namespace crimpl {

namespace {

struct F32 {
    typedef uint32_t Bits;
    static __device__ __forceinline__ float up(uint32_t x) { return __uint_as_float(x); }
    static __device__ __forceinline__ uint32_t down(float x) { return __float_as_uint(x); }
};
// Rounded to nearest even.
struct F16 {
    typedef uint16_t Bits;
    static __device__ __forceinline__ float up(uint16_t x)
    {
        return static_cast<float>(__builtin_bit_cast(_Float16, x));
    }
    static __device__ __forceinline__ uint16_t down(float x)
    {
        return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
    }
};
struct BF16 {
    typedef uint16_t Bits;
    static __device__ __forceinline__ float up(uint16_t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }
    static __device__ __forceinline__ uint16_t down(float x)
    {
        return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
    }
};

// N values side by side, aligned as a whole.
template <class E, uint32_t N>
struct Piece {
    typedef typename E::Bits V __attribute__((ext_vector_type(N)));
    V x;
    static __device__ __forceinline__ Piece load(const typename E::Bits* p)
    {
        return {__builtin_nontemporal_load(reinterpret_cast<const V*>(p))};
    }
    __device__ __forceinline__ void store(typename E::Bits* p) const
    {
        __builtin_nontemporal_store(x, reinterpret_cast<V*>(p));
    }
    __device__ __forceinline__ float get(uint32_t i) const { return E::up(x[i]); }
    __device__ __forceinline__ void set(uint32_t i, float v) { x[i] = E::down(v); }
};
template <class E>
struct Piece<E, 1> {
    typename E::Bits x;
    static __device__ __forceinline__ Piece load(const typename E::Bits* p) { return {__builtin_nontemporal_load(p)}; }
    __device__ __forceinline__ void store(typename E::Bits* p) const { __builtin_nontemporal_store(x, p); }
    __device__ __forceinline__ float get(uint32_t) const { return E::up(x); }
    __device__ __forceinline__ void set(uint32_t, float v) { x = E::down(v); }
};

}  // namespace

}  // namespace crimpl

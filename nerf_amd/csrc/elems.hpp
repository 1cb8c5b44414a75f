// Element types of the operators that take bf16, fp16 or fp32 tensors: 16-byte (or single-element) loads and stores
// with arithmetic in fp32, rounded once to the nearest element value at the store.
#pragma once
#include "common.hpp"

namespace nerf {

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, V>*>(p);
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& x) {
    *reinterpret_cast<Pack<T, V>*>(p) = x;
}

// The same at any address that the elements themselves are aligned to (memory instructions ask for no more); a row of `cols`
// elements is then covered whatever its length by pieces that begin at min(c, cols - V): the last one repeats some columns.
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_any(const T* p) {
    return __builtin_bit_cast(Pack<T, V>, *reinterpret_cast<const Loose<T, V>*>(p));
}
template <typename T, int V>
__device__ __forceinline__ void store_any(T* p, const Pack<T, V>& x) {
    *reinterpret_cast<Loose<T, V>*>(p) = __builtin_bit_cast(Loose<T, V>, x);
}

// elements of a 16-byte access
template <typename T>
constexpr int full_vec() { return 16 / (int)sizeof(T); }

static inline int elem_bytes(int precision) { return precision == NERF_PREC_FP32 ? 4 : 2; }
static inline bool elem_ok(int precision) {
    return precision == NERF_PREC_BF16 || precision == NERF_PREC_FP16 || precision == NERF_PREC_FP32;
}

}  // namespace nerf

// CALL(T) for the element type that `precision` names
#define NERF_ELEM_DISPATCH(precision, CALL)              \
    do {                                                 \
        if ((precision) == NERF_PREC_BF16) CALL(__bf16); \
        else if ((precision) == NERF_PREC_FP16) CALL(_Float16); \
        else CALL(float);                                \
    } while (0)

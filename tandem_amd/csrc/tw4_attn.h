// What the kernels around the paged cache share: the two 16-bit types, their matrix instructions, and page sizes.
//
// Cache: keys and values each [pages, KV heads, page size, head_dim] (any strides of pages, heads and tokens). Slot
// s = page * page_size + offset. A page size is a power of two from 16 on, so the 16 keys of a matrix instruction's tile
// lie in one page.
#pragma once

#include "tw4_common.h"

namespace tw4 {

typedef __bf16 bf1;
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

template <typename T>
struct Vec8;
template <>
struct Vec8<h1> {
    typedef h8 type;
};
template <>
struct Vec8<bf1> {
    typedef bf8 type;
};

// 8 values of a 16-byte chunk as fp32, and back (nearest even).
template <typename T>
__device__ __forceinline__ void to_f32(const u4& v, float (&f)[8]) {
    const auto x = bitcast<typename Vec8<T>::type>(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(x[i]);
}
template <typename T>
__device__ __forceinline__ u4 from_f32(const float (&f)[8]) {
    typename Vec8<T>::type x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<T>(f[i]);
    return bitcast<u4>(x);
}

template <typename T>
__device__ __forceinline__ f4 mma16(const u4& a, const u4& b, const f4& c) {
    if constexpr (__is_same(T, h1))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<h8>(a), bitcast<h8>(b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bitcast<bf8>(a), bitcast<bf8>(b), c, 0, 0, 0);
}

// log2 of a page size the kernels take, else -1.
inline int page_shift(int page_size) {
    for (int s = 4; s <= 8; ++s)
        if (page_size == 1 << s) return s;
    return -1;
}

}  // namespace tw4

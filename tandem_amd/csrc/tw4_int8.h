// What the operators on 8-bit integers share: the two 16-bit types activations come in, and the epilogue of the products.
#pragma once

#include "tw4_common.h"

namespace tw4 {

typedef int i4 __attribute__((ext_vector_type(4)));

// 8 values of a 16-byte chunk as fp32, and fp32 to one value (to nearest even), by type.
template <bool BF16>
__device__ __forceinline__ void chunk_values(const u4& v, float (&f)[8]) {
    if constexpr (BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = bitcast<float>(v[i] << 16);
            f[2 * i + 1] = bitcast<float>(v[i] & 0xFFFF0000u);
        }
    } else {
        chunk_to_f32(v, f);
    }
}

template <bool BF16>
__device__ __forceinline__ uint32_t value16(float f) {
    if constexpr (BF16)
        return bitcast<uint16_t>(static_cast<__bf16>(f));
    else
        return bitcast<uint16_t>(static_cast<h1>(f));
}

template <bool BF16>
__device__ __forceinline__ u4 values_chunk(const float (&f)[8]) {
    u4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = value16<BF16>(f[2 * i]) | value16<BF16>(f[2 * i + 1]) << 16;
    return v;
}

// D += A B on v_mfma_i32_16x16x64_i8: lane (q, r) = (lane / 16, lane % 16) gives row r of A and column r of B, 16 bytes each, at
// the same 16 of the 64 k for both, and holds rows 4 q + i of column r of D. The sums are exact (K < 2^17).
__device__ __forceinline__ i4 mfma_i8(const u4& a, const u4& b, const i4& c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(bitcast<i4>(a), bitcast<i4>(b), c, 0, 0, 0);
}

// Output features n .. n + 3 of one token: sums times both scales, rounded once. wide: N % 4 == 0 and y 8-byte aligned, so that the
// four lie in the row together.
template <bool BF16>
__device__ __forceinline__ void store_features(uint16_t* row, int n, int N, bool wide, const float (&v)[4]) {
    if (wide) {
        if (n < N)
            *reinterpret_cast<u2*>(row + n) =
                u2{value16<BF16>(v[0]) | value16<BF16>(v[1]) << 16, value16<BF16>(v[2]) | value16<BF16>(v[3]) << 16};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < N) row[n + i] = static_cast<uint16_t>(value16<BF16>(v[i]));
    }
}

}  // namespace tw4

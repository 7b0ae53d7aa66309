// What the operators on 8-bit integers share: the two 16-bit types activations come in, SwiGLU, the matrix instruction, the host's look at overlapping
// memory, and the products' arguments and tiles.
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

// The float32 is rounded before it is made a 16-bit value, in every kernel alike: left to itself the compiler folds the last product into
// the conversion (v_fma_mixlo_f16, one rounding) in some of them, and a result would depend on the kernel that a batch takes.
template <bool BF16>
__device__ __forceinline__ uint32_t value16(float f) {
    asm("" : "+v"(f));
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

// g / (1 + exp(-g)) by the reciprocal instruction (1 ulp), for g >= kSiluFar or NaN: a division takes ten instructions. K 4096 x N 24576:
// M = 512 57.3 -> 55.9 us, 2048 191 -> 185; level at 8192, which the card's power bounds.
__device__ __forceinline__ float silu_rcp(float g) { return g * __builtin_amdgcn_rcpf(1.0f + __expf(-g)); }

// Below kSiluFar exp(-g) comes to pass 2^126, whose reciprocal that instruction flushes to 0, and float32 later on. 1 + exp(-g) is exp(-g)
// there, and g exp(g) = (g exp(g / 2)) exp(g / 2) meets subnormal numbers in its last product only.
constexpr float kSiluFar = -87.0f;
__device__ __forceinline__ float silu_far(float g) {
    const float e = __expf(0.5f * g);
    return g * e * e;
}

// g[i] becomes silu(g[i]). Gates that far out are few or none: a wavefront without one jumps over their form (the look costs K 2560 x N
// 19456 at M = 200 0.3 us, 18.1 -> 18.4; M = 5 and 8192 are level).
template <int N>
__device__ __forceinline__ void silu_values(float (&g)[N]) {
    float least = g[0], s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) least = fminf(least, g[i]), s[i] = silu_rcp(g[i]);
    if (__builtin_expect(__ballot(least < kSiluFar) != 0, 0)) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (g[i] < kSiluFar) s[i] = silu_far(g[i]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = s[i];
}

// D += A B on v_mfma_i32_16x16x64_i8: lane (q, r) = (lane / 16, lane % 16) gives row r of A and column r of B, 16 bytes each, at
// the same 16 of the 64 k for both, and holds rows 4 q + i of column r of D. The sums are exact (K < 2^17).
__device__ __forceinline__ i4 mfma_i8(const u4& a, const u4& b, const i4& c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(bitcast<i4>(a), bitcast<i4>(b), c, 0, 0, 0);
}

// Whether so many bytes from a and from b on are apart (host).
inline bool bytes_apart(const void* a, int64_t bytes_a, const void* b, int64_t bytes_b) {
    return static_cast<const char*>(a) + bytes_a <= b || static_cast<const char*>(b) + bytes_b <= a;
}

// Whether rows of `width` bytes from a and b on, so many bytes apart, share no byte (host).
inline bool rows_apart(const void* a, int64_t step_a, const void* b, int64_t step_b, int64_t rows, int64_t width) {
    if (bytes_apart(a, (rows - 1) * step_a + width, b, (rows - 1) * step_b + width)) return true;
    const int64_t off = static_cast<const char*>(b) - static_cast<const char*>(a);
    const int64_t at = (off < 0 ? -off : off) % step_a;  // one's rows may lie between the other's, where both are as far apart
    return step_a == step_b && width <= at && at <= step_a - width;
}

struct Gemm8Args {
    const int8_t* x;
    int64_t x_stride;
    const float* x_scale;
    const int8_t* w;
    int64_t w_stride;
    const float* w_scale;
    uint16_t* y;
    int M, N, K, act, bf16;
    int *ws, *locks;  // splits > 1: partial sums and counters, as many as these
    int64_t ws_words, n_locks;
    hipStream_t st;
};

// The tiles of tw4_gemm8_lds.hip: kernel number, 16-token tiles and 16-row tiles of a wavefront, wavefronts along tokens and rows, slots
// of the ring. Kernel 0 is the streaming one of tw4_gemm8.hip.
#define TW4_GEMM8_LDS(X)                                                                                             \
    X(1, 1, 2, 1, 2, 7) X(2, 1, 2, 1, 2, 3) X(3, 1, 2, 2, 2, 5) X(4, 2, 2, 2, 2, 5) X(5, 2, 2, 2, 4, 6) X(6, 4, 2, 2, 4, 3) \
    X(7, 6, 2, 2, 2, 3) X(8, 4, 6, 2, 2, 2) X(9, 6, 4, 2, 2, 2) X(10, 4, 4, 2, 4, 3) X(11, 4, 4, 4, 2, 3) X(12, 8, 4, 2, 4, 2)
#define TW4_COUNT(...) +1
constexpr int kGemm8Kernels = 1 TW4_GEMM8_LDS(TW4_COUNT);
#undef TW4_COUNT
static_assert(kGemm8Kernels == TW4_GEMM_INT8_KERNELS, "the header's count");

int gemm8_stream(const Gemm8Args& a, int rows);             // tw4_gemm8.hip
int gemm8_lds(const Gemm8Args& a, int kernel, int splits);  // tw4_gemm8_lds.hip

}  // namespace tw4

// y[M, N] = x_scale[m] w_scale[n] sum_k x[m, k] w[n, k] of 8-bit integers, the sum exact in 32 bits, one rounding; or, with
// act, y[M, N / 2] = silu(g) u of the rows w = [gate | up], g and u unrounded.
//
// A workgroup of WK wavefronts takes 16 NT rows of w (with act half of them gate rows, half their up rows) and 16 MT tokens. Each
// wavefront covers a range of K in steps of 64 k, reading the fragments of both operands where they lie (16 rows of 64 bytes); the
// wavefronts' sums are added in LDS.
#include "tw4_int8.h"

namespace tw4 {

template <bool ACT, bool BF16, int MT, int NT, int WK>
__global__ void __launch_bounds__(64 * WK) gemm8_stream_kernel(const int8_t* __restrict__ x, int64_t x_stride,
                                                               const float* __restrict__ x_scale, const int8_t* __restrict__ w,
                                                               int64_t w_stride, const float* __restrict__ w_scale,
                                                               uint16_t* __restrict__ y, int M, int N, int K) {
    static_assert(!ACT || NT % 2 == 0, "gate and up tiles in pairs");
    constexpr int TILES = ACT ? NT / 2 : NT;  // output tiles
    __shared__ i4 part[WK][NT * MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int out = ACT ? N >> 1 : N;
    const int n0 = 16 * TILES * blockIdx.x, m0 = 16 * MT * blockIdx.y;
    const int8_t *wp[NT], *xp[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int n = min(n0 + 16 * (t % TILES) + r, out - 1) + (t >= TILES ? out : 0);  // rows past the end: the last one, not stored
        wp[t] = w + n * w_stride;
    }
#pragma unroll
    for (int b = 0; b < MT; ++b) xp[b] = x + min(m0 + 16 * b + r, M - 1) * x_stride;
    i4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < MT; ++b) acc[t][b] = i4{0, 0, 0, 0};
    const int units = (K + 63) >> 6, first = wave * units / WK, last = (wave + 1) * units / WK;
    for (int i = first; i < last; ++i) {
        const int k = 64 * i + 16 * q;
        const bool in = k < K;  // K % 16 == 0: a lane's 16 bytes are inside or not
        u4 a[NT], b[MT];
#pragma unroll
        for (int t = 0; t < NT; ++t) a[t] = in ? *reinterpret_cast<const u4*>(wp[t] + k) : u4{0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < MT; ++m) b[m] = in ? *reinterpret_cast<const u4*>(xp[m] + k) : u4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[t][m] = mfma_i8(a[t], b[m], acc[t][m]);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) part[wave][t * MT + m][lane] = acc[t][m];
    __syncthreads();
    const bool wide = (out & 3) == 0 && (reinterpret_cast<uintptr_t>(y) & 7) == 0;
    for (int f = wave; f < TILES * MT; f += WK) {
        const int t = f / MT, m = m0 + 16 * (f % MT) + r, n = n0 + 16 * t + 4 * q;
        i4 a{0, 0, 0, 0}, u{0, 0, 0, 0};
#pragma unroll
        for (int v = 0; v < WK; ++v) {
            a += part[v][f][lane];
            if constexpr (ACT) u += part[v][f + TILES * MT][lane];
        }
        if (m >= M) continue;
        const float xs = x_scale[m];
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = min(n + i, out - 1);
            o[i] = static_cast<float>(a[i]) * xs * w_scale[at];
            if constexpr (ACT) o[i] = silu(o[i]) * (static_cast<float>(u[i]) * xs * w_scale[out + at]);
        }
        store_features<BF16>(y + static_cast<int64_t>(m) * out, n, out, wide, o);
    }
}

}  // namespace tw4

using namespace tw4;

extern "C" int tw4_gemm_int8(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride,
                             const float* w_scale, uint16_t* y, int M, int N, int K, int act, int bf16, void* stream) {
    TW4_REQUIRE(x && x_scale && w && w_scale && y, TW4_EINVAL, "gemm_int8: null pointer");
    TW4_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0, TW4_EINVAL,
                "gemm_int8: rows must be 16-byte aligned");
    TW4_REQUIRE(reinterpret_cast<uintptr_t>(x_scale) % 4 == 0 && reinterpret_cast<uintptr_t>(w_scale) % 4 == 0 &&
                    reinterpret_cast<uintptr_t>(y) % 2 == 0,
                TW4_EINVAL, "gemm_int8: scales must be 4-byte aligned and y 2-byte");
    TW4_REQUIRE(M >= 0 && M <= 1 << 20, TW4_EINVAL, "gemm_int8: 0 <= M <= 2^20 (M = %d)", M);
    TW4_REQUIRE(N >= 1 && N <= 1 << 24, TW4_EINVAL, "gemm_int8: 1 <= N <= 2^24 (N = %d)", N);
    TW4_REQUIRE(K >= 16 && K % 16 == 0 && K < 1 << 17, TW4_EINVAL, "gemm_int8: K %% 16 == 0 and 16 <= K < 2^17 (K = %d)", K);
    TW4_REQUIRE(x_stride >= K && x_stride % 16 == 0 && w_stride >= K && w_stride % 16 == 0 && x_stride < 1 << 22 && w_stride < 1 << 22,
                TW4_EINVAL, "gemm_int8: rows at least K and less than 2^22 apart, 16-byte aligned (strides %lld, %lld)",
                static_cast<long long>(x_stride), static_cast<long long>(w_stride));
    TW4_REQUIRE(act == 0 || (act == 1 && N % 2 == 0), TW4_EINVAL, "gemm_int8: act 0, or 1 (SwiGLU) with an even N (act %d, N %d)", act, N);
    if (M == 0) return TW4_OK;
    const int out = act ? N / 2 : N;
    const dim3 grid(static_cast<unsigned>((out + 15) / 16), static_cast<unsigned>((M + 63) / 64));
    auto st = static_cast<hipStream_t>(stream);
#define TW4_GO(ACT, BF16, NT) \
    gemm8_stream_kernel<ACT, BF16, 4, NT, 4><<<grid, 256, 0, st>>>(x, x_stride, x_scale, w, w_stride, w_scale, y, M, N, K)
    if (act && bf16) TW4_GO(true, true, 2);
    else if (act) TW4_GO(true, false, 2);
    else if (bf16) TW4_GO(false, true, 1);
    else TW4_GO(false, false, 1);
#undef TW4_GO
    TW4_LAUNCH_CHECK("gemm_int8: launch");
    return TW4_OK;
}

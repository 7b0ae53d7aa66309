// Rows of activations in 8-bit integers with a scale for each row, alone and behind the decoder layer's add + RMSNorm:
//
//   tw4_quantize_int8:   t = x,       scale = max|t| / 127
//   tw4_rms_norm_int8:   t = s w,     scale = max|t| rstd / 127,  s = x (+ r, fp32; r <- round(s)), rstd = rsqrt(mean(s^2) + eps)
//   both:                code = 127 t / max|t| rounded to nearest, halves to even
//
// rstd is common to a row, so it leaves the codes: they depend on t alone, whose values 64-bit floats hold exactly (24 + 11
// bits), and come out exactly rounded.
#include "tw4_int8.h"

namespace tw4 {

constexpr float kLeast = 0x1p-100f;  // rows whose largest magnitude is below it count as zeros: 127 / max stays finite

template <bool NORM, bool ADD, bool BF16, int T, int J>
__global__ void __launch_bounds__(T) rows_int8_kernel(const u4* __restrict__ x, int64_t x_step, u4* __restrict__ r, int64_t r_step,
                                                      const u4* __restrict__ w, float eps, u2* __restrict__ codes,
                                                      float* __restrict__ scales, int chunks) {
    __shared__ double top_of[T / 64];
    __shared__ float sum_of[T / 64], bad_of[T / 64];
    const int tid = threadIdx.x, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const u4* xr = x + row * x_step;
    u4* rr = r + row * r_step;
    float s[J][8], g[J][8];
    float sum = 0.0f, bad = 0.0f;
    double top = 0.0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int c = T * j + tid;
        u4 xv{}, rv{}, wv{};
        if (c < chunks) {
            xv = xr[c];
            if constexpr (ADD) rv = rr[c];
            if constexpr (NORM) wv = w[c];
        }
        chunk_values<BF16>(xv, s[j]);
        if constexpr (ADD) {
            float b[8];
            chunk_values<BF16>(rv, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[j][i] += b[i];
            if (c < chunks) rr[c] = values_chunk<BF16>(s[j]);
        }
        if constexpr (NORM) chunk_values<BF16>(wv, g[j]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double t = static_cast<double>(s[j][i]) * (NORM ? static_cast<double>(g[j][i]) : 1.0);
            sum = __builtin_fmaf(s[j][i], s[j][i], sum);
            bad = __builtin_fmaf(static_cast<float>(t), 0.0f, bad);  // NaN from the first infinity or NaN on
            top = fmax(top, fabs(t));
        }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        top = fmax(top, __shfl_xor(top, o));
        sum += __shfl_xor(sum, o);
        bad += __shfl_xor(bad, o);
    }
    if ((tid & 63) == 0) top_of[wave] = top, sum_of[wave] = sum, bad_of[wave] = bad;
    __syncthreads();
    sum = 0.0f, bad = 0.0f;
#pragma unroll
    for (int v = 0; v < T / 64; ++v) {
        top = fmax(top, top_of[v]);
        sum += sum_of[v];
        bad += bad_of[v];
    }
    const bool none = !(top >= static_cast<double>(kLeast)) || bad != 0.0f;
    if (tid == 0) {
        const float rstd = NORM ? rsqrtf(sum / static_cast<float>(8 * chunks) + eps) : 1.0f;
        const float scale = static_cast<float>(top) * rstd / 127.0f;
        scales[row] = bad != 0.0f ? __builtin_nanf("") : none ? 0.0f : scale;
    }
    u2* out = codes + row * chunks;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int c = T * j + tid;
        if (c >= chunks) continue;
        uint32_t q[2] = {0, 0};
        if (!none) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double t = static_cast<double>(s[j][i]) * (NORM ? static_cast<double>(g[j][i]) : 1.0);
                const int code = static_cast<int>(rint(127.0 * t / top));
                q[i >> 2] |= (static_cast<uint32_t>(code) & 0xFFu) << 8 * (i & 3);
            }
        }
        out[c] = u2{q[0], q[1]};
    }
}

struct RowsArgs {
    const u4* x;
    int64_t x_step;
    u4* r;
    int64_t r_step;
    const u4* w;
    float eps;
    u2* codes;
    float* scales;
    int M, chunks;
    hipStream_t st;
};

template <bool NORM, bool ADD, bool BF16, int T, int J>
void rows_go(const RowsArgs& a) {
    rows_int8_kernel<NORM, ADD, BF16, T, J><<<static_cast<unsigned>(a.M), T, 0, a.st>>>(a.x, a.x_step, a.r, a.r_step, a.w, a.eps,
                                                                                       a.codes, a.scales, a.chunks);
}

template <bool NORM, bool ADD, bool BF16>
int rows_launch(const RowsArgs& a, const char* who) {
    if (a.chunks <= 64)
        rows_go<NORM, ADD, BF16, 64, 1>(a);
    else if (a.chunks <= 256)
        rows_go<NORM, ADD, BF16, 256, 1>(a);
    else if (a.chunks <= 512)
        rows_go<NORM, ADD, BF16, 256, 2>(a);
    else if (a.chunks <= 1024)
        rows_go<NORM, ADD, BF16, 512, 2>(a);
    else if (a.chunks <= 2048)
        rows_go<NORM, ADD, BF16, 1024, 2>(a);
    else
        rows_go<NORM, ADD, BF16, 1024, 4>(a);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? TW4_OK : tw4host::hip_fail(e, who);
}

int rows_check(const void* x, int64_t x_stride, const void* codes, const void* scales, int M, int K, const char* who) {
    TW4_REQUIRE(x && codes && scales, TW4_EINVAL, "%s: null pointer", who);
    TW4_REQUIRE(K >= 16 && K % 16 == 0 && K <= TW4_ROWS8_MAX, TW4_EINVAL, "%s: K %% 16 == 0 and 16 <= K <= %d (K = %d)", who,
                TW4_ROWS8_MAX, K);
    TW4_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(scales) % 4 == 0,
                TW4_EINVAL, "%s: rows must be 16-byte aligned, scales 4-byte", who);
    TW4_REQUIRE(M >= 0, TW4_EINVAL, "%s: M >= 0 (M = %d)", who, M);
    TW4_REQUIRE(x_stride >= K && x_stride % 8 == 0, TW4_EINVAL, "%s: rows at least K apart, 16-byte aligned (stride %lld)", who,
                static_cast<long long>(x_stride));
    return TW4_OK;
}

}  // namespace tw4

using namespace tw4;

extern "C" int tw4_quantize_int8(const uint16_t* x, int64_t x_stride, int8_t* codes, float* scales, int M, int K, int bf16,
                                 void* stream) {
    int rc = rows_check(x, x_stride, codes, scales, M, K, "quantize_int8");
    if (rc || M == 0) return rc;
    const RowsArgs a{reinterpret_cast<const u4*>(x), x_stride / 8, nullptr, 0, nullptr, 0.0f, reinterpret_cast<u2*>(codes), scales, M,
                     K / 8, static_cast<hipStream_t>(stream)};
    return bf16 ? rows_launch<false, false, true>(a, "quantize_int8: launch") : rows_launch<false, false, false>(a, "quantize_int8: launch");
}

extern "C" int tw4_rms_norm_int8(const uint16_t* x, int64_t x_stride, uint16_t* residual, int64_t r_stride, const uint16_t* weight,
                                 float eps, int8_t* codes, float* scales, int M, int K, int bf16, void* stream) {
    const char* who = "rms_norm_int8";
    int rc = rows_check(x, x_stride, codes, scales, M, K, who);
    if (rc) return rc;
    TW4_REQUIRE(weight && reinterpret_cast<uintptr_t>(weight) % 16 == 0, TW4_EINVAL, "%s: weight must be 16-byte aligned and not null", who);
    if (residual)
        TW4_REQUIRE(reinterpret_cast<uintptr_t>(residual) % 16 == 0 && r_stride >= K && r_stride % 8 == 0, TW4_EINVAL,
                    "%s: residual rows at least K apart, 16-byte aligned (stride %lld)", who, static_cast<long long>(r_stride));
    if (M == 0) return TW4_OK;
    const RowsArgs a{reinterpret_cast<const u4*>(x), x_stride / 8, reinterpret_cast<u4*>(residual), r_stride / 8,
                     reinterpret_cast<const u4*>(weight), eps, reinterpret_cast<u2*>(codes), scales, M, K / 8,
                     static_cast<hipStream_t>(stream)};
    if (residual) return bf16 ? rows_launch<true, true, true>(a, "rms_norm_int8: launch") : rows_launch<true, true, false>(a, "rms_norm_int8: launch");
    return bf16 ? rows_launch<true, false, true>(a, "rms_norm_int8: launch") : rows_launch<true, false, false>(a, "rms_norm_int8: launch");
}

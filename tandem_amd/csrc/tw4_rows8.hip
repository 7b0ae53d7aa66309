// Rows of activations in 8-bit integers with a scale for each row, alone and behind the decoder layer's add + RMSNorm:
//
//   tw4_quantize_int8:   t = x,       scale = max|t| / 127
//   tw4_rms_norm_int8:   t = s w,     scale = max|t| rstd / 127,  s = x (+ r, fp32; r <- round(s)), rstd = rsqrt(mean(s^2) + eps)
//   both:                code = 127 t / max|t| rounded to nearest, halves to even
//
// rstd is common to a row, so it leaves the codes: they depend on t alone, whose values 64-bit floats hold exactly (24 + 11
// bits), and come out exactly rounded. 32 bits decide nearly all of them: r = fl(t) fl(127 / fl(max|t|)) is within 4 roundings, 127
// 2^-22 = 3.03e-5, of 127 t / max|t|; only where r is nearer than that to a border between two codes (one value in 16000, and exact
// ties) the comparison of 254 |t| with (2 c + 1) max|t| is made, whose sides 64 bits hold exactly.
//
// A workgroup per row, W wavefronts of J chunks per lane (8 values, 16 bytes), all loaded before any math and kept for the second
// pass.
// Bounds. Few rows: the launch (1.8 us) and two round trips to memory: K 4096, M = 1 2.3 us, with add + norm 2.8; wavefronts of one
// chunk each are fastest (K 5120, M = 40, add + norm: 8 of 2 chunks 3.7, 4 of 3 3.8, 16 of 2 4.4). Many rows: memory, at a copy's 5.15 TB/s
// or above, with fewer wavefronts of more chunks: us at M = 8192, K 4096: quantised 19.3 (5.2 TB/s), norm 21.3 (4.7), add + norm 42.7
// (5.5), in 4 wavefronts of 2; 8 of 1 22.3, 26.7, 42.2; 2 of 4 21.1, 21.8, 44.0. M = 4096, K 12288: 27.9, 32.6, 69 in 8 of 3; 16 of 2 27.5,
// 55, 82. Dividing every value in 64 bits took 54 us where 27.9 are now (M = 4096, K 12288, quantised). Four rows per
// workgroup, a wavefront each, were slower than one at every width (K 512, M = 16384, add + norm 13.9 against 13.4).
#include "tw4_rows8.h"

namespace tw4 {

template <bool NORM, bool ADD, bool BF16, int W, int J>
__global__ void __launch_bounds__(64 * W) rows_int8_kernel(const u4* __restrict__ x, int64_t x_step, u4* __restrict__ r,
                                                           int64_t r_step, const u4* __restrict__ w, float eps,
                                                           u2* __restrict__ codes, float* __restrict__ scales, int chunks) {
    __shared__ Row8Shared<NORM, W, J> shared;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x;
    Row8Loads<J> loads;
    row8_load<NORM, ADD, W, J>(loads, x + row * x_step, r + row * r_step, w, chunks, wave, lane);
    row8_quantize<NORM, ADD, BF16, W, J>(loads, shared, r + row * r_step, codes + row * chunks, scales + row, eps, chunks, wave, lane);
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

template <bool NORM, bool ADD, bool BF16, int W, int J>
int rows_go(const RowsArgs& a) {
    TW4_REQUIRE(a.M * (64LL * W) < 1LL << 32, TW4_EINVAL, "%s: M = %d is too many rows of %d", NORM ? "rms_norm_int8" : "quantize_int8", a.M, 8 * a.chunks);
    if constexpr (ADD)  // rows are read and written by different workgroups at once
        TW4_REQUIRE(rows_apart(a.x, 16 * a.x_step, a.r, 16 * a.r_step, a.M, 16LL * a.chunks), TW4_EINVAL,
                    "rms_norm_int8: the residual needs memory of its own");
    rows_int8_kernel<NORM, ADD, BF16, W, J>
        <<<static_cast<unsigned>(a.M), 64 * W, 0, a.st>>>(a.x, a.x_step, a.r, a.r_step, a.w, a.eps, a.codes, a.scales, a.chunks);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? TW4_OK : tw4host::hip_fail(e, NORM ? "rms_norm_int8: launch" : "quantize_int8: launch");
}

// Few rows: one chunk per lane, as far as 8 wavefronts go; many: two or three, and fewer wavefronts (both sides above).
constexpr int kManyShort = 1024, kMany = 256;

template <bool NORM, bool ADD, bool BF16>
int rows_launch(const RowsArgs& a) {
    const int need = (a.chunks + 63) / 64;  // chunks of all wavefronts' lanes
    if (need <= 1) return rows_go<NORM, ADD, BF16, 1, 1>(a);
    if (need <= 2) return rows_go<NORM, ADD, BF16, 2, 1>(a);
    if (need <= 4) return a.M < kManyShort ? rows_go<NORM, ADD, BF16, 4, 1>(a) : rows_go<NORM, ADD, BF16, 2, 2>(a);
    if (need <= 8) return a.M < kMany ? rows_go<NORM, ADD, BF16, 8, 1>(a) : rows_go<NORM, ADD, BF16, 4, 2>(a);
    if (need <= 12) return a.M < kMany ? rows_go<NORM, ADD, BF16, 8, 2>(a) : rows_go<NORM, ADD, BF16, 4, 3>(a);
    if (need <= 16) return rows_go<NORM, ADD, BF16, 8, 2>(a);
    if (need <= 24) return rows_go<NORM, ADD, BF16, 8, 3>(a);
    if (need <= 32) return rows_go<NORM, ADD, BF16, 8, 4>(a);
    if (need <= 48) return rows_go<NORM, ADD, BF16, 8, 6>(a);
    if (need <= 60) return rows_go<NORM, ADD, BF16, 12, 5>(a);
    return rows_go<NORM, ADD, BF16, 8, 8>(a);
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
    return bf16 ? rows_launch<false, false, true>(a) : rows_launch<false, false, false>(a);
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
    if (residual) return bf16 ? rows_launch<true, true, true>(a) : rows_launch<true, true, false>(a);
    return bf16 ? rows_launch<true, false, true>(a) : rows_launch<true, false, false>(a);
}

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
#include "tw4_int8.h"

namespace tw4 {

constexpr float kLeast = 0x1p-100f;  // rows whose largest magnitude is below it count as zeros: 127 / max stays finite
constexpr float kMagic = 12582912.0f;    // 1.5 2^23: a float32 of its binade counts by ones, so that adding it rounds, halves to even
constexpr float kBorder = 0.5f - 3.1e-5f;

// The larger of both, NaN if either is (v_maximum3_f32): an infinity or a NaN in a row comes out as its maximum.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Largest of the 64 lanes' values.
__device__ __forceinline__ float wave_largest(float v) {
    v = larger(v, lane_xor1(v));
    v = larger(v, lane_xor2(v));
    v = larger(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, false)));
    v = larger(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, false)));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = larger(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return larger(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The code of t (fl(t) tf) where r = tf fl(127 / fl(top)) is next to a border: the codes of r's size c and c + 1 are compared with t itself.
__device__ __forceinline__ float border_code(float r, double t, double top) {
    const float c = floorf(fabsf(r));
    const double at = 254.0 * fabs(t), border = (2.0 * static_cast<double>(c) + 1.0) * top;
    const bool odd = static_cast<int>(c) & 1;
    const float n = at > border || (at == border && odd) ? c + 1.0f : c;
    return copysignf(n, r);
}

template <bool NORM, bool ADD, bool BF16, int W, int J>
__global__ void __launch_bounds__(64 * W) rows_int8_kernel(const u4* __restrict__ x, int64_t x_step, u4* __restrict__ r,
                                                                  int64_t r_step, const u4* __restrict__ w, float eps,
                                                                  u2* __restrict__ codes, float* __restrict__ scales, int chunks) {
    __shared__ double top_of[W];
    __shared__ float topf_of[W], group_of[NORM ? 4 * W * J : 1];  // group_of: sums of squares of 16 chunks
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x;
    const u4* xr = x + row * x_step;
    u4* rr = r + row * r_step;
    u4 xv[J], rv[J], wv[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int c = 64 * (W * j + wave) + lane;
        xv[j] = rv[j] = wv[j] = u4{0, 0, 0, 0};
        if (c < chunks) {
            xv[j] = xr[c];
            if constexpr (ADD) rv[j] = rr[c];
            if constexpr (NORM) wv[j] = w[c];
        }
    }
    float s[J][8], t[NORM ? J : 1][8];
    float topf = 0.0f, most[J];  // most: of a chunk
    const auto tf = [&](int j, int i) -> float { return NORM ? t[NORM ? j : 0][i] : s[j][i]; };
#pragma unroll
    for (int j = 0; j < J; ++j) {
        chunk_values<BF16>(xv[j], s[j]);
        if constexpr (ADD) {
            float b[8];
            chunk_values<BF16>(rv[j], b);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[j][i] += b[i];
        }
        if constexpr (NORM) {
            float g[8];
            chunk_values<BF16>(wv[j], g);
#pragma unroll
            for (int i = 0; i < 8; ++i) t[j][i] = s[j][i] * g[i];
        }
        most[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) most[j] = larger(most[j], fabsf(tf(j, i)));
        topf = larger(topf, most[j]);
        if constexpr (NORM) {
            const float q = row16_sum(sumsq8(s[j]));
            if ((lane & 15) == 0) group_of[4 * (W * j + wave) + (lane >> 4)] = q;
        }
    }
    topf = wave_largest(topf);
    double top = static_cast<double>(topf);
    if constexpr (NORM) {
        // the exact largest is among those that round to topf
        double mine = 0.0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (most[j] != topf) continue;
            float g[8];
            chunk_values<BF16>(wv[j], g);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (fabsf(t[j][i]) == topf) mine = fmax(mine, fabs(static_cast<double>(s[j][i]) * static_cast<double>(g[i])));
        }
        top = 0.0;
        for (uint64_t lanes = __ballot(mine > 0.0); lanes; lanes &= lanes - 1) {  // one lane, nearly always
            const int l = __builtin_ctzll(lanes);
            const uint64_t bits = bitcast<uint64_t>(mine);
            const uint64_t other = static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<int>(bits >> 32), l)) << 32 |
                                   static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(bits), l));
            top = fmax(top, bitcast<double>(other));
        }
    }
    if constexpr (W > 1) {
        if (lane == 0) top_of[wave] = top, topf_of[wave] = topf;
    }
    __syncthreads();
    if constexpr (W > 1) {
        top = 0.0, topf = 0.0f;
#pragma unroll
        for (int v = 0; v < W; ++v) {
            if constexpr (NORM) top = fmax(top, top_of[v]);
            topf = larger(topf, topf_of[v]);
        }
        if constexpr (!NORM) top = static_cast<double>(topf);
    }
    const bool nan = !(topf < __builtin_inff()), none = nan || topf < kLeast;
    if (wave == 0) {  // rstd in the order of the other norms: the same bits whatever W and J
        const float rstd = NORM ? norm_rstd(group_of, (chunks + 15) / 16, 8 * chunks, eps, lane) : 1.0f;
        if (lane == 0) scales[row] = nan ? __builtin_nanf("") : none ? 0.0f : topf * rstd / 127.0f;
    }
    const float inv = 127.0f / topf;
    const uint32_t keep = none ? 0u : ~0u;
    u2* out = codes + row * chunks;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int c = 64 * (W * j + wave) + lane;
        if (c >= chunks) continue;
        if constexpr (ADD) rr[c] = values_chunk<BF16>(s[j]);
        float n[8], far = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = tf(j, i) * inv;
            n[i] = v + kMagic;
            far = fmaxf(far, fabsf(v - (n[i] - kMagic)));
        }
        if (far > kBorder && !none) {
            float g[8];
            if constexpr (NORM) chunk_values<BF16>(wv[j], g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = tf(j, i) * inv;
                if (fabsf(v - (n[i] - kMagic)) > kBorder)
                    n[i] = border_code(v, static_cast<double>(s[j][i]) * (NORM ? static_cast<double>(g[i]) : 1.0), top) + kMagic;
            }
        }
        uint32_t q[2];  // the codes are the lowest bytes
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(n[4 * h + 1]), __float_as_uint(n[4 * h]), 0x0C0C0400);
            const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(n[4 * h + 3]), __float_as_uint(n[4 * h + 2]), 0x04000C0C);
            q[h] = (lo | hi) & keep;
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

template <bool NORM, bool ADD, bool BF16, int W, int J>
int rows_go(const RowsArgs& a) {
    TW4_REQUIRE(a.M * (64LL * W) < 1LL << 32, TW4_EINVAL, "%s: M = %d is too many rows of %d", NORM ? "rms_norm_int8" : "quantize_int8", a.M, 8 * a.chunks);
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

// A row of activations in 8 bits in a workgroup's registers (tw4_rows8.hip says how the codes come out exactly rounded): shared by the kernels
// that write such rows and the product of one token, which has its row made on the way.
#pragma once

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

// W wavefronts have J chunks of 8 values per lane, chunk c = 64 (W j + wave) + lane.
template <int J>
struct Row8Loads {
    u4 x[J], r[J], w[J];
};

template <bool NORM, int W, int J>
struct Row8Shared {
    double top_of[W];
    float topf_of[W], group_of[NORM ? 4 * W * J : 1];  // group_of: sums of squares of 16 chunks
};

template <bool NORM, bool ADD, int W, int J>
__device__ __forceinline__ void row8_load(Row8Loads<J>& v, const u4* x, const u4* r, const u4* w, int chunks, int wave, int lane) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int c = 64 * (W * j + wave) + lane;
        v.x[j] = v.r[j] = v.w[j] = u4{0, 0, 0, 0};
        if (c < chunks) {
            v.x[j] = x[c];
            if constexpr (ADD) v.r[j] = r[c];
            if constexpr (NORM) v.w[j] = w[c];
        }
    }
}

// Run by the whole workgroup (one barrier inside). sums: where x + r goes (ADD), or null; codes: the row's; scale: written by one lane.
template <bool NORM, bool ADD, bool BF16, int W, int J>
__device__ __forceinline__ void row8_quantize(const Row8Loads<J>& loads, Row8Shared<NORM, W, J>& sh, u4* sums, u2* codes, float* scale, float eps,
                                              int chunks, int wave, int lane) {
    float s[J][8], t[NORM ? J : 1][8];
    float topf = 0.0f, most[J];  // most: of a chunk
    const auto tf = [&](int j, int i) -> float { return NORM ? t[NORM ? j : 0][i] : s[j][i]; };
#pragma unroll
    for (int j = 0; j < J; ++j) {
        chunk_values<BF16>(loads.x[j], s[j]);
        if constexpr (ADD) {
            float b[8];
            chunk_values<BF16>(loads.r[j], b);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[j][i] += b[i];
        }
        if constexpr (NORM) {
            float g[8];
            chunk_values<BF16>(loads.w[j], g);
#pragma unroll
            for (int i = 0; i < 8; ++i) t[j][i] = s[j][i] * g[i];
        }
        most[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) most[j] = larger(most[j], fabsf(tf(j, i)));
        topf = larger(topf, most[j]);
        if constexpr (NORM) {
            const float q = row16_sum(sumsq8(s[j]));
            if ((lane & 15) == 0) sh.group_of[4 * (W * j + wave) + (lane >> 4)] = q;
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
            chunk_values<BF16>(loads.w[j], g);
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
        if (lane == 0) sh.top_of[wave] = top, sh.topf_of[wave] = topf;
    }
    __syncthreads();
    if constexpr (W > 1) {
        top = 0.0, topf = 0.0f;
#pragma unroll
        for (int v = 0; v < W; ++v) {
            if constexpr (NORM) top = fmax(top, sh.top_of[v]);
            topf = larger(topf, sh.topf_of[v]);
        }
        if constexpr (!NORM) top = static_cast<double>(topf);
    }
    const bool nan = !(topf < __builtin_inff()), none = nan || topf < kLeast;
    if (wave == 0) {  // rstd in the order of the other norms: the same bits whatever W and J
        const float rstd = NORM ? norm_rstd(sh.group_of, (chunks + 15) / 16, 8 * chunks, eps, lane) : 1.0f;
        const bool lost = !(rstd > 0.0f && rstd < __builtin_inff());  // the squares' sum has left float32's range: not a scale of 0
        if (lane == 0) *scale = nan || (lost && !none) ? __builtin_nanf("") : none ? 0.0f : topf * rstd / 127.0f;
    }
    const float inv = 127.0f / topf;
    const uint32_t keep = none ? 0u : ~0u;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int c = 64 * (W * j + wave) + lane;
        if (c >= chunks) continue;
        if constexpr (ADD)
            if (sums) sums[c] = values_chunk<BF16>(s[j]);
        float n[8], far = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = tf(j, i) * inv;
            n[i] = v + kMagic;
            far = fmaxf(far, fabsf(v - (n[i] - kMagic)));
        }
        if (far > kBorder && !none) {
            float g[8];
            if constexpr (NORM) chunk_values<BF16>(loads.w[j], g);
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
        codes[c] = u2{q[0], q[1]};
    }
}

}  // namespace tw4

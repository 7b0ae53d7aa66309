// y[M, N] = x_scale[m] w_scale[n] sum_k x[m, k] w[n, k] of 8-bit integers, the sum exact in 32 bits, one rounding; or, with
// act, y[M, N / 2] = silu(g) u of the rows w = [gate | up], g and u unrounded.
//
// The kernel for few tokens streams w through registers. A workgroup of 16 wavefronts takes 16 rows of w and 16 tokens. Units of 128 k
// go to the wavefronts in turn, so that the workgroup reads each row in pieces of 2 KB; each wavefront has one unit in flight ahead of
// the math. The wavefronts' sums are added in LDS.
#include <math.h>

#include "tw4_int8.h"

namespace tw4 {

constexpr int kStreamWaves = 16;

struct Stream8Regs {
    u4 a[2], b[2];
};

template <bool BF16>
__global__ void __launch_bounds__(64 * kStreamWaves) gemm8_stream_kernel(const int8_t* __restrict__ x, uint32_t x_stride,
                                                                         const float* __restrict__ x_scale, const int8_t* __restrict__ w,
                                                                         uint32_t w_stride, const float* __restrict__ w_scale,
                                                                         uint16_t* __restrict__ y, int M, int N, int K) {
    __shared__ i4 part[kStreamWaves][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const int n0 = 16 * blockIdx.x, m0 = 16 * blockIdx.y;
    // rows past the end: the last one, not stored; k past the end: past the resources' records, zeros
    const int rows = min(N - n0, 16), tokens = min(M - m0, 16);
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(w + static_cast<int64_t>(n0) * w_stride), 0,
                                                                        (rows - 1) * w_stride + K, kBufferFlags);
    const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(x + static_cast<int64_t>(m0) * x_stride), 0,
                                                                        (tokens - 1) * x_stride + K, kBufferFlags);
    const uint32_t wo = static_cast<uint32_t>(min(r, rows - 1)) * w_stride + 16 * q, xo = static_cast<uint32_t>(min(r, tokens - 1)) * x_stride + 16 * q;
    const int units = (K + 127) >> 7, steps = (units - wave + kStreamWaves - 1) / kStreamWaves;  // of this wavefront's units
    const auto load = [&](Stream8Regs& v, int s) {
        const int k = 128 * (s * kStreamWaves + wave);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t past = k + 64 * h + 16 * q < K ? 0u : 0x80000000u;
            v.a[h] = bitcast<u4>(__builtin_amdgcn_raw_buffer_load_b128(wr, (wo | past) + 64 * h, k, 2));  // non-temporal: read once
            v.b[h] = bitcast<u4>(__builtin_amdgcn_raw_buffer_load_b128(xr, (xo | past) + 64 * h, k, 0));
        }
    };
    i4 acc{0, 0, 0, 0};
    const auto multiply = [&](const Stream8Regs& v) {
#pragma unroll
        for (int h = 0; h < 2; ++h) acc = mfma_i8(v.a[h], v.b[h], acc);
    };
    Stream8Regs v0, v1;
    if (steps > 0) load(v0, 0);
    for (int s = 0; s < steps; s += 2) {
        if (s + 1 < steps) load(v1, s + 1);
        __builtin_amdgcn_sched_barrier(0);  // the loads above the math
        multiply(v0);
        if (s + 1 >= steps) break;
        if (s + 2 < steps) load(v0, s + 2);
        __builtin_amdgcn_sched_barrier(0);
        multiply(v1);
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave != 0) return;
    const int m = m0 + r, n = n0 + 4 * q;
    const float xs = x_scale[min(m, M - 1)];
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = w_scale[min(n + i, N - 1)];
#pragma unroll
    for (int v = 1; v < kStreamWaves; ++v) acc += part[v][lane];
    if (m >= M) return;
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = static_cast<float>(acc[i]) * xs * s[i];
    store_features<BF16>(y + static_cast<int64_t>(m) * N, n, N, (N & 3) == 0 && (reinterpret_cast<uintptr_t>(y) & 7) == 0, o);
}

int gemm8_stream(const Gemm8Args& a) {
    TW4_REQUIRE(!a.act, TW4_ECONFIG, "gemm_int8: no SwiGLU in the streaming kernel");
    const dim3 grid(static_cast<unsigned>((a.N + 15) / 16), static_cast<unsigned>((a.M + 15) / 16));
    const auto kernel = a.bf16 ? gemm8_stream_kernel<true> : gemm8_stream_kernel<false>;
    kernel<<<grid, 64 * kStreamWaves, 0, a.st>>>(a.x, static_cast<uint32_t>(a.x_stride), a.x_scale, a.w, static_cast<uint32_t>(a.w_stride),
                                                 a.w_scale, a.y, a.M, a.N, a.K);
    TW4_LAUNCH_CHECK("gemm_int8: launch");
    return TW4_OK;
}

// The rule. A kernel's time is predicted from the sizes alone, the fastest (kernel, K splits) taken. Its terms follow the kernels:
//   units U = output tiles x splits, dealt to the CUs: the busiest runs n = ceil(U / CUs) of them, occ at a time;
//   each unit has its stages along K (128 k; the streaming kernel's 16 wavefronts share them), and each round of occ units a start and
//   an end;
//   a stage takes longer with more units on the CU, and with more CUs at work (cu; for the streaming kernel: with more tokens);
//   splits add a wait, the traffic of the partial sums, and a step for each part that the last workgroup adds;
//   beside all this the bytes: what is read and written once at a rate of its own.
// Coefficients in microseconds on MI355X (256 CUs), a row for one tile of tokens (w read once, not kept) and one for more, from least
// squares on relative errors over 520 sizes (20 K x N, M = 1 .. 8192, w streamed from HBM) x up to 60 kernels and splits each
// (profiles/gemm_int8_rule_sweep.jsonl). The choice is 1.2 % slower than the fastest that was timed on average, 31 % at
// most.
struct Gemm8Cost {
    double start, round, stage, share, split, part, rate, step, cu;
};
struct Gemm8Row {
    int bm, bn, occ, least, most;  // tile, workgroups of a CU, tokens it is for
    Gemm8Cost one, more;
};
constexpr Gemm8Row kGemm8Rows[kGemm8Kernels] = {
    {16, 16, 2, 1, 48, {1.432, 0.03182, 1.396, 0.4754, 1, 0.2, 3.759, 0.3, 0.3415},
     {1.432, 0.03182, 1.396, 0.4754, 1, 0.2, 3.759, 0.3, 0.3415}},
    {16, 64, 2, 1, 16, {1.043, 2.466, 0.1504, 1.253, 0.606, 0.828, 5.535, 0.3353, 0.3957},
     {1.043, 2.466, 0.1504, 1.253, 0.606, 0.828, 5.535, 0.3353, 0.3957}},
    {16, 64, 5, 1, 16, {1.753, 1.157, 0.3101, 0.2732, 0.6548, 0.8535, 5.033, 0.3633, 0.03282},
     {1.753, 1.157, 0.3101, 0.2732, 0.6548, 0.8535, 5.033, 0.3633, 0.03282}},
    {32, 64, 2, 1, 200, {1.374, 2.106, 0.178, 1.243, 0.7155, 0.4386, 5.725, 0.3136, 0.2173},
     {1.465, 1.774, 0.1462, 0.8874, 0.8115, 0.3415, 3.743, 0.3517, 0.3565}},
    {64, 64, 2, 17, 1100, {1.316, 2.308, 0.2421, 1.137, 0.7823, 0.2945, 5.818, 0.3858, 0.1972},
     {1.425, 2.263, 0.153, 0.9155, 0.7636, 0.2411, 3.299, 0.394, 0.6335}},
    {64, 128, 2, 17, 1600, {1.698, 1.962, 0.4409, 1.302, 0.7004, 0.288, 4.981, 0.4271, 0.06092},
     {1.631, 2.242, 0.2836, 0.766, 0.4939, 0.263, 3.182, 0.3965, 0.4844}},
    {128, 128, 1, 48, 2048, {0.5382, 4.068, 0.4841, 0.5, 0.7206, 0.1981, 4.563, 0.6378, 0.3615},
     {1.192, 3.459, 0.3894, 0.5, 0.6309, 0.2254, 3.111, 0.5572, 0.414}},
    {192, 64, 1, 100, 4096, {1.106, 3.245, 0.4275, 0.5, 0.843, 0.2283, 3.84, 0.7679, 0.3268},
     {1.597, 3.72, 0.3053, 0.5, 0.8003, 0.1767, 2.906, 0.8219, 0.5293}},
    {128, 192, 2, 65, 1 << 20, {1.757, 4.944, 0.9339, 0.7345, 0.9842, 0.1316, 4.726, 1.397, 0.2274},
     {0.2578, 6.523, 0.7848, 0.2714, 1.554, 0.1234, 2.781, 1.293, 0.2602}},
    {192, 128, 2, 129, 1 << 20, {2.609, 2.363, 0.9088, 0.5419, 1.25, 0.2082, 4.277, 1.31, 0.1995},
     {0.8359, 5.816, 0.7369, 0.3387, 1.259, 0.15, 3.08, 1.241, 0.2547}},
    {128, 256, 1, 65, 1 << 20, {2.144, 4.186, 0.7909, 0.5, 1.299, 0.1618, 5.488, 0.876, 0.4925},
     {0.5045, 6.247, 0.6347, 0.5, 0.5077, 0.1863, 3.056, 1.051, 0.3332}},
    {256, 128, 1, 96, 1 << 20, {1.602, 4.435, 0.6056, 0.5, 0.5437, 0.1833, 4.045, 1.124, 0.5252},
     {1.175, 6.368, 0.4713, 0.5, 0.3402, 0.1605, 4.646, 1.083, 0.7362}},
    {256, 256, 1, 160, 1 << 20, {2.665, 4.276, 1.438, 0.5, 2.693, 0.1677, 4.321, 3.593, 0.4025},
     {0.5145, 9.145, 1.201, 0.5, 1.468, 0.1513, 3.119, 3.448, 0.2847}},
};

static double gemm8_cost(int kernel, int M, int out, int N, int K, int act, int splits, int cus) {
    const Gemm8Row& t = kGemm8Rows[kernel];
    const int64_t mb = (M + t.bm - 1) / t.bm;
    const Gemm8Cost& c = mb > 1 ? t.more : t.one;
    const int features = act ? t.bn / 2 : t.bn;
    const double units = static_cast<double>(mb * ((out + features - 1) / features)) * splits;
    const int all = (K + 127) / 128, ways = kernel ? splits : kStreamWaves, stages = (all + ways - 1) / ways;
    const double n = ceil(units / cus), full = floor(n / t.occ), rest = n - full * t.occ;
    const double stage = c.stage * (1 + c.cu * (kernel ? fmin(1.0, units / cus) : (M < 16 ? M : 16) / 16.0));
    double us = c.start + ceil(n / t.occ) * c.round + stages * stage * (full * (1 + c.share * (t.occ - 1)) + (rest > 0 ? 1 + c.share * (rest - 1) : 0));
    if (splits > 1) us += c.split + c.part * units * t.bm * t.bn * 4e-6 + c.step * (splits - 1);
    const double bytes = static_cast<double>(N) * K * (kernel ? 1 : mb) + static_cast<double>(M) * K + 2.0 * M * out;
    const double moved = c.start + bytes / (c.rate * 1e6);
    us *= us;
    return sqrt(sqrt(us * us + moved * moved * moved * moved));
}

static void gemm8_plan(int M, int N, int K, int act, int cus, int* out) {
    constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16};
    const int features = act ? N / 2 : N, stages = (K + 127) / 128;
    double best = INFINITY;
    for (int k = 0; k < kGemm8Kernels; ++k) {
        const Gemm8Row& t = kGemm8Rows[k];
        if (M < t.least || M > t.most || (k == 0 && act)) continue;
        const int tile = act ? t.bn / 2 : t.bn;
        const int64_t tiles = static_cast<int64_t>((M + t.bm - 1) / t.bm) * ((features + tile - 1) / tile);
        for (int s : kSplits) {
            const int64_t words = tiles * s * t.bm * t.bn;
            if (s > 1 && (k == 0 || 2 * s > stages || words > TW4_AUTO_SPLIT_FLOATS || tiles > TW4_AUTO_SPLIT_COUNTERS)) break;
            const double us = gemm8_cost(k, M, features, N, K, act, s, cus);
            if (us >= best) continue;
            best = us;
            out[0] = k, out[1] = s, out[2] = s > 1 ? static_cast<int>(words) : 0, out[3] = s > 1 ? static_cast<int>(tiles) : 0;
        }
    }
}

static int gemm8_check_sizes(int M, int N, int K, int act) {
    TW4_REQUIRE(M >= 0 && M <= 1 << 20, TW4_EINVAL, "gemm_int8: 0 <= M <= 2^20 (M = %d)", M);
    TW4_REQUIRE(N >= 1 && N <= 1 << 24, TW4_EINVAL, "gemm_int8: 1 <= N <= 2^24 (N = %d)", N);
    TW4_REQUIRE(K >= 16 && K % 16 == 0 && K < 1 << 17, TW4_EINVAL, "gemm_int8: K %% 16 == 0 and 16 <= K < 2^17 (K = %d)", K);
    TW4_REQUIRE(act == 0 || (act == 1 && N % 2 == 0), TW4_EINVAL, "gemm_int8: act 0, or 1 (SwiGLU) with an even N (act %d, N %d)", act, N);
    return TW4_OK;
}

}  // namespace tw4

using namespace tw4;

extern "C" int tw4_gemm_int8_plan(int M, int N, int K, int act, int cus, int* out) {
    const int rc = gemm8_check_sizes(M, N, K, act);
    if (rc) return rc;
    TW4_REQUIRE(M >= 1 && cus >= 1 && out, TW4_EINVAL, "gemm_int8_plan: M, cus >= 1 and out");
    gemm8_plan(M, N, K, act, cus, out);
    return TW4_OK;
}

extern "C" int tw4_gemm_int8(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride,
                             const float* w_scale, uint16_t* y, int32_t* ws, int64_t ws_words, int32_t* locks, int64_t n_locks, int M,
                             int N, int K, int act, int bf16, int kernel, int splits, void* stream) {
    TW4_REQUIRE(x && x_scale && w && w_scale && y, TW4_EINVAL, "gemm_int8: null pointer");
    TW4_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0, TW4_EINVAL,
                "gemm_int8: rows must be 16-byte aligned");
    TW4_REQUIRE(reinterpret_cast<uintptr_t>(x_scale) % 4 == 0 && reinterpret_cast<uintptr_t>(w_scale) % 4 == 0 &&
                    reinterpret_cast<uintptr_t>(y) % 2 == 0,
                TW4_EINVAL, "gemm_int8: scales must be 4-byte aligned and y 2-byte");
    const int rc = gemm8_check_sizes(M, N, K, act);
    if (rc) return rc;
    TW4_REQUIRE(x_stride >= K && x_stride % 16 == 0 && w_stride >= K && w_stride % 16 == 0 && x_stride < 1 << 22 && w_stride < 1 << 22,
                TW4_EINVAL, "gemm_int8: rows at least K and less than 2^22 apart, 16-byte aligned (strides %lld, %lld)",
                static_cast<long long>(x_stride), static_cast<long long>(w_stride));
    TW4_REQUIRE(kernel >= 0 && kernel < kGemm8Kernels, TW4_ECONFIG, "gemm_int8: kernel %d", kernel);
    TW4_REQUIRE(splits >= 1 && splits <= (K + 127) / 128 && (kernel || splits == 1), TW4_ECONFIG,
                "gemm_int8: 1 .. K / 128 splits, 1 for kernel 0 (kernel %d, splits %d, K %d)", kernel, splits, K);
    if (M == 0) return TW4_OK;
    const Gemm8Args a{x, x_stride, x_scale, w, w_stride, w_scale, y, M, N, K, act, bf16, ws, locks, ws_words, n_locks,
                      static_cast<hipStream_t>(stream)};
    return kernel ? gemm8_lds(a, kernel, splits) : gemm8_stream(a);
}

// y[M, N] = x_scale[m] w_scale[n] sum_k x[m, k] w[n, k] of 8-bit integers, the sum exact in 32 bits, one rounding; or, with
// act, y[M, N / 2] = silu(g) u of the rows w = [gate | up], g and u unrounded.
//
// The kernel for few tokens streams w through registers. A workgroup of 16 wavefronts takes `rows` rows of w, up to NT tiles of 16,
// and 16 tokens; as many rows as give every CU the same work. Units of 128 k go to the wavefronts in turn, so that the workgroup reads
// each row in pieces of 2 KB; each wavefront has one unit in flight ahead of the math. The wavefronts' sums are added in LDS.
// Bound by reading w behind a launch: K 4096 x N 6144 at M = 1 7.3 us (3.4 TB/s; 25 MB at 5.9 TB/s, what a plain read reaches, are 4.3, the
// launch and the first and last round trips the rest), K 12288 x N 4096 12.3 (4.1 TB/s). 4 or 8 wavefronts per workgroup, or 2 units ahead:
// within 5 %. Two 16-row tiles per workgroup where one fills the CUs: 20-60 % slower.
#include <math.h>

#include "tw4_rows8.h"

namespace tw4 {

constexpr int kStreamWaves = 16;

template <int NT>
struct Stream8Regs {
    u4 a[NT][2], b[2];
};

template <int NT, bool BF16>
__global__ void __launch_bounds__(64 * kStreamWaves) gemm8_stream_kernel(const int8_t* __restrict__ x, uint32_t x_stride,
                                                                         const float* __restrict__ x_scale, const int8_t* __restrict__ w,
                                                                         uint32_t w_stride, const float* __restrict__ w_scale,
                                                                         uint16_t* __restrict__ y, int M, int N, int K, int rows_each) {
    __shared__ i4 part[kStreamWaves][NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const int n0 = rows_each * blockIdx.x, m0 = 16 * blockIdx.y;
    // what lies past the rows, the tokens or K is past the resources' records: zeros, nothing read
    const int rows = min(N - n0, rows_each), tokens = min(M - m0, 16);
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(w + static_cast<int64_t>(n0) * w_stride), 0,
                                                                        (rows - 1) * w_stride + K, kBufferFlags);
    const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(x + static_cast<int64_t>(m0) * x_stride), 0,
                                                                        (tokens - 1) * x_stride + K, kBufferFlags);
    uint32_t wo[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) wo[t] = 16 * t + r < rows ? static_cast<uint32_t>(16 * t + r) * w_stride + 16 * q : 0x80000000u;
    const uint32_t xo = r < tokens ? static_cast<uint32_t>(r) * x_stride + 16 * q : 0x80000000u;
    const int units = (K + 127) >> 7, steps = (units - wave + kStreamWaves - 1) / kStreamWaves;  // of this wavefront's units
    const auto load = [&](Stream8Regs<NT>& v, int s) {
        const int k = 128 * (s * kStreamWaves + wave);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t past = k + 64 * h + 16 * q < K ? 0u : 0x80000000u;
#pragma unroll
            for (int t = 0; t < NT; ++t)
                v.a[t][h] = bitcast<u4>(__builtin_amdgcn_raw_buffer_load_b128(wr, (wo[t] | past) + 64 * h, k, 2));  // non-temporal: read once
            v.b[h] = bitcast<u4>(__builtin_amdgcn_raw_buffer_load_b128(xr, (xo | past) + 64 * h, k, 0));
        }
    };
    i4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = i4{0, 0, 0, 0};
    const auto multiply = [&](const Stream8Regs<NT>& v) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t] = mfma_i8(v.a[t][h], v.b[h], acc[t]);
    };
    Stream8Regs<NT> v0, v1;
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
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    if (wave >= NT) return;  // wavefront t adds tile t
    const int m = m0 + r, at = 16 * wave + 4 * q, n = n0 + at;
    const float xs = x_scale[min(m, M - 1)];
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = w_scale[min(n + i, N - 1)];
    i4 sum{0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < kStreamWaves; ++v) sum += part[v][wave][lane];
    if (m >= M) return;
    uint16_t* row = y + static_cast<int64_t>(m) * N + n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i < rows) row[i] = static_cast<uint16_t>(value16<BF16>(static_cast<float>(sum[i]) * xs * s[i]));
}

// One token, its row put in 8 bits on the way (the bits of the kernels that do it alone). The streaming kernel above; every workgroup makes the
// whole row, in LDS, while its first rows of w are on the way: TILES tiles of 16 outputs, with SwiGLU one of gate rows and one of up rows.
// Workgroup 0 writes the new residual, to memory of its own: others still read the old one.
// Against the two kernels in a graph, us (weights from HBM; SwiGLU: the tiled kernel with K splits): row alone, norm, add + norm:
//   K 4096 x N 6144   8.3, 8.5, 8.6 (9.2, 9.7, 9.7)     K 9728 x N 2560      8.6, 9.5, 9.6 (10.1, 11.4, 11.3)
//   K 512 x N 1024    3.5, 4.6, 4.6 (4.5, 5.3, 5.0)     K 2064 x 2501 pairs  6.1, 6.7, 6.7 (9.5, 10.1, 10.2)
// and 8 to 10 where a caller waits for the host (16.5 to 18). More outputs than one workgroup a CU holds lose, each round making the row again:
//   K 8192 x N 10240  20.8, 25.8, 25.8 (18.2, 19, 19)   K 4096 x 14336 pairs  31, 35, 36 (25, 25, 25.5)
// and so does SwiGLU in 32 pairs a workgroup (K 2560 x 6912 pairs 12.2, 12.1, 12.1 (10.1, 10.7, 10.8)), so that it is left at 16.
template <int TILES, bool ACT, bool NORM, bool ADD, bool BF16, int J>
__global__ void __launch_bounds__(64 * kStreamWaves) token8_kernel(const u4* __restrict__ x, const u4* __restrict__ r, u4* __restrict__ r_out,
                                                                   const u4* __restrict__ norm_weight, float eps, const int8_t* __restrict__ w,
                                                                   uint32_t w_stride, const float* __restrict__ w_scale,
                                                                   uint16_t* __restrict__ y, int N, int K, int rows_each) {
    constexpr int NT = ACT ? 2 * TILES : TILES;
    constexpr bool late = NORM && NT * J > 2;  // 128 registers do not hold the row and both steps
    __shared__ Row8Shared<NORM, kStreamWaves, J> shared;
    __shared__ u2 codes[64 * kStreamWaves * J];
    __shared__ i4 part[kStreamWaves][NT][64];
    __shared__ float x_scale;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, q = lane >> 4;
    const int out = ACT ? N >> 1 : N, n0 = rows_each * blockIdx.x, chunks = K >> 3;
    Row8Loads<J> row;
    row8_load<NORM, ADD, kStreamWaves, J>(row, x, r, norm_weight, chunks, wave, lane);
    // what lies past the rows or K is past the resources' records: zeros, nothing read
    const int rows = min(out - n0, rows_each), size = (rows - 1) * w_stride + K;
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(w + static_cast<int64_t>(n0) * w_stride), 0, size, kBufferFlags);
    const __amdgpu_buffer_rsrc_t ur =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(w + static_cast<int64_t>(ACT ? out + n0 : n0) * w_stride), 0, size, kBufferFlags);
    uint32_t wo[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) wo[t] = 16 * t + lr < rows ? static_cast<uint32_t>(16 * t + lr) * w_stride + 16 * q : 0x80000000u;
    const int units = (K + 127) >> 7, steps = (units - wave + kStreamWaves - 1) / kStreamWaves;  // of this wavefront's units
    const auto load = [&](u4 (&v)[NT][2], int s) {
        const int k = 128 * (s * kStreamWaves + wave);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t past = k + 64 * h + 16 * q < K ? 0u : 0x80000000u;
#pragma unroll
            for (int t = 0; t < NT; ++t)
                v[t][h] = bitcast<u4>(__builtin_amdgcn_raw_buffer_load_b128(t < TILES ? wr : ur, (wo[t % TILES] | past) + 64 * h, k, 2));
        }
    };
    i4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = i4{0, 0, 0, 0};
    const char* xc = reinterpret_cast<const char*>(codes) + 16 * q;  // every column is the token: one is stored
    const auto multiply = [&](const u4 (&v)[NT][2], int s) {
        const int k = 128 * (s * kStreamWaves + wave);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u4 b = *reinterpret_cast<const u4*>(xc + k + 64 * h);
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t] = mfma_i8(v[t][h], b, acc[t]);
        }
    };
    u4 v0[NT][2], v1[NT][2];
    if (steps > 0) load(v0, 0);
    if (!late && steps > 1) load(v1, 1);
    __builtin_amdgcn_sched_barrier(0);
    row8_quantize<NORM, ADD, BF16, kStreamWaves, J>(row, shared, blockIdx.x == 0 ? r_out : nullptr, codes, &x_scale, eps, chunks, wave, lane);
    if (late && steps > 1) load(v1, 1);
    __syncthreads();
    for (int s = 0; s < steps; s += 2) {
        multiply(v0, s);
        if (s + 1 >= steps) break;
        if (s + 2 < steps) load(v0, s + 2);
        __builtin_amdgcn_sched_barrier(0);
        multiply(v1, s + 1);
        if (s + 3 < steps) load(v1, s + 3);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    if (wave >= TILES || lr != 0) return;  // wavefront t adds tile t
    const int at = 16 * wave + 4 * q, n = n0 + at;
    i4 sum{0, 0, 0, 0}, up{0, 0, 0, 0};
#pragma unroll 4
    for (int v = 0; v < kStreamWaves; ++v) {
        sum += part[v][wave][lane];
        if constexpr (ACT) up += part[v][wave + TILES][lane];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (at + i >= rows) break;
        float v[1] = {static_cast<float>(sum[i]) * x_scale * w_scale[n + i]};
        if constexpr (ACT) {
            silu_values(v);
            v[0] *= static_cast<float>(up[i]) * x_scale * w_scale[out + n + i];
        }
        y[n + i] = static_cast<uint16_t>(value16<BF16>(v[0]));
    }
}

struct Token8Args {
    const u4 *x, *r;
    u4* r_out;
    const u4* norm_weight;
    float eps;
    const int8_t* w;
    uint32_t w_stride;
    const float* w_scale;
    uint16_t* y;
    int N, K, rows;
    hipStream_t st;
};

template <int TILES, bool ACT, bool NORM, bool ADD, bool BF16>
int token8_launch(const Token8Args& a) {
    const int out = ACT ? a.N / 2 : a.N;
    const unsigned grid = static_cast<unsigned>((out + a.rows - 1) / a.rows);
    const auto kernel = a.K <= 512 * kStreamWaves ? token8_kernel<TILES, ACT, NORM, ADD, BF16, 1> : token8_kernel<TILES, ACT, NORM, ADD, BF16, 2>;
    kernel<<<grid, 64 * kStreamWaves, 0, a.st>>>(a.x, a.r, a.r_out, a.norm_weight, a.eps, a.w, a.w_stride, a.w_scale, a.y, a.N, a.K, a.rows);
    TW4_LAUNCH_CHECK("token_int8: launch");
    return TW4_OK;
}

template <int TILES, bool ACT, bool BF16>
int token8_norm(const Token8Args& a) {
    if (!a.norm_weight) return token8_launch<TILES, ACT, false, false, BF16>(a);
    return a.r ? token8_launch<TILES, ACT, true, true, BF16>(a) : token8_launch<TILES, ACT, true, false, BF16>(a);
}

template <bool BF16>
int token8_any(const Token8Args& a, int act) {
    if (act) return token8_norm<1, true, BF16>(a);
    return a.rows <= 16 ? token8_norm<1, false, BF16>(a) : token8_norm<2, false, BF16>(a);
}

// Rows of w per workgroup of the streaming kernel: what gives every CU one workgroup, where that is 4 to 32 rows, else 16. M = 1, us, with
// 16 rows each: K 4096 x N 6144 7.4 (8.2), K 9728 x N 2560 7.9 (9.9), K 8192 x N 512 6.1 (7.7), K 2064 x N 5001 5.3 (6.0).
static int stream8_rows(int N, int cus) {
    const int each = (N + cus - 1) / cus;
    return each > 32 ? 16 : each < 4 ? 4 : each;
}

int gemm8_stream(const Gemm8Args& a, int rows) {
    TW4_REQUIRE(!a.act, TW4_ECONFIG, "gemm_int8: no SwiGLU in the streaming kernel");
    const dim3 grid(static_cast<unsigned>((a.N + rows - 1) / rows), static_cast<unsigned>((a.M + 15) / 16));
    TW4_REQUIRE(grid.y < 1 << 16, TW4_ECONFIG, "gemm_int8: M <= 2^20 - 16 for the streaming kernel (M %d)", a.M);
    TW4_REQUIRE(grid.x * (64LL * kStreamWaves) < 1LL << 32, TW4_ECONFIG, "gemm_int8: N = %d is too many rows of w for %d a workgroup", a.N, rows);
    const auto kernel = rows <= 16 ? (a.bf16 ? gemm8_stream_kernel<1, true> : gemm8_stream_kernel<1, false>)
                                   : (a.bf16 ? gemm8_stream_kernel<2, true> : gemm8_stream_kernel<2, false>);
    kernel<<<grid, 64 * kStreamWaves, 0, a.st>>>(a.x, static_cast<uint32_t>(a.x_stride), a.x_scale, a.w, static_cast<uint32_t>(a.w_stride),
                                                 a.w_scale, a.y, a.M, a.N, a.K, rows);
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
// (profiles/gemm_int8_rule_sweep.jsonl). The choice is 0.9 % slower than the fastest that was timed on average, 20 % at
// most. The times are those of the tiles listed in tw4_int8.h and their epilogue: what changes either makes them stale.
struct Gemm8Cost {
    double start, round, stage, share, split, part, rate, step, cu;
};
struct Gemm8Row {
    int bm, bn, occ, least, most;  // tile, workgroups of a CU, tokens it is for
    Gemm8Cost one, more;
};
constexpr Gemm8Row kGemm8Rows[kGemm8Kernels] = {
    {16, 16, 2, 1, 48, {2.006, 0.0404, 0.9011, 0.7127, 1, 0.2, 4.215, 0.3, 0.5808},
     {2.006, 0.0404, 0.9011, 0.7127, 1, 0.2, 4.215, 0.3, 0.5808}},
    {16, 64, 2, 1, 16, {1.075, 2.266, 0.1511, 1.197, 0.7192, 0.8719, 5.66, 0.3479, 0.4062},
     {1.075, 2.266, 0.1511, 1.197, 0.7192, 0.8719, 5.66, 0.3479, 0.4062}},
    {16, 64, 5, 1, 16, {1.953, 0.5751, 0.3161, 0.2639, 0.8462, 0.9349, 5.181, 0.373, 0.02961},
     {1.953, 0.5751, 0.3161, 0.2639, 0.8462, 0.9349, 5.181, 0.373, 0.02961}},
    {32, 64, 2, 1, 200, {1.401, 1.908, 0.1816, 1.213, 0.8341, 0.4644, 5.823, 0.3286, 0.2125},
     {1.431, 1.725, 0.1484, 0.8889, 0.9028, 0.3455, 3.762, 0.3651, 0.3336}},
    {64, 64, 2, 17, 1100, {1.272, 2.407, 0.2147, 1.198, 0.9773, 0.2784, 6.186, 0.3893, 0.3374},
     {1.541, 2.178, 0.1584, 1.106, 0.8578, 0.2606, 3.462, 0.409, 0.4391}},
    {64, 128, 1, 17, 1600, {0.6257, 3.355, 0.3741, 0.5, 1.021, 0.2248, 4.766, 0.4157, 0.2747},
     {1.42, 2.543, 0.2623, 0.5, 0.7342, 0.2412, 3.277, 0.4192, 0.5235}},
    {128, 128, 1, 48, 2048, {0.5995, 3.757, 0.4858, 0.5, 0.8329, 0.2038, 4.74, 0.6828, 0.3688},
     {1.256, 3.112, 0.3904, 0.5, 0.6549, 0.2295, 3.025, 0.6031, 0.4285}},
    {192, 64, 1, 100, 4096, {1.341, 2.825, 0.4221, 0.5, 0.9907, 0.2522, 4.439, 0.7727, 0.3601},
     {1.433, 3.447, 0.3145, 0.5, 0.8059, 0.1902, 2.68, 0.8677, 0.4794}},
    {128, 192, 2, 65, 1 << 20, {1.814, 4.734, 0.935, 0.6605, 1.004, 0.1143, 4.959, 1.509, 0.2237},
     {0.1866, 6.255, 0.7796, 0.2627, 1.395, 0.1239, 2.824, 1.42, 0.2704}},
    {192, 128, 2, 129, 1 << 20, {2.937, 1.886, 0.9098, 0.5362, 1.39, 0.2002, 4.871, 1.388, 0.1955},
     {0.7776, 5.342, 0.7345, 0.3317, 1.109, 0.1562, 2.929, 1.366, 0.2663}},
    {128, 256, 1, 65, 1 << 20, {2.105, 3.737, 0.7957, 0.5, 1.454, 0.1432, 6.805, 1.016, 0.5145},
     {0.659, 5.642, 0.6385, 0.5, 0.5123, 0.1937, 3.156, 1.142, 0.3352}},
    {256, 128, 1, 96, 1 << 20, {1.903, 3.708, 0.6029, 0.5, 0.6856, 0.1807, 4.557, 1.279, 0.5604},
     {1.203, 5.711, 0.4825, 0.5, 0.3244, 0.1771, 3.293, 1.104, 0.694}},
    {256, 256, 1, 160, 1 << 20, {2.705, 3.972, 1.437, 0.5, 3.409, 0.1492, 3.737, 3.916, 0.2705},
     {0.5704, 8.532, 1.212, 0.5, 1.722, 0.1521, 2.879, 3.68, 0.2629}},
};

static double gemm8_cost(int kernel, int M, int out, int N, int K, int act, int splits, int cus) {
    const Gemm8Row& t = kGemm8Rows[kernel];
    const int64_t mb = (M + t.bm - 1) / t.bm;
    const Gemm8Cost& c = mb > 1 ? t.more : t.one;
    const int features = kernel == 0 ? stream8_rows(N, cus) : act ? t.bn / 2 : t.bn;
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
            out[0] = k, out[1] = k ? s : stream8_rows(N, cus), out[2] = s > 1 ? static_cast<int>(words) : 0, out[3] = s > 1 ? static_cast<int>(tiles) : 0;
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

extern "C" int tw4_token_int8(const uint16_t* x, const uint16_t* residual, uint16_t* residual_out, const uint16_t* norm_weight, float eps,
                              const int8_t* w, int64_t w_stride, const float* w_scale, uint16_t* y, int N, int K, int act, int bf16, int cus,
                              void* stream) {
    TW4_REQUIRE(x && w && w_scale && y, TW4_EINVAL, "token_int8: null pointer");
    TW4_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(residual) % 16 == 0 && reinterpret_cast<uintptr_t>(residual_out) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(norm_weight) % 16 == 0,
                TW4_EINVAL, "token_int8: rows must be 16-byte aligned");
    TW4_REQUIRE(reinterpret_cast<uintptr_t>(w_scale) % 4 == 0 && reinterpret_cast<uintptr_t>(y) % 2 == 0, TW4_EINVAL,
                "token_int8: scales must be 4-byte aligned and y 2-byte");
    TW4_REQUIRE(!residual == !residual_out && (!residual || norm_weight), TW4_EINVAL,
                "token_int8: a residual comes with a norm weight and memory for the new one");
    const int rc = gemm8_check_sizes(1, N, K, act);
    if (rc) return rc;
    TW4_REQUIRE(K <= TW4_TOKEN_INT8_MAX, TW4_EINVAL, "token_int8: K <= %d (K = %d)", TW4_TOKEN_INT8_MAX, K);
    TW4_REQUIRE(w_stride >= K && w_stride % 16 == 0 && w_stride < 1 << 22, TW4_EINVAL,
                "token_int8: rows at least K and less than 2^22 apart, 16-byte aligned (stride %lld)", static_cast<long long>(w_stride));
    TW4_REQUIRE(cus >= 1, TW4_EINVAL, "token_int8: cus >= 1");
    const int out = act ? N / 2 : N, rows = stream8_rows(out, cus);
    TW4_REQUIRE((out + rows - 1) / rows <= cus && rows <= (act ? 16 : 32), TW4_ECONFIG,
                "token_int8: at most 32 outputs, or 16 of SwiGLU, a CU (%d outputs, %d CUs)", out, cus);
    const int64_t row = 2LL * K;  // bytes; some workgroups write while others still read
    for (const uint16_t* p : {x, residual, norm_weight})
        TW4_REQUIRE(!p || !residual_out || bytes_apart(p, row, residual_out, row), TW4_EINVAL, "token_int8: the new residual needs memory of its own");
    for (const uint16_t* p : {x, residual, norm_weight, static_cast<const uint16_t*>(residual_out)})
        TW4_REQUIRE(!p || bytes_apart(p, row, y, 2LL * out), TW4_EINVAL, "token_int8: y needs memory of its own");
    const Token8Args a{reinterpret_cast<const u4*>(x), reinterpret_cast<const u4*>(residual), reinterpret_cast<u4*>(residual_out),
                       reinterpret_cast<const u4*>(norm_weight), eps, w, static_cast<uint32_t>(w_stride), w_scale, y, N, K, rows,
                       static_cast<hipStream_t>(stream)};
    return bf16 ? token8_any<true>(a, act) : token8_any<false>(a, act);
}

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
    TW4_REQUIRE(splits >= 1 && splits <= (kernel ? (K + 127) / 128 : 32), TW4_ECONFIG,
                "gemm_int8: 1 .. K / 128 splits, 1 .. 32 rows of kernel 0 (kernel %d, splits %d, K %d)", kernel, splits, K);
    if (M == 0) return TW4_OK;
    const Gemm8Args a{x, x_stride, x_scale, w, w_stride, w_scale, y, M, N, K, act, bf16, ws, locks, ws_words, n_locks,
                      static_cast<hipStream_t>(stream)};
    return kernel ? gemm8_lds(a, kernel, splits) : gemm8_stream(a, splits);
}

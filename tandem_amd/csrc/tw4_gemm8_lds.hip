// The product of 8-bit integers for more tokens than a few: both operands through LDS by direct-to-LDS loads.
//
// Workgroup tile BM x BN = (WM wavefronts x 16 TM tokens) x (WN wavefronts x 16 TN rows of w); a stage is 128 k (128 bytes of each
// row), two substeps of 64 k, in a ring of R slots.
//   LDS:   slot row rho (tokens, then rows of w) is 128 bytes, position p of which holds 16-byte chunk p ^ ((rho >> 1) & 7): the 16
//          lanes of a fragment read (16 rows, one chunk) touch all 64 banks once.
//   act:   rows of w are [gate | up]: the first BN / 2 of the tile are gate rows, the others their up rows, and a wavefront's
//          first TN / 2 tiles are the gates of the others, so that both lie in one lane's registers.
//   loop:  substep 0 of stage i multiplies while substep 1's fragments are read; then the wavefront waits for its own loads of stage i + 1
//          and the workgroup meets; substep 1 multiplies while stage i + 1's first fragments are read, and stage i's slot, which
//          nobody reads any more, takes the loads of stage i + R.
//   tails: rows past the end read the last one (not stored). Chunks past K, which a row has in its last stage only, are zeros: their load
//          offsets are past the resources' records.
//   near:  where all tokens are one tile, w is read once, by non-temporal loads.
//   end:   the scales are read beside the last stages' waits; results go through LDS, so that stores write whole rows.
//
// What bounds it. Long products: the matrix cores and what feeds them at the clock the card's power leaves: K 4096 x N 24576 SwiGLU at
// M = 8192 keeps the cores busy 58 % of the cycles at 1.8 GHz, wavefronts wait 37 % of theirs (stages come from past L2: 1.2 GB of
// it, and with every load a hit the loop runs 20 % faster), LDS is busy 25 %. 674-702 us, 2.35-2.45 POP/s, where the library's int8 product
// without scales or SwiGLU takes 765; K 12288 x N 4096 304 (341), K 4096 x N 4096 113-119 (126); at M = 512 18 (22), K 12288 40 (45).
// Middle sizes: how fast stages come into LDS, 58-72 KB/us a CU with all CUs at work whatever the tile's shape (the fitted stages of tw4_gemm8.hip; the
// products of a stage at 5 POP/s are 14 to 56 % of that time, and a second workgroup of the small tiles on the CU overlaps with nothing), and how evenly the
// tiles divide over the CUs. Few tokens: reading w, 5.0 TB/s of it (K 4096 x N 24576, M = 1 .. 16: 20-22 us).
// Measured steps, us, K 4096: results straight from the accumulators, 8 bytes a lane, and the scales read for each tile: M = 8192, N 4096 134,
// through LDS 115; N 5001 (K 2064), M = 2048 45 -> 36. Non-temporal w: N 24576, M = 16 21.9 -> 19.8, N 34816 (K 5120) 41.8 -> 38.1.
// v_mfma_i32_32x32x32_i8 instead, the same tiles: 5-30 % slower at every size. Stages of 64 k in 4 or 5 slots (a barrier
// each, the loads farther ahead): 3 % slower at M = 8192, 2 % faster in one round of tiles. 128 x 256 in 4 wavefronts of 128 x 64: 20-40 %
// slower than in 8 of 64 x 64. 2, 4 or 5 slots for 128 x 128: level. 5 for 64 x 64: M = 200, N 4096 11.8 -> 10.6.
#include "tw4_int8.h"
#include "tw4_lds.h"

namespace tw4 {

// Orders this wavefront's LDS accesses before and after it (they run in order; the compiler keeps the order too).
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ROWS x COLUMNS 16-bit values in LDS (rows PITCH bytes apart) to global rows `out` values apart, V values (a T) a lane and store; only
// the first `rows` and `columns` (a multiple of V, or none).
template <int V, int ROWS, int COLUMNS, int PITCH, class T>
__device__ __forceinline__ void store_rows(uint16_t* __restrict__ to, int out, const char* from, int rows, int columns, int lane) {
    constexpr int PER_ROW = COLUMNS / V, ALL = ROWS * PER_ROW;
#pragma unroll 8
    for (int i = 0; i < (ALL + 63) / 64; ++i) {
        const int at = 64 * i + lane, row = at / PER_ROW, c = V * (at % PER_ROW);
        if ((ALL % 64 == 0 || at < ALL) && row < rows && c < columns)
            *reinterpret_cast<T*>(to + static_cast<int64_t>(row) * out + c) = *reinterpret_cast<const T*>(from + row * PITCH + 2 * c);
    }
}

#define TW4_STEP_FENCE __builtin_amdgcn_sched_barrier(0)

template <int TM_, int TN_, int WM_, int WN_, int R_, bool NT_ = false>
struct Gemm8Cfg {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, R = R_;
    static constexpr bool NT = NT_;
    static constexpr int BM = 16 * TM * WM, BN = 16 * TN * WN, WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int SLOT = 128 * (BM + BN);                    // bytes
    static constexpr int XI = BM / 8 / WAVES, WI = BN / 8 / WAVES;  // 1 KB loads of a stage per wavefront, 8 rows each
    static constexpr int LOADS = XI + WI;
    static constexpr int LDS_BYTES = R * SLOT;
    static constexpr int PER_SIMD = WAVES / 4 * (160 * 1024 / LDS_BYTES) > 1 && TM * TN <= 32 ? 2 : 1;
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole loads");
    static_assert(WAVES % 2 == 0, "a lane's chunk is the same in all of its loads");
    static_assert(R >= 2 && (R - 1) * LOADS < 64, "s_waitcnt vmcnt immediate");
    static_assert(LDS_BYTES <= 160 * 1024, "one workgroup's LDS");
};

// The accumulators stay in accumulation registers for the whole loop: left to the compiler they move between the register files.
__device__ __forceinline__ void mfma_i8_acc(i4& c, const u4& a, const u4& b) {
    asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

template <class C>
struct Gemm8Regs {
    u4 a[2][C::TN], b[2][C::TM];  // fragments of w and x, of this substep and the next
};

template <class C>
struct Gemm8Loads {
    u4 x, w, up;                           // resources of the tile's tokens, (gate) rows and up rows
    uint32_t xoff[C::XI], woff[C::WI];     // this lane's byte offsets
    uint32_t lds;                          // this wavefront's first byte in a slot
};

// Load I of a stage into the slot at LDS byte address `slot`; tail: added to the offsets, past the records where the lane's chunk lies
// past K.
template <int I, class C, bool ACT>
__device__ __forceinline__ void gemm8_load(uint32_t slot, const Gemm8Loads<C>& l, const u4& xr, const u4& wr, const u4& ur,
                                           uint32_t koff, uint32_t tail) {
    if constexpr (I < C::XI) {
        lds_dma16<1024 * I * C::WAVES>(xr, l.xoff[I] + tail, koff, slot + l.lds);
    } else {
        constexpr int J = I - C::XI;
        lds_dma16<128 * C::BM + 1024 * J * C::WAVES, C::NT>(ACT && J >= C::WI / 2 ? ur : wr, l.woff[J] + tail, koff, slot + l.lds);
    }
}

template <int I, int S, class C, bool ACT>
__device__ __forceinline__ void gemm8_loads_at(int k, uint32_t slot, const Gemm8Loads<C>& l, const u4& xr, const u4& wr, const u4& ur,
                                               uint32_t koff, uint32_t tail) {
    if constexpr (I < C::LOADS) {
        if ((2 * I + 1) * S / (2 * C::LOADS) == k) gemm8_load<I, C, ACT>(slot, l, xr, wr, ur, koff, tail);
        gemm8_loads_at<I + 1, S, C, ACT>(k, slot, l, xr, wr, ur, koff, tail);
    }
}

// One substep: TM x TN products from register set CUR, between which the other set is read (ap, bp: its first fragments in LDS) and,
// with LOAD, a stage's loads are issued.
template <class C, int CUR, bool LOAD, bool ACT>
__device__ __forceinline__ void gemm8_substep(Gemm8Regs<C>& v, i4 (&acc)[C::TN][C::TM], const char* ap, const char* bp, uint32_t slot,
                                              const Gemm8Loads<C>& l, const u4& xr, const u4& wr, const u4& ur, uint32_t koff, uint32_t tail) {
    constexpr int S = C::TM * C::TN, F = C::TM + C::TN;
#pragma unroll
    for (int t = 0; t < C::TN; ++t) {
#pragma unroll
        for (int b = 0; b < C::TM; ++b) {
            const int k = t * C::TM + b;
            mfma_i8_acc(acc[t][b], v.a[CUR][t], v.b[CUR][b]);
#pragma unroll
            for (int f = 0; f < F; ++f)  // fragment f in the first three quarters of the steps: x's first, then w's
                if (f * 3 * S / (4 * F) == k) {
                    if (f < C::TM)
                        v.b[1 - CUR][f] = *reinterpret_cast<const u4*>(bp + 2048 * f);
                    else if (ACT && f - C::TM >= C::TN / 2)
                        v.a[1 - CUR][f - C::TM] = *reinterpret_cast<const u4*>(ap + 64 * C::BN + 2048 * (f - C::TM - C::TN / 2));
                    else
                        v.a[1 - CUR][f - C::TM] = *reinterpret_cast<const u4*>(ap + 2048 * (f - C::TM));
                }
            if constexpr (LOAD) gemm8_loads_at<0, S, C, ACT>(k, slot, l, xr, wr, ur, koff, tail);
            TW4_STEP_FENCE;
        }
    }
}

template <class C, bool ACT>
__device__ __forceinline__ void gemm8_read(u4 (&a)[C::TN], u4 (&b)[C::TM], const char* ap, const char* bp) {
#pragma unroll
    for (int f = 0; f < C::TM; ++f) b[f] = *reinterpret_cast<const u4*>(bp + 2048 * f);
#pragma unroll
    for (int f = 0; f < C::TN; ++f)
        a[f] = *reinterpret_cast<const u4*>(ap + (ACT && f >= C::TN / 2 ? 64 * C::BN + 2048 * (f - C::TN / 2) : 2048 * f));
}

// The splits' sums of a tile: each workgroup stores its own, the last to arrive adds the others' to its own (whole numbers: any order
// gives the same), returns the tile's counter to zero and goes on to the epilogue (true). Stores and loads are coherent across the
// XCDs' caches as in finish_unit; the barrier orders every wavefront's stores before the count.
template <class C>
__device__ __forceinline__ bool gemm8_join(i4 (&acc)[C::TN][C::TM], int splits, int tile, int split, int wave, int lane, int tid,
                                           int* __restrict__ ws, int* __restrict__ locks, int* flag) {
    constexpr int F = C::TN * C::TM, FC = F % 8 == 0 ? 8 : F % 6 == 0 ? 6 : F;  // fragments of a wavefront, and how many are loaded at a time
    static_assert(F % FC == 0, "whole rounds");
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(ws, 0, 0x7FFFFFFF, kBufferFlags);
    const auto part = [&](int s) { return ((tile * splits + s) * C::WAVES + wave) * (F * 1024); };  // bytes, below 2^31 (host)
    const int mine = part(split);
#pragma unroll
    for (int t = 0; t < C::TN; ++t)
#pragma unroll
        for (int b = 0; b < C::TM; ++b)
            __builtin_amdgcn_raw_buffer_store_b128(bitcast<u4>(acc[t][b]), rs, ((t * C::TM + b) * 64 + lane) * 16, mine, kCoherentAux);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) *flag = __hip_atomic_fetch_add(locks + tile, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == splits - 1;
    __syncthreads();
    const bool last = *flag;
    __syncthreads();  // the flag's place is free again
    if (!last) return false;
    for (int s = 1; s < splits; ++s) {
        const int other = part(split + s < splits ? split + s : split + s - splits);
#pragma unroll
        for (int f0 = 0; f0 < F; f0 += FC) {
            u4 p[FC];
#pragma unroll
            for (int f = 0; f < FC; ++f) p[f] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(rs, ((f0 + f) * 64 + lane) * 16, other, kCoherentAux));
#pragma unroll
            for (int f = 0; f < FC; ++f) {
                acc[(f0 + f) / C::TM][(f0 + f) % C::TM] += bitcast<i4>(p[f]);
                asm volatile("" : "+a"(acc[(f0 + f) / C::TM][(f0 + f) % C::TM]));  // back where the loop left it
            }
        }
    }
    if (tid == 0) __hip_atomic_store(locks + tile, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}

template <class C, bool ACT, bool BF16>
__global__ void __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(C::PER_SIMD)))
gemm8_lds_kernel(const int8_t* __restrict__ x, uint32_t x_stride, const float* __restrict__ x_scale, const int8_t* __restrict__ w,
                 uint32_t w_stride, const float* __restrict__ w_scale, uint16_t* __restrict__ y, int* __restrict__ ws,
                 int* __restrict__ locks, int M, int N, int K, int mb, int nb, int splits) {
    __shared__ u4 ring[C::R * C::SLOT / 16];
    static_assert(!ACT || (C::TN % 2 == 0 && C::WI % 2 == 0), "gate and up in pairs of tiles, and apart in the loads");
    constexpr int TM = C::TM, TN = C::TN, R = C::R;
    constexpr int FEATURES = ACT ? C::BN / 2 : C::BN;  // of the output
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave % C::WN, wm = wave / C::WN, r = lane & 15, q = lane >> 4;
    const int out = ACT ? N >> 1 : N;

    // work unit -> (tile, split); tiles in bands of 8 token blocks, each XCD a contiguous range
    const int unit = xcd_remap(blockIdx.x, gridDim.x);
    const int tile = unit / splits, split = unit - tile * splits;
    const int band = tile / (8 * nb), band_rows = min(mb - band * 8, 8), rin = tile - band * 8 * nb;
    const int m0 = (band * 8 + rin % band_rows) * C::BM, n0 = rin / band_rows * FEATURES;

    Gemm8Loads<C> l;
    const int rows = min(M - m0, C::BM), features = min(out - n0, FEATURES);
    l.x = lds_rsrc(x + static_cast<int64_t>(m0) * x_stride);
    l.w = lds_rsrc(w + static_cast<int64_t>(n0) * w_stride);
    l.up = ACT ? lds_rsrc(w + static_cast<int64_t>(out + n0) * w_stride) : l.w;
    const uint32_t x_size = static_cast<uint32_t>(rows - 1) * x_stride + K, w_size = static_cast<uint32_t>(features - 1) * w_stride + K;
    l.x.z = x_size;
    l.w.z = l.up.z = w_size;
    // load j (rows 8 j .. 8 j + 7 of its operand) is wavefront j % WAVES's
    const int chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
#pragma unroll
    for (int i = 0; i < C::XI; ++i) l.xoff[i] = static_cast<uint32_t>(min(8 * (i * C::WAVES + wave) + (lane >> 3), rows - 1)) * x_stride + 16 * chunk;
#pragma unroll
    for (int i = 0; i < C::WI; ++i) {
        const int row = (8 * (i * C::WAVES + wave) + (lane >> 3)) % FEATURES;
        l.woff[i] = static_cast<uint32_t>(min(row, features - 1)) * w_stride + 16 * chunk;
    }
    l.lds = 1024 * wave;
    const int all = (K + 127) >> 7;  // stages of the tile, of which this unit has [first, first + stages), one at least
    const int first = static_cast<int>(static_cast<int64_t>(split) * all / splits);
    const int stages = static_cast<int>(static_cast<int64_t>(split + 1) * all / splits) - first;
    const uint32_t past = 128 * (all - 1) + 16 * chunk >= K ? 0x80000000u : 0u;  // in the tile's last stage

    const uint32_t ring_addr = static_cast<uint32_t>(reinterpret_cast<size_t>((lds_void*)ring));
    const auto issue_all = [&](int st, int slot) {
        u4 xr = l.x, wr = l.w, ur = l.up;
        const bool on = st < stages;
        xr.z = __builtin_amdgcn_readfirstlane(on ? x_size : 0u);
        wr.z = ur.z = __builtin_amdgcn_readfirstlane(on ? w_size : 0u);
        gemm8_loads_at<0, 1, C, ACT>(0, ring_addr + slot * C::SLOT, l, xr, wr, ur, 128u * (first + st), first + st == all - 1 ? past : 0u);
    };
    i4 acc[TN][TM];
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int b = 0; b < TM; ++b) acc[t][b] = i4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < R; ++s) issue_all(s, s);

    // this lane's first fragments in a slot, substep 0 (substep 1: ^ 64)
    const int at = 128 * r + 16 * (q ^ (r >> 1));
    const int bo = 2048 * TM * wm + at, ao = 128 * C::BM + 2048 * (ACT ? TN / 2 : TN) * wn + at;
    const char* base = reinterpret_cast<const char*>(ring);
    Gemm8Regs<C> regs;
    wait_stage<(R - 1) * C::LOADS>();
    ring_barrier();
    gemm8_read<C, ACT>(regs.a[0], regs.b[0], base + ao, base + bo);
    int slot = 0;
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int b = 0; b < TM; ++b) asm volatile("" : "+a"(acc[t][b]));
    asm volatile("s_nop 4" ::: "memory");  // the zeros are written before the first product reads them
    for (int i = 0; i < stages; ++i) {
        const char* cur = base + slot * C::SLOT;
        const uint32_t cur_addr = ring_addr + slot * C::SLOT;
        slot = slot + 1 == R ? 0 : slot + 1;
        const char* nxt = base + slot * C::SLOT;
        const u4 none{};
        gemm8_substep<C, 0, false, ACT>(regs, acc, cur + (ao ^ 64), cur + (bo ^ 64), 0, l, none, none, none, 0, 0);
        wait_stage<(R - 2) * C::LOADS>();
        ring_barrier();
        const int st = i + R;
        u4 xr = l.x, wr = l.w, ur = l.up;
        const bool on = st < stages;
        xr.z = __builtin_amdgcn_readfirstlane(on ? x_size : 0u);
        wr.z = ur.z = __builtin_amdgcn_readfirstlane(on ? w_size : 0u);
        gemm8_substep<C, 1, true, ACT>(regs, acc, nxt + ao, nxt + bo, cur_addr, l, xr, wr, ur, 128u * (first + st),
                                       first + st == all - 1 ? past : 0u);
    }
    // The epilogue. Each wavefront has its part of the ring for itself: the scales of its tokens and rows of w, and TB token tiles of
    // results.
    constexpr int TILES = ACT ? TN / 2 : TN;
    constexpr int PART = C::LDS_BYTES / C::WAVES / 16 * 16, SCALES = 64 * (TM + TN);  // bytes
    constexpr int ROW = 32 * TILES + 16;  // a token's results, 16 bytes behind them against bank conflicts
    constexpr int FIT = (PART - SCALES) / (16 * ROW);
    constexpr int TB = FIT >= TM ? TM : FIT >= TM / 2 && TM % 2 == 0 ? TM / 2 : 1;
    static_assert(FIT >= 1 && TM % TB == 0, "one token tile at least");
    constexpr int PER_LANE = (TM + TN + 3) / 4;
    float scale[PER_LANE];
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {  // tokens first, then rows of w: gate rows, then up rows
        const int at = 64 * i + lane, f = at - 16 * TM;
        const int n = min(n0 + 16 * TILES * wn + f % (16 * TILES), out - 1) + (f >= 16 * TILES ? out : 0);
        if (at < 16 * TM)
            scale[i] = x_scale[min(m0 + 16 * TM * wm + at, M - 1)];
        else if (f < 16 * TN)
            scale[i] = w_scale[n];
    }
    wait_stage<0>();  // the empty loads past the end still write their slots
    ring_barrier();   // in every wavefront: the ring is free
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");  // the last products have been written back
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int b = 0; b < TM; ++b) asm volatile("" : "+a"(acc[t][b]));

    if (splits > 1) {
        if (!gemm8_join<C>(acc, splits, tile, split, wave, lane, tid, ws, locks, reinterpret_cast<int*>(ring))) return;  // the ring is done with
    }

    char* mine = reinterpret_cast<char*>(ring) + wave * PART;
    float* scales = reinterpret_cast<float*>(mine + PART - SCALES);
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i)
        if (64 * i + lane < 16 * (TM + TN)) scales[64 * i + lane] = scale[i];
    wave_fence();
    // the four features of tile t, token tile b, that this lane holds
    const auto values = [&](int t, int b, float (&v)[4]) {
        const float xs = scales[16 * b + r];
        const f4 s = *reinterpret_cast<const f4*>(scales + 16 * (TM + t) + 4 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(acc[t][b][i]) * xs * s[i];
        if constexpr (ACT) {
            const f4 u = *reinterpret_cast<const f4*>(scales + 16 * (TM + TILES + t) + 4 * q);
            silu_values(v);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] *= static_cast<float>(acc[t + TILES][b][i]) * xs * u[i];
        }
    };
    // Results go through LDS, so that a store instruction writes whole rows of the wavefront's features: 8 values a lane where rows are
    // that aligned, else 2 or 1.
    const int width = (out & 7) == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0  ? 8
                      : (out & 1) == 0 && (reinterpret_cast<uintptr_t>(y) & 3) == 0 ? 2
                                                                                     : 1;
#pragma unroll
    for (int b0 = 0; b0 < TM; b0 += TB) {
#pragma unroll
        for (int b = b0; b < b0 + TB; ++b)
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                TW4_STEP_FENCE;  // one tile's values at a time: all of them at once do not fit the registers
                float v[4];
                values(t, b, v);
                *reinterpret_cast<u2*>(mine + (16 * (b - b0) + r) * ROW + 32 * t + 8 * q) =
                    u2{value16<BF16>(v[0]) | value16<BF16>(v[1]) << 16, value16<BF16>(v[2]) | value16<BF16>(v[3]) << 16};
            }
        wave_fence();
        uint16_t* to = y + static_cast<int64_t>(m0 + 16 * (TM * wm + b0)) * out + n0 + 16 * TILES * wn;
        const int rows = min(M - m0 - 16 * (TM * wm + b0), 16 * TB), columns = min(out - n0 - 16 * TILES * wn, 16 * TILES);
        if (width == 8)
            store_rows<8, 16 * TB, 16 * TILES, ROW, u4>(to, out, mine, rows, columns, lane);
        else if (width == 2)
            store_rows<2, 16 * TB, 16 * TILES, ROW, uint32_t>(to, out, mine, rows, columns, lane);
        else
            store_rows<1, 16 * TB, 16 * TILES, ROW, uint16_t>(to, out, mine, rows, columns, lane);
        wave_fence();
    }
}

template <class C, bool ACT, bool BF16>
int gemm8_lds_launch(const Gemm8Args& a, int splits) {
    constexpr int FEATURES = ACT ? C::BN / 2 : C::BN;
    const int out = ACT ? a.N / 2 : a.N, mb = (a.M + C::BM - 1) / C::BM, nb = (out + FEATURES - 1) / FEATURES;
    const int64_t units = static_cast<int64_t>(mb) * nb * splits;
    TW4_REQUIRE(units * C::THREADS < int64_t(1) << 32, TW4_EINVAL, "gemm_int8: too many tiles (M %d, N %d)", a.M, a.N);
    if (splits > 1) {
        const int64_t ints = units * C::BM * C::BN;
        TW4_REQUIRE(a.ws && a.locks, TW4_EINVAL, "gemm_int8: splits take a workspace");
        TW4_REQUIRE(ints <= a.ws_words && ints < kMaxPartialFloats && static_cast<int64_t>(mb) * nb <= a.n_locks, TW4_ESPACE,
                    "gemm_int8: %lld partial sums and %d counters", static_cast<long long>(ints), mb * nb);
    }
    gemm8_lds_kernel<C, ACT, BF16><<<static_cast<unsigned>(units), C::THREADS, 0, a.st>>>(
        a.x, static_cast<uint32_t>(a.x_stride), a.x_scale, a.w, static_cast<uint32_t>(a.w_stride), a.w_scale, a.y, a.ws, a.locks, a.M, a.N,
        a.K, mb, nb, splits);
    TW4_LAUNCH_CHECK("gemm_int8: launch");
    return TW4_OK;
}

template <int TM, int TN, int WM, int WN, int R, bool ACT, bool BF16>
int gemm8_lds_near(const Gemm8Args& a, int splits) {
    // one tile of tokens: w is read once, by loads that do not keep it
    if constexpr (16 * TM * WM <= 128)
        if (a.M <= 16 * TM * WM) return gemm8_lds_launch<Gemm8Cfg<TM, TN, WM, WN, R, true>, ACT, BF16>(a, splits);
    if constexpr (16 * TM * WM > 16) return gemm8_lds_launch<Gemm8Cfg<TM, TN, WM, WN, R, false>, ACT, BF16>(a, splits);
    tw4host::set_error("gemm_int8: a tile of %d tokens (M %d)", 16 * TM * WM, a.M);
    return TW4_ECONFIG;
}

template <int TM, int TN, int WM, int WN, int R>
int gemm8_lds_any(const Gemm8Args& a, int splits) {
    static_assert(TN % 2 == 0, "gate and up in pairs of tiles");
    if (a.act) return a.bf16 ? gemm8_lds_near<TM, TN, WM, WN, R, true, true>(a, splits) : gemm8_lds_near<TM, TN, WM, WN, R, true, false>(a, splits);
    return a.bf16 ? gemm8_lds_near<TM, TN, WM, WN, R, false, true>(a, splits) : gemm8_lds_near<TM, TN, WM, WN, R, false, false>(a, splits);
}

int gemm8_lds(const Gemm8Args& a, int kernel, int splits) {
    switch (kernel) {
#define TW4_CASE(ID, TM, TN, WM, WN, R) \
    case ID: return gemm8_lds_any<TM, TN, WM, WN, R>(a, splits);
        TW4_GEMM8_LDS(TW4_CASE)
#undef TW4_CASE
        default: break;
    }
    tw4host::set_error("gemm_int8: kernel %d", kernel);
    return TW4_ECONFIG;
}

}  // namespace tw4

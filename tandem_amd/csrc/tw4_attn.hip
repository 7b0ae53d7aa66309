// Causal attention of new tokens over a paged cache, grouped-query heads. Request i of the batch has len_i keys in its pages, the
// last n_i of them those of its new tokens (rows start_i .. start_i + n_i - 1 of q); new token t sees the keys
// j <= len_i - n_i + t:
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale (q . k_j) - max)
//
// in one pass over the keys with a running maximum and sum in fp32 (the online softmax: when a block of keys raises the maximum,
// what was summed so far is scaled by exp(old - new)).
//
// The G = heads / kv_heads query heads of a KV head are rows of one tile, row r = t G + g, so a KV head's keys are read once for
// all of them. Scores are computed transposed, S^T = K Q^T: a lane of the matrix instruction's result then holds one row's scores
// of several keys, its limit, maximum and sum are one register each, and its probabilities are already where the second
// product O^T = V^T P^T wants them (the order of keys inside a product is free: K's rows and V^T's columns only have to agree).
// Probabilities are rounded to the cache's type for that product (at most half a step of the type, relative, each: the same size
// as the rounding of the result); their sum is of the unrounded values. fp16 has 14 binary places below 1 before its steps stop shrinking,
// and a long context can hold many keys of less than that each, so there both sums are of 2^14 p (2^6 p in the chunk kernel, whose p reaches
// 2^8): the factor cancels in their quotient.
//
// Rows kernel: a workgroup has one tile of 16 MT rows and a range of keys; its four wavefronts take blocks of 32 keys in turn, each
// with a softmax of its own, joined at the end. K comes straight into registers (a lane has 16 bytes of a key: half lines, which the
// first-level cache joins, so they are ordinary loads), V as whole rows past the caches and through a wavefront's own LDS, read back
// transposed; both a block ahead. It is bound by reading K and V: 3 requests of 40002 keys, 16 + 8 heads of 128, 75-77 us (6.4-6.6 TB/s; a plain
// read reaches 7.1), 32 of 1 to 8192 keys, 32 + 8 heads, 91-94 (5.8-6.0). Measured and not kept: V by ordinary loads 113 us at 32 requests against 92, K
// through LDS as well 100, three wavefronts per SIMD (they spill) 95. With few rows in flight the keys are split over up to `splits`
// workgroups; the last to arrive joins their results in order: one request of 1024 keys 9.4-9.6 us, most of it seven dependent round trips
// to memory (length, table, keys, store of the partial result, counter, load of all of them, store of the row), of 32001 keys 31.
//
// Tiles of 128 rows (chunks of prompts): the chunk kernel below. Its K and V are read by 128 rows at a time from LDS.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "tw4_attn.h"
#include "tw4_lds.h"

namespace tw4 {

struct AttnArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const int32_t* table;
    const int32_t* lens;
    const int32_t* starts;  // null: one row per request
    uint16_t* out;          // [tokens, heads, D]
    float* ws;
    int32_t* locks;
    int64_t q_token, q_head, page_stride, head_stride, token_stride, table_stride;
    float scale;  // times log2(e)
    int tokens, batch, heads, kv_heads, group, num_pages, width, shift, splits, part_rows;
};

constexpr int kTileFloats = 4;  // per row of a partial result beside its D sums: maximum, sum, and two that keep rows 16-byte aligned
constexpr int kMinKeys = 128;  // of a split

// A tile of rows: its request, first row, and the keys it can see.
struct Tile {
    int request, first, rows;  // rows of the request from `first` on, at least 1
    int start, before;         // the request's first token; keys before its new tokens' own: token t sees before + t and all below
};

// Slot s of the grid is the first tile of request s, and from slot `batch` on a further one: of request i, the last with
// base_i = floor(start_i G / B) <= s - batch. A request has at most floor(n_i G / B) of those, and the base of the next is at least as far
// on, so no scan of the lengths is needed; slots past a request's rows have none. So the slots of requests of one tile each, which
// most calls have, lie together: with one or two slots in turn for a request, where the second is empty, the work gathered on half of the
// shader engines (3 requests of 2 new tokens, 64 + 8 heads, 8000 keys: 31.6 us against 28.2; 40
// of 8, 32 + 8 heads, 3000 keys: 108 against 88).
template <int B>
__device__ __forceinline__ bool find_tile(const AttnArgs& a, int slot, int lane, Tile& t) {
    int start, have;  // tokens of the request that q has
    int64_t fresh;    // new tokens that its keys count, those behind q's last row among them
    if (a.starts) {
        t.request = slot, t.first = 0;
        if (slot >= a.batch) {
            slot -= a.batch;
            int lo = 0, step = 64;  // a wavefront looks at 64 requests at a time
            while (step < a.batch) step *= 64;
            for (; step > 1;) {
                step /= 64;
                const int64_t i = lo + static_cast<int64_t>(lane) * step;
                bool before = false;
                if (i < a.batch) before = static_cast<int64_t>(min(max(a.starts[i], 0), a.tokens)) * a.group / B <= slot;
                lo += step * max(__popcll(__ballot(before)) - 1, 0);
            }
            t.request = __builtin_amdgcn_readfirstlane(lo);
            const int64_t base = static_cast<int64_t>(min(max(a.starts[t.request], 0), a.tokens)) * a.group / B;
            t.first = (slot - static_cast<int>(base) + 1) * B;
        }
        const int from = a.starts[t.request], to = a.starts[t.request + 1];
        start = min(max(from, 0), a.tokens);
        have = min(max(to, start), a.tokens) - start;
        fresh = static_cast<int64_t>(to) - from;
    } else {
        const int per = (a.group + B - 1) / B;
        t.request = slot / per;
        start = t.request;
        have = 1, fresh = 1;
        t.first = (slot - t.request * per) * B;
    }
    t.start = start;
    // with rows there is fresh >= have, so before + t < len; no token number reaches 2^30, so what lies further down sees nothing either
    t.before = static_cast<int>(max(max(a.lens[t.request], 0) - fresh, static_cast<int64_t>(-(1 << 30))));
    t.rows = have * a.group - t.first;
    return t.first >= 0 && t.rows > 0;
}

// Where the 16 bytes of chunk c of row r lie in a wavefront's V tile of D-value rows: the chunks of a row change places with
// the row in pairs of 32 bytes, so that a transposed read (4 rows of 32 bytes for each 16 lanes) meets every bank once.
template <int D>
__device__ __forceinline__ int v_chunk(int r, int c) {
    return D == 128 ? r * 16 + (c ^ ((r & 7) << 1)) : r * 8 + (c ^ (((r >> 1) & 3) << 1));
}

__device__ __forceinline__ u2 read_tr(const u4* lds, int byte) {
    typedef __attribute__((address_space(3))) s4 lds_s4;
    return bitcast<u2>(__builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s4*)(reinterpret_cast<const char*>(lds) + byte)));
}

// Largest of the four values a column has in lanes c, c + 16, c + 32, c + 48. A NaN is passed over.
__device__ __forceinline__ float max_rows(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float s = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(s), __float_as_uint(s), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ bool odd16(uint32_t v, uint32_t exponent) {  // either half infinite or NaN
    return (v & exponent) == exponent || ((v >> 16) & exponent) == exponent;
}

// The page table by scalar loads: no kernel here writes it.
typedef const __attribute__((address_space(4))) int32_t const_int;

__device__ __forceinline__ u4 read_odd_free(u4 w, uint32_t exponent) {  // infinities and NaN of 16-bit halves as zero
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & exponent) == exponent) w[i] &= 0xFFFF0000u;
        if (((w[i] >> 16) & exponent) == exponent) w[i] &= 0xFFFFu;
    }
    return w;
}

constexpr float kNone = -__builtin_inff();

// Probabilities of at most 2^BITS are summed times 2^kLift, up to 2^14 of fp16's 2^16 (bf16 has fp32's exponents).
template <typename T, int BITS>
constexpr float kLift = __is_same(T, h1) ? 14 - BITS : 0;

template <typename T, int D, int MT>
__global__ void __launch_bounds__(256, 2) rows_kernel(AttnArgs a) {
    constexpr int B = 16 * MT, KS = D / 32, DT = D / 16, C = D / 8, VJ = C / 2;  // VJ: 1 KB loads of 32 keys
    constexpr uint32_t kExponent = __is_same(T, h1) ? 0x7C00u : 0x7F80u;
    static_assert(32 * D * 2 * 4 >= 4 * 16 * D * 4, "the join of 16 rows uses the V tiles' LDS");
    __shared__ u4 lds[4 * 32 * C];
    __shared__ float stat[2][4][B];
    __shared__ int last_flag;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15, g4 = lane >> 4;
    const int slot = blockIdx.x / a.kv_heads, head = blockIdx.x - slot * a.kv_heads, split = blockIdx.y;
    Tile t;
    if (!find_tile<B>(a, slot, lane, t)) return;

    // this lane's rows: limits (last key seen), queries
    int limit[MT], low = 0x7FFFFFFF, high = -1;
    u4 q[MT][KS];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int r = t.first + 16 * m + c16;
        const bool there = 16 * m + c16 < t.rows;
        const int tok = r / a.group, g = r - tok * a.group;
        limit[m] = there ? t.before + tok : -1;
        if (there) low = min(low, limit[m]), high = max(high, limit[m]);
        const uint16_t* src = a.q + (t.start + tok) * a.q_token + (head * a.group + g) * a.q_head + 8 * g4;
#pragma unroll
        for (int s = 0; s < KS; ++s) q[m][s] = there ? *reinterpret_cast<const u4*>(src + 32 * s) : u4{0, 0, 0, 0};
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) low = min(low, __shfl_xor(low, d)), high = max(high, __shfl_xor(high, d));
    low = __builtin_amdgcn_readfirstlane(low), high = __builtin_amdgcn_readfirstlane(high);

    // keys [0, end), this workgroup's share [begin, stop) of them
    const int end = static_cast<int>(min(static_cast<int64_t>(high) + 1, static_cast<int64_t>(a.width) << a.shift));
    int begin = 0, stop = max(end, 0), parts = 1;
    if (a.splits > 1 && end > 0) {
        const int share = max((end + a.splits - 1) / a.splits, kMinKeys);
        const int whole = (share + 127) & ~127;
        parts = (end + whole - 1) / whole;
        if (split >= parts) return;
        begin = split * whole;
        stop = min(end, begin + whole);
    } else if (split > 0) {
        return;
    }

    f4 o[MT][DT];
    float top[MT], sum[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        top[m] = kNone, sum[m] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[m][d] = f4{0, 0, 0, 0};
    }
    u4* vt = lds + wave * 32 * C;
    const_int* table = (const_int*)(a.table + t.request * a.table_stride);
    const char* kh = reinterpret_cast<const char*>(a.k + head * a.head_stride);
    const char* vh = reinterpret_cast<const char*>(a.v + head * a.head_stride);
    const int final16 = (stop - 1) & ~15;  // the last 16 keys that are there
    const uint32_t token_bytes = static_cast<uint32_t>(a.token_stride) * 2;

    // A block of 32 keys is two halves of 16, each in one page. Table entries are fetched a block before the keys they lead to,
    // K a block before its product, V a block before it goes to LDS: each load has a block's arithmetic to arrive in.
    u4 kf[2][KS], vf[VJ];
    auto pages = [&](int base) {
        return int2{table[min(base, final16) >> a.shift], table[min(base + 16, final16) >> a.shift]};
    };
    auto there = [&](int page) { return static_cast<uint32_t>(page) < static_cast<uint32_t>(a.num_pages); };
    // byte offset of half h's first key; a page the table does not have is page 0, read and left out
    auto offset = [&](int base, int h, int page) {
        const int first = min(base + 16 * h, final16);
        return ((there(page) ? page : 0) * a.page_stride + (first & ((1 << a.shift) - 1)) * a.token_stride) * 2;
    };
    auto last_row = [&](int base, int h) { return min(stop - 1 - min(base + 16 * h, final16), 15); };
    auto load_k = [&](int base, int2 page) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const char* src = kh + offset(base, h, h ? page.y : page.x);
            const uint32_t lane_off = min(c16, last_row(base, h)) * token_bytes + 16 * g4;
#pragma unroll
            for (int s = 0; s < KS; ++s) kf[h][s] = *reinterpret_cast<const u4*>(src + (lane_off + 64 * s));
        }
    };
    auto load_v = [&](int base, int2 page) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const char* src = vh + offset(base, h, h ? page.y : page.x);
            const int last = last_row(base, h);
#pragma unroll
            for (int j = 0; j < VJ / 2; ++j)  // chunk lane % C of row lane / C + j (64 / C)
                vf[h * (VJ / 2) + j] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(
                    src + (min(lane / C + j * (64 / C), last) * token_bytes + 16 * (lane % C))));
        }
    };
    auto block = [&](int base, int2 page, int2 next, auto more, auto careful) {
        constexpr bool kMore = decltype(more)::value, kMasked = decltype(careful)::value;
        const int absent = (there(page.x) ? 0 : 1) | (there(page.y) ? 0 : 2);
        f4 s[MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m) s[m][0] = s[m][1] = f4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                s[m][0] = mma16<T>(kf[0][i], q[m][i], s[m][0]);
                s[m][1] = mma16<T>(kf[1][i], q[m][i], s[m][1]);
            }
        if constexpr (kMore) load_k(base + 128, next);
        // A probability of zero does not take an infinity or NaN away: where some row does not see a key, such values are left out
        // of the product and added to the rows that see them.
        bool odd = false;
        if constexpr (kMasked) {
#pragma unroll
            for (int j = 0; j < VJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) odd |= odd16(vf[j][i], kExponent);
            odd = __ballot(odd) != 0;
        }
#pragma unroll
        for (int j = 0; j < VJ; ++j) vt[v_chunk<D>(lane / C + j * (64 / C), lane % C)] = vf[j];
        if constexpr (kMore) load_v(base + 128, next);

        u4 p[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = s[m][i >> 2][i & 3] * a.scale;
            if constexpr (kMasked) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int key = base + 16 * (i >> 2) + 4 * g4 + (i & 3);
                    if (key > min(limit[m], stop - 1) || (absent >> (i >> 2) & 1)) x[i] = kNone;
                }
            }
            float high8 = x[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) high8 = fmaxf(high8, x[i]);
            const float now = fmaxf(top[m], max_rows(high8));
            const float zero = now == kNone ? 0.0f : now;  // a row that has seen nothing yet
            const float keep = __builtin_amdgcn_exp2f(top[m] - zero), lifted = zero - kLift<T, 0>;
            top[m] = now;
            sum[m] *= keep;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = __builtin_amdgcn_exp2f(x[i] - lifted);
                sum[m] += x[i];
            }
            p[m] = from_f32<T>(x);
#pragma unroll
            for (int d = 0; d < DT; ++d) o[m][d] *= keep;
        }
        // V back, transposed: 4 rows x 16 columns for each 16 lanes
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
        if (kMasked && odd) {
#pragma unroll 1
            for (int key = 0; key < 32; ++key)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if (base + key > min(limit[m], stop - 1) || (absent >> (key >> 4) & 1)) continue;
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        const u2 four = *reinterpret_cast<const u2*>(reinterpret_cast<const char*>(vt) +
                                                                     v_chunk<D>(key, 2 * d + (g4 >> 1)) * 16 + (g4 & 1) * 8);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint16_t bits = static_cast<uint16_t>(four[i >> 1] >> (16 * (i & 1)));
                            if ((bits & kExponent) == kExponent) o[m][d][i] += static_cast<float>(bitcast<T>(bits));
                        }
                        __builtin_amdgcn_sched_barrier(0);  // one at a time: the rare path is not to take registers
                    }
                }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int r = 4 * g4 + (c16 >> 2), c = 2 * d + ((c16 & 3) >> 1), half = (c16 & 1) * 8;
            const u2 lo = read_tr(vt, v_chunk<D>(r, c) * 16 + half), hi = read_tr(vt, v_chunk<D>(r + 16, c) * 16 + half);
            u4 w = u4{lo.x, lo.y, hi.x, hi.y};
            if (kMasked && odd) w = read_odd_free(w, kExponent);
#pragma unroll
            for (int m = 0; m < MT; ++m) o[m][d] = mma16<T>(w, p[m], o[m][d]);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
    };
    // Blocks that every row sees whole come first and run without a mask; from the first one that some row does not (or a page
    // that is none) on, all are masked.
    int base = begin + 32 * wave;
    if (base < stop) {
        int2 page = pages(base), next = pages(min(base + 128, final16));
        load_k(base, page);
        load_v(base, page);
        const int clear = min(low + 1, stop);
        auto step = [&](auto careful) {
            const int2 after = pages(min(base + 256, final16));
            block(base, page, next, std::true_type(), careful);
            page = next, next = after;
            base += 128;
        };
        while (base + 128 < stop && base + 32 <= clear && there(page.x) && there(page.y)) step(std::false_type());
        while (base + 128 < stop) step(std::true_type());
        block(base, page, next, std::false_type(), std::true_type());
    }

    // the four wavefronts' results become one, 16 rows at a time through LDS
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const float l = sum_rows(sum[m]);
        if (g4 == 0) stat[0][wave][16 * m + c16] = top[m], stat[1][wave][16 * m + c16] = l;
    }
    float* od = reinterpret_cast<float*>(lds);  // [wave][row][D]
    constexpr int PER = D / 16;                 // values of a row per thread: row threadIdx / 16
    const int row = threadIdx.x >> 4, col = (threadIdx.x & 15) * PER;
    const int unit = slot * a.kv_heads + head;
    constexpr int kRowFloats = D + kTileFloats;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(a.ws, 0, 0x7FFFFFFF, kBufferFlags);
    float res[MT][PER], rtop[MT], rsum[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f4*>(od + (wave * 16 + c16) * D + 16 * d + 4 * g4) = o[m][d];
        __syncthreads();
        rtop[m] = kNone;
#pragma unroll
        for (int w = 0; w < 4; ++w) rtop[m] = fmaxf(rtop[m], stat[0][w][16 * m + row]);
        const float zero = rtop[m] == kNone ? 0.0f : rtop[m];
        rsum[m] = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) res[m][i] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            // a wavefront without keys has sums of zero
            const float f = __builtin_amdgcn_exp2f(stat[0][w][16 * m + row] - zero);
            rsum[m] += f * stat[1][w][16 * m + row];
#pragma unroll
            for (int i = 0; i < PER; ++i) res[m][i] += f * od[(w * 16 + row) * D + col + i];
        }
    }
    if (parts > 1) {
        // [unit][split][row][D + 4]: the sums, then maximum and sum; rows that are there only
        const int64_t mine = (static_cast<int64_t>(unit) * a.splits + split) * a.part_rows;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (16 * m + row >= t.rows) continue;
            const int to = static_cast<int>((mine + 16 * m + row) * kRowFloats * 4);
#pragma unroll
            for (int i = 0; i < PER; i += 4)
                __builtin_amdgcn_raw_buffer_store_b128(bitcast<u4>(f4{res[m][i], res[m][i + 1], res[m][i + 2], res[m][i + 3]}), rs,
                                                       to + (col + i) * 4, 0, kCoherentAux);
            if (col == 0)
                __builtin_amdgcn_raw_buffer_store_b64(u2{__float_as_uint(rtop[m]), __float_as_uint(rsum[m])}, rs, to + D * 4, 0,
                                                      kCoherentAux);
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (threadIdx.x == 0)
            last_flag = __hip_atomic_fetch_add(a.locks + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
        __syncthreads();
        if (!last_flag) return;
        // Of the 16 rows' threads those of rows that are not there help with the others: 16 / R groups of R rows (R a power of two) take
        // every (16 / R)-th part, eight of them in flight, and are added in order.
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int have = min(t.rows - 16 * m, 16);
            if (have <= 0) break;
            const int bits = have > 8 ? 4 : have > 4 ? 3 : have > 2 ? 2 : have - 1;
            const int jrow = min(row & ((1 << bits) - 1), have - 1), group = row >> bits, groups = 16 >> bits;
            float jtop = kNone, jsum = 0.0f, jres[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) jres[i] = 0.0f;
            constexpr int VB = 8;
            for (int s0 = group; s0 < parts; s0 += VB * groups) {
                u2 ms[VB];
                f4 x[VB][PER / 4];
#pragma unroll
                for (int v = 0; v < VB; ++v) {
                    const int s = min(s0 + v * groups, parts - 1);  // past the last: read again, not added
                    const int from = static_cast<int>(
                        ((static_cast<int64_t>(unit) * a.splits + s) * a.part_rows + 16 * m + jrow) * kRowFloats * 4);
                    ms[v] = bitcast<u2>(__builtin_amdgcn_raw_buffer_load_b64(rs, from + D * 4, 0, kCoherentAux));
#pragma unroll
                    for (int i = 0; i < PER / 4; ++i)
                        x[v][i] = bitcast<f4>(__builtin_amdgcn_raw_buffer_load_b128(rs, from + (col + 4 * i) * 4, 0, kCoherentAux));
                }
                float now = jtop;
#pragma unroll
                for (int v = 0; v < VB; ++v) now = fmaxf(now, __uint_as_float(ms[v].x));
                const float zero = now == kNone ? 0.0f : now, keep = __builtin_amdgcn_exp2f(jtop - zero);
                jtop = now;
                jsum *= keep;
#pragma unroll
                for (int i = 0; i < PER; ++i) jres[i] *= keep;
#pragma unroll
                for (int v = 0; v < VB; ++v) {
                    if (s0 + v * groups >= parts) break;
                    const float f = __builtin_amdgcn_exp2f(__uint_as_float(ms[v].x) - zero);
                    jsum += f * __uint_as_float(ms[v].y);
#pragma unroll
                    for (int i = 0; i < PER; ++i) jres[i] += f * x[v][i >> 2][i & 3];
                }
            }
            __syncthreads();
            if ((threadIdx.x & 15) == 0) stat[0][0][row] = jtop, stat[1][0][row] = jsum;
#pragma unroll
            for (int i = 0; i < PER; ++i) od[row * D + col + i] = jres[i];
            __syncthreads();
            rtop[m] = kNone, rsum[m] = 0.0f;
            for (int g = 0; g < groups; ++g) rtop[m] = fmaxf(rtop[m], stat[0][0][(g << bits) + jrow]);
            const float zero = rtop[m] == kNone ? 0.0f : rtop[m];
#pragma unroll
            for (int i = 0; i < PER; ++i) res[m][i] = 0.0f;
            for (int g = 0; g < groups; ++g) {
                const float f = __builtin_amdgcn_exp2f(stat[0][0][(g << bits) + jrow] - zero);
                rsum[m] += f * stat[1][0][(g << bits) + jrow];
#pragma unroll
                for (int i = 0; i < PER; ++i) res[m][i] += f * od[((g << bits) + jrow) * D + col + i];
            }
        }
        if (threadIdx.x == 0) __hip_atomic_store(a.locks + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        if (16 * m + row >= t.rows) continue;
        const int r = t.first + 16 * m + row, tok = r / a.group, g = r - tok * a.group;
        const bool nothing = rsum[m] == 0.0f;  // no key, or none with a score above -inf: zero (the largest adds 1)
        const float inv = 1.0f / rsum[m];
        uint16_t* dst = a.out + (static_cast<int64_t>(t.start + tok) * a.heads + head * a.group + g) * D + col;
        T y[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) y[i] = static_cast<T>(nothing ? 0.0f : res[m][i] * inv);
        if constexpr (PER == 8) {
            *reinterpret_cast<u4*>(dst) = *reinterpret_cast<const u4*>(y);
        } else {
            *reinterpret_cast<u2*>(dst) = *reinterpret_cast<const u2*>(y);
        }
    }
}

template <typename T>
__device__ __forceinline__ f16v mma32(const u4& a, const u4& b, const f16v& c) {
    if constexpr (__is_same(T, h1))
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(bitcast<h8>(a), bitcast<h8>(b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(bitcast<bf8>(a), bitcast<bf8>(b), c, 0, 0, 0);
}

// Chunk kernel: a tile of 128 rows, 32 for each of four wavefronts; K and V in tiles of 64 keys through LDS by direct loads, two stages
// each: while a tile is computed the next one is on its way. A wavefront fetches 16 keys of each tile, which lie in one page. Two workgroups
// share a CU, and their wavefronts' products and exponentials fill each other's time. A wavefront issues one instruction in four cycles,
// whatever its kind, so the loop over unmasked tiles computes no address: a lane's places change stage by a bit.
// A prompt of 8192 tokens, 32 + 8 heads of 128, 551-594 us (925-998 TFLOP/s; between cards), 5 chunks of up to 700 tokens behind up to 5000 keys, 40 + 8
// heads, 167-177 (760-805). The matrix cores run half of the cycles, at the 1.8 GHz that the card's power leaves (hipBLASLt's product of 8192^3:
// 1530 TFLOP/s); every wavefront reads all of K and V from LDS, 128 KB a tile and workgroup, which takes 62 % of the cycles. Measured and not
// kept: 64 rows a wavefront, half the LDS reads but a SIMD's registers for one wavefront, 638 us against 577; the scores a tile ahead
// 575 against 570; wavefront priorities 557 against 560.
// Lane (c, h) = (lane % 32, lane / 32): scores S^T of row c, keys 8 (i / 4) + 4 h + i % 4 of 32.
template <typename T, int D>
__global__ void __launch_bounds__(256, 2) chunk_kernel(AttnArgs a) {
    constexpr int B = 128, KEYS = 64, C = D / 8, KS = D / 16, DT = D / 32, ROWS = 64 / C, NJ = 16 / ROWS;  // ROWS of a 1 KB load
    constexpr int TILE = KEYS * C;                                                                          // 16-byte chunks of a tile
    constexpr uint32_t kExponent = __is_same(T, h1) ? 0x7C00u : 0x7F80u;
    __shared__ u4 lds[2 * 2 * TILE];  // K [stage][key][chunk], V alike
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c32 = lane & 31, h = lane >> 5;
    // The last rows of a prompt see the most keys: they go first, but behind all requests' first tiles, or the last to start would be one
    // of the longest request's (5 chunks as above: 218 us).
    const int turn_of = blockIdx.x / a.kv_heads, head = blockIdx.x - turn_of * a.kv_heads;
    const int slot = a.starts && turn_of >= a.batch ? static_cast<int>(gridDim.x / a.kv_heads) - 1 - (turn_of - a.batch) : turn_of;
    const int split = blockIdx.y;
    Tile t;
    if (!find_tile<B>(a, slot, lane, t)) return;

    const int r = t.first + 32 * wave + c32, tok = r / a.group;
    const bool mine = 32 * wave + c32 < t.rows, active = 32 * wave < t.rows;  // this lane, this wavefront has a row
    const int limit = mine ? t.before + tok : -1;
    u4 q[KS];
    {
        const uint16_t* src = a.q + (t.start + tok) * a.q_token + (head * a.group + r - tok * a.group) * a.q_head + 8 * h;
#pragma unroll
        for (int e = 0; e < KS; ++e) q[e] = mine ? *reinterpret_cast<const u4*>(src + 16 * e) : u4{0, 0, 0, 0};
    }
    const int tile_high = t.before + (t.first + min(t.rows, B) - 1) / a.group;  // the last key a row of the tile sees
    const int end = static_cast<int>(min(static_cast<int64_t>(tile_high) + 1, static_cast<int64_t>(a.width) << a.shift));
    int begin = 0, stop = max(end, 0), parts = 1;
    if (a.splits > 1 && end > 0) {
        const int share = (max((end + a.splits - 1) / a.splits, kMinKeys) + KEYS - 1) & ~(KEYS - 1);
        parts = (end + share - 1) / share;
        if (split >= parts) return;
        begin = split * share;
        stop = min(end, begin + share);
    } else if (split > 0) {
        return;
    }

    const f16v none = {};
    f16v o[DT], s[2];
    float top = kNone, sum = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = none;

    const_int* table = (const_int*)(a.table + t.request * a.table_stride);
    const uint16_t* kh = a.k + head * a.head_stride;
    const uint16_t* vh = a.v + head * a.head_stride;
    const int final16 = (stop - 1) & ~15;
    const uint32_t token_bytes = static_cast<uint32_t>(a.token_stride) * 2;
    const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void*)lds));
    // where chunk c of key r lies in a tile: places of 16 bytes such that the reads below meet every bank once
    auto k_place = [](int row, int c) { return c ^ (D == 128 ? row & 15 : (row >> 1) & 7); };
    auto v_place = [](int row, int c) { return c ^ (D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2); };
    auto there = [&](int page) { return static_cast<uint32_t>(page) < static_cast<uint32_t>(a.num_pages); };
    auto entry = [&](int key) { return static_cast<int>(table[min(key, final16) >> a.shift]); };
    // offset of this wavefront's 16 keys of the tile at `key`, in values; a page the table does not have is page 0, read and left out
    auto place_of = [&](int key, int page) {
        const int first = min(key + 16 * wave, final16);
        return (there(page) ? page : 0) * a.page_stride + (first & ((1 << a.shift) - 1)) * a.token_stride;
    };
    // What a lane loads of 16 whole keys; K's chunks change places with all of the row's number, V's with the part of it that every
    // load of a lane has.
    uint32_t k_from[NJ];
#pragma unroll
    for (int e = 0; e < NJ; ++e)
        k_from[e] = (e * ROWS + lane / C) * token_bytes + 16 * k_place(e * ROWS + lane / C, lane % C);
    const uint32_t v_from = lane / C * token_bytes + 16 * v_place(lane / C, lane % C);
    uint32_t to = __builtin_amdgcn_readfirstlane(lds_base + wave * (16 * C * 16));  // the place in K's stage, V's 2 tiles on
    // keys key + 16 wave .. + 15 into a stage; past the last key its values again, which nothing sees
    auto fetch_k = [&](int key, int64_t at) {
        const u4 rs = lds_rsrc(kh + at);
        const int last = stop - 1 - min(key + 16 * wave, final16);
        uint32_t from[NJ];
#pragma unroll
        for (int e = 0; e < NJ; ++e) from[e] = k_from[e];
        if (last < 15) {
#pragma unroll
            for (int e = 0; e < NJ; ++e) {
                const int row = e * ROWS + lane / C;
                from[e] = min(row, last) * token_bytes + 16 * k_place(row, lane % C);
            }
        }
        lds_dma16<0>(rs, from[0], 0, to);
        lds_dma16<1024>(rs, from[1], 0, to);
        if constexpr (NJ == 4) {
            lds_dma16<2048>(rs, from[2], 0, to);
            lds_dma16<3072>(rs, from[3], 0, to);
        }
    };
    auto fetch_v = [&](int key, int64_t at) {
        constexpr int S = 2 * TILE * 16;
        const u4 rs = lds_rsrc(vh + at);
        const int last = stop - 1 - min(key + 16 * wave, final16);
        if (last < 15) {
            auto from = [&](int e) {
                return static_cast<uint32_t>(min(e * ROWS + lane / C, last)) * token_bytes + 16 * v_place(lane / C, lane % C);
            };
            lds_dma16<S>(rs, from(0), 0, to);
            lds_dma16<S + 1024>(rs, from(1), 0, to);
            if constexpr (NJ == 4) {
                lds_dma16<S + 2048>(rs, from(2), 0, to);
                lds_dma16<S + 3072>(rs, from(3), 0, to);
            }
            return;
        }
        lds_dma16<S>(rs, v_from, 0, to);
        lds_dma16<S + 1024>(rs, v_from, ROWS * token_bytes, to);
        if constexpr (NJ == 4) {
            lds_dma16<S + 2048>(rs, v_from, 2 * ROWS * token_bytes, to);
            lds_dma16<S + 3072>(rs, v_from, 3 * ROWS * token_bytes, to);
        }
    };

    const int g = (lane >> 4) & 1, i16 = lane & 15;
    // a lane's places in LDS: chunk 2 s + h of key c; 16 keys' 8 (j / 4) + 4 h + j % 4 in place 8 h + j, values 32 d ..
    int k_lane[KS], v_lane[DT];
#pragma unroll
    for (int e = 0; e < KS; ++e) k_lane[e] = (c32 * C + k_place(c32, 2 * e + h)) * 16;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        const int row = 4 * h + (i16 >> 2);
        v_lane[d] = (2 * TILE + row * C + v_place(row, 4 * d + 2 * g + ((i16 & 3) >> 1))) * 16 + (i16 & 1) * 8;
    }
    auto read_k = [&](int e) {  // step e / 2 of keys 32 (e % 2) ..
        return *reinterpret_cast<const u4*>(reinterpret_cast<const char*>(lds) + k_lane[e >> 1] + (e & 1) * (32 * C * 16));
    };
    auto read_v = [&](int e) {  // keys 16 (e / DT) .., values 32 (e % DT) ..
        const int at = v_lane[e % DT] + (e / DT) * (16 * C * 16);
        const u2 lo = read_tr(lds, at), hi = read_tr(lds, at + 8 * C * 16);
        return u4{lo.x, lo.y, hi.x, hi.y};
    };
    auto scores = [&] {
        u4 k[2 * KS];
        constexpr int KA = 6;  // reads ahead of their products
#pragma unroll
        for (int e = 0; e < KA; ++e) k[e] = read_k(e);
#pragma unroll
        for (int e = 0; e < 2 * KS; ++e) {
            if (e + KA < 2 * KS) k[e + KA] = read_k(e + KA);
            s[e & 1] = mma32<T>(k[e], q[e >> 1], e < 2 ? none : s[e & 1]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto best_of = [&] {
        float best = s[0][0];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) best = fmaxf(best, s[n][i]);
        const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(best), __float_as_uint(best), false, false);
        return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])) * a.scale;
    };
    // The sums are scaled to a new maximum only when it is more than 2^8 times the old: probabilities up to 256 instead of 1 are as
    // exact, and most tiles need no pass over the sums.
    auto raise = [&](float best) {
        if (__ballot(best > top + 8.0f)) {
            const float now = fmaxf(top, best), keep = __builtin_amdgcn_exp2f(top - (now == kNone ? 0.0f : now));
            top = now;
            sum *= keep;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= keep;
        }
        return (top == kNone ? 0.0f : top) - kLift<T, 8>;  // none: nothing seen yet
    };
    // four probabilities, of keys 16 u + 8 x + 4 h ..
    auto weights = [&](int u, int x, float zero) {
        f4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u >> 1][8 * (u & 1) + 4 * x + i], a.scale, -zero));
            sum += w[i];
        }
        return w;
    };
    auto pack = [](const f4& x, const f4& y) {
        const float w[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        return from_f32<T>(w);
    };

    // Keys below `clear` are seen by every row and lie in pages that are there.
    int clear = min(t.before + t.first / a.group + 1, stop);
    int ahead = 0;  // the table's entry of this wavefront's keys of the next tile
    if (begin < stop) {
        const int64_t at = place_of(begin, entry(begin + 16 * wave));
        ahead = entry(begin + KEYS + 16 * wave);
        fetch_k(begin, at);
        fetch_v(begin, at);
        int* first_gone = reinterpret_cast<int*>(lds + TILE);  // the second stage is not in use yet
        if (threadIdx.x == 0) *first_gone = 0x7FFFFFFF;
        __syncthreads();
        const int e1 = (stop - 1) >> a.shift;
        int gone = 0x7FFFFFFF;
#pragma unroll 4
        for (int e = (begin >> a.shift) + static_cast<int>(threadIdx.x); e <= e1; e += 256)
            if (!there(a.table[t.request * a.table_stride + e])) gone = min(gone, e << a.shift);
        if (gone != 0x7FFFFFFF) atomicMin(first_gone, gone);
        __syncthreads();
        clear = min(clear, __builtin_amdgcn_readfirstlane(*first_gone));
    }
    // Start of the tile at `key`: it has arrived, and the next one is sent for, into the place of the one before it.
    auto turn = [&](int key) {
        wait_stage<0>();
        ring_barrier();
        to ^= TILE * 16;
        if (key + KEYS < stop) {
            const int64_t at = place_of(key + KEYS, ahead);
            fetch_k(key + KEYS, at);
            fetch_v(key + KEYS, at);
            ahead = entry(key + 2 * KEYS + 16 * wave);
        }
    };
    auto other_stage = [&] {
#pragma unroll
        for (int e = 0; e < KS; ++e) k_lane[e] ^= TILE * 16;
#pragma unroll
        for (int d = 0; d < DT; ++d) v_lane[d] ^= TILE * 16;
    };
    int base = begin;
    for (; base + KEYS <= clear; base += KEYS) {
        turn(base);  // a wavefront without rows goes along
        scores();
        u4 v[4 * DT];
        constexpr int VA = DT;  // reads ahead of their products
        const float zero = raise(best_of());
#pragma unroll
        for (int e = 0; e < VA; ++e) v[e] = read_v(e);
        f4 x = weights(0, 0, zero), y = weights(0, 1, zero);
        u4 p = pack(x, y);
        __builtin_amdgcn_sched_barrier(0);
        // a step: the products of 16 keys beside the probabilities of the next 16
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const int e = u * DT + d;
                if (e + VA < 4 * DT) v[e + VA] = read_v(e + VA);
                o[d] = mma32<T>(v[e], p, o[d]);
                if (u < 3 && d == 0) x = weights(u + 1, 0, zero);
                if (u < 3 && d == DT / 2) y = weights(u + 1, 1, zero);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (u < 3) p = pack(x, y);
        }
        other_stage();
    }
    // From the first tile on that some row does not see whole, or that lies in a page that is none, all are masked.
    for (; base < stop; base += KEYS) {
        turn(base);
        if (!active) continue;
        scores();
        const u4* vt = lds + (2 + ((base - begin) / KEYS & 1)) * TILE;
        const int off = (there(entry(base)) ? 0 : 1) | (there(entry(base + 16)) ? 0 : 2) | (there(entry(base + 32)) ? 0 : 4) |
                        (there(entry(base + 48)) ? 0 : 8);
        bool odd = false;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = 32 * n + 8 * (i >> 2) + 4 * h + (i & 3);
                if (base + key > min(limit, stop - 1) || (off >> (key >> 4) & 1)) s[n][i] = kNone;
            }
        // A probability of zero does not take an infinity or NaN away: where some row does not see a key, such values are left out
        // of the product and added to the rows that see them.
#pragma unroll 2
        for (int e = 0; e < TILE / 64; ++e) {
            const u4 w = vt[64 * e + lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) odd |= odd16(w[i], kExponent);
        }
        odd = __ballot(odd) != 0;
        const float zero = raise(best_of());
        if (odd) {
#pragma unroll 1
            for (int key = 0; key < KEYS; ++key) {
                if (base + key > min(limit, stop - 1) || (off >> (key >> 4) & 1)) continue;
#pragma unroll
                for (int i = 0; i < 4 * DT; ++i) {  // four values from 8 i + 4 h on
                    const u2 four = *reinterpret_cast<const u2*>(reinterpret_cast<const char*>(vt) +
                                                                 (key * C + v_place(key, i)) * 16 + h * 8);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint16_t bits = static_cast<uint16_t>(four[e >> 1] >> (16 * (e & 1)));
                        if ((bits & kExponent) == kExponent) o[i >> 2][4 * (i & 3) + e] += static_cast<float>(bitcast<T>(bits));
                    }
                    __builtin_amdgcn_sched_barrier(0);  // one at a time: the rare path is not to take registers
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const f4 x = weights(u, 0, zero), y = weights(u, 1, zero);
            const u4 p = pack(x, y);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                u4 w = read_v(u * DT + d);
                if (odd) w = read_odd_free(w, kExponent);
                o[d] = mma32<T>(w, p, o[d]);
            }
        }
        other_stage();
    }

    {
        const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
        sum = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    }
    if (parts > 1) {
        // [unit][split][row][D + 4]: the sums, then maximum and sum
        const int unit = slot * a.kv_heads + head;
        constexpr int kRowFloats = D + kTileFloats;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(a.ws, 0, 0x7FFFFFFF, kBufferFlags);
        const int64_t first_row = static_cast<int64_t>(unit) * a.splits * a.part_rows + 32 * wave + c32;
        if (mine) {
            const int to = static_cast<int>((first_row + static_cast<int64_t>(split) * a.part_rows) * kRowFloats * 4);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    __builtin_amdgcn_raw_buffer_store_b128(bitcast<u4>(f4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]}), rs,
                                                           to + (32 * d + 2 * i + 4 * h) * 4, 0, kCoherentAux);
            if (h == 0)
                __builtin_amdgcn_raw_buffer_store_b64(u2{__float_as_uint(top), __float_as_uint(sum)}, rs, to + D * 4, 0, kCoherentAux);
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        int* flag = reinterpret_cast<int*>(lds);
        if (threadIdx.x == 0)
            *flag = __hip_atomic_fetch_add(a.locks + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
        __syncthreads();
        if (!*flag) return;
        if (mine) {
            top = kNone, sum = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] = none;
            for (int part = 0; part < parts; ++part) {
                const int from = static_cast<int>((first_row + static_cast<int64_t>(part) * a.part_rows) * kRowFloats * 4);
                const u2 ms = bitcast<u2>(__builtin_amdgcn_raw_buffer_load_b64(rs, from + D * 4, 0, kCoherentAux));
                f4 x[4 * DT];
#pragma unroll
                for (int i = 0; i < 4 * DT; ++i)
                    x[i] = bitcast<f4>(__builtin_amdgcn_raw_buffer_load_b128(rs, from + (8 * i + 4 * h) * 4, 0, kCoherentAux));
                const float other = __uint_as_float(ms.x), now = fmaxf(top, other), zero = now == kNone ? 0.0f : now;
                const float keep = __builtin_amdgcn_exp2f(top - zero), f = __builtin_amdgcn_exp2f(other - zero);
                top = now;
                sum = sum * keep + f * __uint_as_float(ms.y);
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * keep + f * x[4 * d + (i >> 2)][i & 3];
            }
        }
        if (threadIdx.x == 0) __hip_atomic_store(a.locks + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // a lane has 4 of every 8 values: the halves of the wavefront exchange blocks, so that each stores 16 bytes
    const bool nothing = sum == 0.0f;  // no key, or none with a score above -inf: zero
    const float inv = 1.0f / sum;
    uint16_t* dst = a.out + (static_cast<int64_t>(t.start + tok) * a.heads + head * a.group + r - tok * a.group) * D + 8 * h;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = nothing ? 0.0f : o[d][8 * b + i] * inv;
            const u4 y = from_f32<T>(x);
            const auto e = __builtin_amdgcn_permlane32_swap(y[0], y[2], false, false);
            const auto f = __builtin_amdgcn_permlane32_swap(y[1], y[3], false, false);
            if (mine) *reinterpret_cast<u4*>(dst + 32 * d + 16 * b) = u4{e[0], f[0], e[1], f[1]};
        }
}

constexpr int64_t kWorkspaceFloats = TW4_AUTO_SPLIT_FLOATS;

int64_t tile_slots(int tokens, int batch, int group, int rows, bool single) {
    if (single) return static_cast<int64_t>(batch) * ((group + rows - 1) / rows);
    return static_cast<int64_t>(tokens) * group / rows + batch;
}

template <typename T, int D>
int attn_launch(const AttnArgs& a, int rows, unsigned units, hipStream_t st) {
    const dim3 grid(units, a.splits);
    if (rows == 16)
        rows_kernel<T, D, 1><<<grid, 256, 0, st>>>(a);
    else if (rows == 32)
        rows_kernel<T, D, 2><<<grid, 256, 0, st>>>(a);
    else
        chunk_kernel<T, D><<<grid, 256, 0, st>>>(a);
    TW4_LAUNCH_CHECK("paged_attention: launch");
    return TW4_OK;
}

}  // namespace tw4

using namespace tw4;

// Microseconds of a call with tiles of kRows[i] rows and `splits` splits, as fitted to 300 calls of all sizes with each tile and 1 to 128
// splits (batches 1 to 200, 1 to 2000 new tokens, 0 to 100000 keys, heads of 64 and 128). A workgroup takes `start`, its keys' latency,
// and, with splits, the store of its part and the last one's reading of all; two workgroups share a CU, so beyond 2 cus of them the keys'
// throughput counts. What the rule picks took 1.013 times the fastest tile and split on average, 1.18 at most (4 chunks of 65 tokens: 11.8
// us with 16 rows, 10.0 with 128); on 75 calls it was not fitted to 1.017, 1.18 at most (5 chunks of up to 188 tokens of 7 heads behind up
// to 1908 keys: 32.9 us with 3 splits, 27.8 with one); profiles/paged_attention_rule_sweep.jsonl has them all. Without it: tiles by rows
// alone (16, 32, or 128 past 32 rows) and splits for two workgroups per CU took 1.3 on average, 5.8 at most (7 new tokens of 24 heads over
// 7638 keys: 119 us with tiles of 128 rows and 60 splits, 20.4 with 16 rows and 12).
constexpr int kRows[3] = {16, 32, 128};
double cost_us(int i, int64_t units, int splits, int group, int head_dim, int max_keys, int single, int cus) {
    constexpr double kStart[3] = {6.097, 7.606, 7.066}, kLatency[3] = {0.0089, 0.0092, 0.0165}, kRate[3] = {0.0185, 0.0165, 0.0443},
                     kJoin[3] = {0.36, 0.288, 0.373};
    const int quantum = kRows[i] == 128 ? 64 : 128;
    const int64_t share =
        (std::max<int64_t>((static_cast<int64_t>(max_keys) + splits - 1) / splits, kMinKeys) + quantum - 1) / quantum * quantum;
    const int64_t parts = std::max<int64_t>((max_keys + share - 1) / share, 1);
    const double keys = static_cast<double>(std::min<int64_t>(share, max_keys)) * (head_dim == 64 ? 0.467 : 1.0);
    const double load = static_cast<double>(units) * parts / (2.0 * cus);
    const double rounds = load > 1.0 ? load + 0.074 * (std::ceil(load) - load) : load;
    double us = kStart[i] + std::pow(std::pow(kLatency[i] * keys, 1.5) + std::pow(kRate[i] * keys * rounds, 1.5), 1 / 1.5) +
                1.945 * std::max(load - 1.0, 0.0);
    if (parts > 1) us += 2.246 + kJoin[i] * parts * (single ? std::min(kRows[i], group) : kRows[i]) / 16.0 + 2.004 * load;
    return us;
}

// out: rows of a tile, splits, workspace floats, counters
extern "C" int tw4_paged_attention_plan(int tokens, int batch, int heads, int kv_heads, int head_dim, int max_query, int max_keys,
                                        int single, int cus, int* out) {
    TW4_REQUIRE(out && tokens >= 0 && batch >= 0 && kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0 && head_dim >= 1 && cus >= 1 &&
                    max_keys >= 0 && max_query >= 0,
                TW4_EINVAL, "paged_attention_plan: bad sizes");
    const int group = heads / kv_heads;
    double best = 0.0;
    int rows = 0, splits = 1;
    int64_t units = 0, part = 0;
    for (int i = 0; i < 3; ++i) {
        // A tile no larger than a request's rows need (16 rows against 32, the fastest split of each: 3 new tokens of 32 + 8 heads over
        // 2000 keys 12.8 us against 14.6, 60 of those 73.1 against 74.2, 33 requests of 16 rows 14.7 against 17.0; 3 of 16 rows over
        // 8000 keys 28.2 against 26.4)
        if (i > 0 && kRows[i - 1] >= static_cast<int64_t>(max_query) * group) break;
        const int64_t u = tile_slots(tokens, batch, group, kRows[i], single) * kv_heads;
        const int64_t floats = static_cast<int64_t>(single ? std::min(kRows[i], group) : kRows[i]) * (head_dim + kTileFloats);
        // those that can have rows
        const int64_t per = (static_cast<int64_t>(max_query) * group + kRows[i] - 1) / kRows[i], work = std::min(u, batch * per * kv_heads);
        // and what fills the CUs once or twice
        const int once = static_cast<int>(work ? 2 * cus / work : 0), twice = static_cast<int>(work ? 4 * cus / work : 0);
        for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 64, once, twice}) {
            if (s < 1 || (s > 1 && (static_cast<int64_t>(s - 1) * kMinKeys >= max_keys || u * s * floats > kWorkspaceFloats ||
                                    u > TW4_AUTO_SPLIT_COUNTERS)))
                continue;
            const double us = cost_us(i, work, s, group, head_dim, max_keys, single, cus);
            if (rows == 0 || us < best) best = us, rows = kRows[i], splits = s, units = u, part = floats;
        }
    }
    out[0] = rows;
    out[1] = static_cast<int>(splits);
    out[2] = splits > 1 ? static_cast<int>(units * splits * part) : 0;
    out[3] = splits > 1 ? static_cast<int>(units) : 0;
    return TW4_OK;
}

extern "C" int tw4_paged_attention(const uint16_t* q, int64_t q_token, int64_t q_head, const uint16_t* k, const uint16_t* v,
                                   int64_t page_stride, int64_t head_stride, int64_t token_stride, int num_pages, int page_size,
                                   const int32_t* table, int64_t table_stride, int width, const int32_t* lens,
                                   const int32_t* starts, uint16_t* out, float* ws, int64_t ws_floats, int32_t* locks,
                                   int64_t n_locks, int tokens, int batch, int heads, int kv_heads, int head_dim, float scale,
                                   int rows, int splits, int bf16, void* stream) {
    TW4_REQUIRE(tokens >= 0 && batch >= 0 && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, TW4_EINVAL,
                "paged_attention: heads a multiple of kv_heads (%d, %d)", heads, kv_heads);
    TW4_REQUIRE(head_dim == 64 || head_dim == 128, TW4_EINVAL, "paged_attention: head_dim 64 or 128 (%d)", head_dim);
    const int shift = page_shift(page_size);
    TW4_REQUIRE(shift >= 0, TW4_EINVAL, "paged_attention: page_size 16, 32, 64, 128 or 256 (%d)", page_size);
    TW4_REQUIRE(scale > 0.0f && scale < 1e30f, TW4_EINVAL, "paged_attention: a positive scale (%g)", scale);
    TW4_REQUIRE(rows == 16 || rows == 32 || rows == 128, TW4_ECONFIG,
                "paged_attention: tiles of 16, 32 or 128 rows (%d)", rows);
    TW4_REQUIRE(width >= 0 && num_pages >= 0 && static_cast<int64_t>(num_pages) * page_size < 1LL << 31 &&
                    static_cast<int64_t>(width) * page_size <= 1LL << 30,
                TW4_EINVAL, "paged_attention: fewer than 2^31 slots, at most 2^30 keys of a request (%d pages of %d, %d per request)",
                num_pages, page_size, width);
    TW4_REQUIRE(static_cast<int64_t>(tokens) * heads <= 1LL << 30, TW4_EINVAL, "paged_attention: too many rows (%d tokens)", tokens);
    TW4_REQUIRE(starts || tokens == batch, TW4_EINVAL, "paged_attention: without query starts one token per request (%d, %d)",
                tokens, batch);
    if (tokens == 0 || batch == 0) return TW4_OK;
    TW4_REQUIRE(q && out && lens && (!width || table) && (!num_pages || (k && v)), TW4_EINVAL, "paged_attention: null pointer");
    TW4_REQUIRE(num_pages > 0 || width == 0, TW4_EINVAL, "paged_attention: a cache without pages");
    for (const void* p : {static_cast<const void*>(q), static_cast<const void*>(k), static_cast<const void*>(v),
                          static_cast<const void*>(out)})
        TW4_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, TW4_EINVAL, "paged_attention: operands must be 16-byte aligned");
    TW4_REQUIRE(token_stride >= 0 && token_stride < 1LL << 26, TW4_EINVAL, "paged_attention: token stride (%lld)",
                static_cast<long long>(token_stride));
    TW4_REQUIRE(q_token % 8 == 0 && q_head % 8 == 0 && page_stride % 8 == 0 && head_stride % 8 == 0 && token_stride % 8 == 0,
                TW4_EINVAL, "paged_attention: strides must be multiples of 8");
    const int group = heads / kv_heads;
    const int64_t slots = tile_slots(tokens, batch, group, rows, !starts), units = slots * kv_heads;
    // a launch has fewer than 2^32 threads along an axis
    TW4_REQUIRE(units < 1LL << 24 && splits >= 1 && splits <= 65535, TW4_EINVAL, "paged_attention: grid (%lld tiles, %d splits)",
                static_cast<long long>(units), splits);
    const int part_rows = starts ? rows : std::min(rows, group);
    if (splits > 1) {
        const int64_t need = units * splits * part_rows * (head_dim + kTileFloats);
        TW4_REQUIRE(ws && locks && need <= ws_floats && need < kMaxPartialFloats && units <= n_locks, TW4_ESPACE,
                    "paged_attention: %d splits need %lld floats and %lld counters (got %lld, %lld)", splits,
                    static_cast<long long>(need), static_cast<long long>(units), static_cast<long long>(ws_floats),
                    static_cast<long long>(n_locks));
    }
    const AttnArgs a{q, k, v, table, lens, starts, out, ws, locks, q_token, q_head, page_stride, head_stride, token_stride,
                     table_stride, scale * 1.44269504088896340736f, tokens, batch, heads, kv_heads, group, num_pages, width, shift,
                     splits, part_rows};
    auto st = static_cast<hipStream_t>(stream);
    if (bf16) return head_dim == 64 ? attn_launch<bf1, 64>(a, rows, static_cast<unsigned>(units), st) : attn_launch<bf1, 128>(a, rows, static_cast<unsigned>(units), st);
    return head_dim == 64 ? attn_launch<h1, 64>(a, rows, static_cast<unsigned>(units), st) : attn_launch<h1, 128>(a, rows, static_cast<unsigned>(units), st);
}

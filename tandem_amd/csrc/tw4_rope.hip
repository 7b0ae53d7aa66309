// RMS norm of each query and key head, the rotation by position, and the writes of keys and values into the paged cache,
// in one pass over a projection's output qkv = [q | k | v], rows of (heads + 2 kv_heads) D values of fp16 or bf16:
//
//   y = x rsqrt(mean(x^2) + eps) w             for a query or key head x of D values (w absent: y = x)
//   out[i]         = y[i] cos[p][i] - y[i + D/2] sin[p][i]
//   out[i + D/2]   = y[i + D/2] cos[p][i] + y[i] sin[p][i],     i < D/2, p the token's position
//
// in fp32 with one rounding at the end. A head is D / 8 lanes of 16 bytes, so a wavefront holds 4 heads of 128 (8 of 64);
// the partner of a value lies D / 16 lanes away and comes as the raw 16 bytes (four exchanges instead of eight of fp32).
// Values are copied as they are.
//
// It moves 2 (heads + 2 kv_heads) D values a token and is bound by memory, or by its launch: 32 + 8 heads of 128 into the cache, one
// token 2.6 us, 1024 tokens 7.7, 8192 tokens 38.9 (206 MB read and written at 5.3 TB/s; a copy of 1 GiB runs at 5.2). A wavefront takes
// U groups of heads of one token, all loaded before any arithmetic; each one's cosines and sines are 32 bytes a lane from the caches.
#include "tw4_attn.h"

namespace tw4 {

struct RopeArgs {
    const uint16_t* qkv;
    int64_t row_stride;
    const int32_t* positions;
    const float* table;
    const uint16_t* q_weight;
    const uint16_t* k_weight;
    uint16_t* q_out;
    uint16_t* k_out;
    uint16_t* v_out;
    const int32_t* slots;
    int64_t page_stride, head_stride, token_stride;
    float eps;
    int tokens, heads, kv_heads, table_rows, num_pages, page_shift, groups;
};

// Sum over the C lanes of a head (aligned), the same bits in each of them.
template <int C>
__device__ __forceinline__ float head_sum(float v) {
    if constexpr (C == 16) return row16_sum(v);
    v += lane_xor1(v);
    v += lane_xor2(v);
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, false));  // half mirror
}

template <typename T, int D, int U>
__global__ void __launch_bounds__(256) rope_kernel(RopeArgs a) {
    constexpr int C = D / 8, HPG = 64 / C;  // chunks of a head, heads of a group
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t parts = (a.groups + U - 1) / U, unit = blockIdx.x * 4 + wave;  // units below 2^31
    const int t = unit / parts, part = unit - t * parts;
    if (t >= a.tokens) return;
    const int c = lane % C, sub = lane / C;
    const int all = a.heads + 2 * a.kv_heads, rotated = a.heads + a.kv_heads;
    const uint16_t* row = a.qkv + t * a.row_stride;

    u4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int head = (part * U + u) * HPG + sub;
        raw[u] = head < all ? *reinterpret_cast<const u4*>(row + static_cast<int64_t>(head) * D + 8 * c) : u4{0, 0, 0, 0};
    }
    const int p = a.positions[t];
    const int slot = a.slots ? a.slots[t] : 0;
    const bool known = static_cast<uint32_t>(p) < static_cast<uint32_t>(a.table_rows);
    const float* turn = a.table + static_cast<int64_t>(known ? p : 0) * D + 8 * (c % (C / 2));
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
        *reinterpret_cast<f4*>(cs + i) = *reinterpret_cast<const f4*>(turn + i);
        *reinterpret_cast<f4*>(sn + i) = *reinterpret_cast<const f4*>(turn + D / 2 + i);
    }
    if (!known) {  // a position the table does not have must not pass for another one
#pragma unroll
        for (int i = 0; i < 8; ++i) cs[i] = __builtin_nanf("");
    }
    const bool high = c >= C / 2;
    const bool kept = a.slots == nullptr || (slot >= 0 && (slot >> a.page_shift) < a.num_pages);
    const int64_t at = (slot >> a.page_shift) * a.page_stride + (slot & ((1 << a.page_shift) - 1)) * a.token_stride;

#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int head = (part * U + u) * HPG + sub;
        u4 other;
#pragma unroll
        for (int i = 0; i < 4; ++i) other[i] = __shfl_xor(static_cast<int>(raw[u][i]), C / 2);
        float x[8], y[8];
        to_f32<T>(raw[u], x);
        to_f32<T>(other, y);
        const uint16_t* w = head < a.heads ? a.q_weight : a.k_weight;
        const float rstd = rsqrtf(head_sum<C>(sumsq8(x)) / static_cast<float>(D) + a.eps);
        if (head < rotated && w) {
            float wx[8], wy[8];
            to_f32<T>(*reinterpret_cast<const u4*>(w + 8 * c), wx);
            to_f32<T>(*reinterpret_cast<const u4*>(w + 8 * (c ^ (C / 2))), wy);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = x[i] * rstd * wx[i];
                y[i] = y[i] * rstd * wy[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = high ? x[i] * cs[i] + y[i] * sn[i] : x[i] * cs[i] - y[i] * sn[i];
        const u4 out = from_f32<T>(x);
        if (head < a.heads) {
            *reinterpret_cast<u4*>(a.q_out + (static_cast<int64_t>(t) * a.heads + head) * D + 8 * c) = out;
        } else if (head < all && kept) {
            const int kv = head < rotated ? head - a.heads : head - rotated;
            if (!a.slots) {
                if (head < rotated)
                    *reinterpret_cast<u4*>(a.k_out + (static_cast<int64_t>(t) * a.kv_heads + kv) * D + 8 * c) = out;
            } else {
                uint16_t* dst = (head < rotated ? a.k_out : a.v_out) + at + kv * a.head_stride + 8 * c;
                *reinterpret_cast<u4*>(dst) = head < rotated ? out : raw[u];
            }
        }
    }
}

constexpr int64_t kManyGroups = 1 << 16;

template <typename T, int D>
int rope_launch(RopeArgs& a, hipStream_t st) {
    constexpr int HPG = 512 / D;
    // without a cache the values are not touched
    const int all = a.heads + (a.slots ? 2 : 1) * a.kv_heads;
    a.groups = (all + HPG - 1) / HPG;
    auto blocks = [&](int u) {
        return (static_cast<int64_t>(a.tokens) * ((a.groups + u - 1) / u) + 3) / 4;
    };
    // a launch has fewer than 2^32 threads
    TW4_REQUIRE(blocks(D == 128 ? 4 : 1) < (1LL << 24), TW4_EINVAL, "norm_rope: too many values (%d tokens)", a.tokens);
    // One group a wavefront has the most loads under way (64 tokens 2.8 us against 4.2 with four). Where the data pass what the caches
    // hold, four that share the angles' loads are faster: heads of 128, 32 + 8 of them, 8192 tokens 43.3 us -> 38.9, 6000 33.1 -> 30.1, 4000
    // level at 22.8, 2000 13.2 -> 13.8; heads of 64 17.4 -> 19.0 at 6000.
    if constexpr (D == 128) {
        if (static_cast<int64_t>(a.tokens) * a.groups >= kManyGroups) {
            rope_kernel<T, D, 4><<<static_cast<unsigned>(blocks(4)), 256, 0, st>>>(a);
            TW4_LAUNCH_CHECK("norm_rope: launch");
            return TW4_OK;
        }
    }
    rope_kernel<T, D, 1><<<static_cast<unsigned>(blocks(1)), 256, 0, st>>>(a);
    TW4_LAUNCH_CHECK("norm_rope: launch");
    return TW4_OK;
}

}  // namespace tw4

using namespace tw4;

extern "C" int tw4_norm_rope(const uint16_t* qkv, int64_t row_stride, const int32_t* positions, const float* table,
                             int table_rows, const uint16_t* q_weight, const uint16_t* k_weight, float eps,
                             uint16_t* q_out, uint16_t* k_out, uint16_t* v_out, const int32_t* slots, int num_pages,
                             int page_size, int64_t page_stride, int64_t head_stride, int64_t token_stride, int tokens,
                             int heads, int kv_heads, int head_dim, int bf16, void* stream) {
    TW4_REQUIRE(qkv && positions && table && q_out && k_out && (!slots || v_out), TW4_EINVAL, "norm_rope: null pointer");
    for (const void* p : {static_cast<const void*>(qkv), static_cast<const void*>(table), static_cast<const void*>(q_weight),
                          static_cast<const void*>(k_weight), static_cast<const void*>(q_out),
                          static_cast<const void*>(k_out), static_cast<const void*>(v_out)})
        TW4_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, TW4_EINVAL, "norm_rope: operands must be 16-byte aligned");
    TW4_REQUIRE(tokens >= 0 && heads >= 1 && kv_heads >= 1 && heads <= 1 << 16 && kv_heads <= heads, TW4_EINVAL,
                "norm_rope: tokens >= 0, 1 <= kv_heads <= heads <= 65536 (%d, %d, %d)", tokens, heads, kv_heads);
    TW4_REQUIRE(head_dim == 64 || head_dim == 128, TW4_EINVAL, "norm_rope: head_dim 64 or 128 (%d)", head_dim);
    TW4_REQUIRE(table_rows >= 1, TW4_EINVAL, "norm_rope: an empty rotation table");
    TW4_REQUIRE(row_stride % 8 == 0 && row_stride >= static_cast<int64_t>(heads + 2 * kv_heads) * head_dim, TW4_EINVAL,
                "norm_rope: rows of (heads + 2 kv_heads) head_dim values, a stride that is a multiple of 8 (%lld)",
                static_cast<long long>(row_stride));
    int shift = 0;
    if (slots) {
        shift = page_shift(page_size);
        TW4_REQUIRE(shift >= 0, TW4_EINVAL, "norm_rope: page_size 16, 32, 64, 128 or 256 (%d)", page_size);
        TW4_REQUIRE(num_pages >= 0 && static_cast<int64_t>(num_pages) * page_size < (1LL << 31), TW4_EINVAL,
                    "norm_rope: fewer than 2^31 slots (%d pages)", num_pages);
        TW4_REQUIRE(page_stride % 8 == 0 && head_stride % 8 == 0 && token_stride % 8 == 0, TW4_EINVAL,
                    "norm_rope: cache strides must be multiples of 8");
    }
    if (tokens == 0) return TW4_OK;
    RopeArgs a{qkv, row_stride, positions, table, q_weight, k_weight, q_out, k_out, v_out, slots, page_stride, head_stride,
               token_stride, eps, tokens, heads, kv_heads, table_rows, num_pages, shift, 0};
    auto st = static_cast<hipStream_t>(stream);
    if (bf16) return head_dim == 64 ? rope_launch<bf1, 64>(a, st) : rope_launch<bf1, 128>(a, st);
    return head_dim == 64 ? rope_launch<h1, 64>(a, st) : rope_launch<h1, 128>(a, st);
}

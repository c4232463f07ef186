// fe_attention_cache.cuh — what the kernels of the paged 8-bit cache and its attention share:
// arguments, the reading of a sequence's offsets, and the launcher of the tile kernel.
#pragma once

#include "fe_e4m3.cuh"
#include "fe_internal.h"

namespace fe {

struct CacheArgs {
    const __nv_bfloat16 *qkv;
    const int32_t *cu, *past, *table;
    const uint8_t *k, *v;
    const float *ks, *vs;
    __nv_bfloat16 *out;
    float *part_o;  // [T * q_heads][splits][hd], splits > 1
    float *part_mn; // [T * q_heads][splits][4]: reference of O, of the sum, the sum, -
    int64_t total, row;
    int batch, max_len, width, pages, page_log2, q_heads, kv_heads, group, causal;
    int splits;
    float scale_log2;
};

constexpr int kMaxCacheTokens = 1 << 30;  // of a sequence: token indexes fit 32 bits with room

// One sequence of the batch: false when it is empty, and (with a report) when its offsets do not describe it.
struct CacheSeq {
    int t0, len, past, kv;  // first row, new tokens, tokens before them, tokens in the cache
};

__device__ __forceinline__ bool load_seq(const CacheArgs &a, int b, CacheSeq &s, int *status)
{
    s.t0 = a.cu[b];
    const int t1 = a.cu[b + 1];
    s.past = a.past[b];
    if (t1 == s.t0) return false;
    const int64_t len = static_cast<int64_t>(t1) - s.t0, kv = s.past + len;
    const bool ok = s.t0 >= 0 && len > 0 && t1 <= a.total && len <= a.max_len && s.past >= 0 && kv <= kMaxCacheTokens &&
                    kv <= (static_cast<int64_t>(a.width) << a.page_log2);
    s.len = static_cast<int>(len);
    s.kv = static_cast<int>(kv);
    if (!ok && threadIdx.x == 0) report(status, DEV_BAD_INPUT);
    return ok;
}

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A part of a row's softmax: its sum of weights times codes is 2^m O, its sum of weights 2^n l.  Each has a
// reference of its own, since a page's value scale (any size, 0 among them) is in the first sum's weights only.
// Without a reference (-inf) O or l is zero, or a NaN that stays.
struct RowPart {
    float m, n, l;
};

// What a part's O or l counts for beside the references' maximum
__device__ __forceinline__ float part_weight(float reference, float top)
{
    return reference == -INFINITY ? 1.f : exp2_fast(reference - top);
}

// 1 / l (0 for a row that sees nothing) and 2^(m - n) in two factors, each of them in range
struct RowFactor {
    float inv, a, b;
    __device__ __forceinline__ float operator()(float o) const { return o * inv * a * b; }
};

__device__ __forceinline__ RowFactor row_factor(float m, float n, float l)
{
    const float x = m == -INFINITY ? 0.f : m - n, half = truncf(0.5f * x);
    return {l == 0.f ? 0.f : 1.0f / l, exp2_fast(half), exp2_fast(x - half)};
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Rows of a sequence's key-value head (tokens x query heads of its group) per unit of the tile kernel.
int attention_cache_tile_rows(int head_dim);
cudaError_t launch_attention_cache_tiles(const CacheArgs &a, int head_dim, int *status, cudaStream_t s, fe_status *st);

}  // namespace fe

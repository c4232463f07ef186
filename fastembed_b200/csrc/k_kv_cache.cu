// k_kv_cache.cu — the write into the paged 8-bit key-value cache.
//
// The cache holds pages of `page` tokens: codes e4m3 [pages, kv_heads, page, hd] for K and for
// V, and one fp32 scale per (page, kv head) for each.  A value is code * scale.  Scales are
// powers of two (or 0 for a page whose tokens are all zero): the smallest 2^e with
// amax <= 448 * 2^e over every token written to the page so far, e >= -80.  A power of two
// loses no precision to a code's 3 mantissa bits, and when a later token raises the scale the
// older codes of that page are re-encoded by an exact shift of their exponent (only codes that
// fall below the subnormal range round), so a page filled token by token holds what it would
// hold filled at once, up to that.
//
// A token whose key or value of a head has a non-finite element gets the NaN code in all of that
// head's key, and zeros for such elements of its value: every query that sees the token gets
// NaN, and none that does not (attention weights of zero never meet a NaN value).
//
// One CTA per (page that the new tokens reach, kv head) handles K and V together: new rows are
// read once into registers (16 bytes a thread, hd / 8 threads a token), the block maximum
// decides the scale, codes go out 8 bytes a thread.  Bound by HBM for prompts (2 bytes in, 1
// out per element) and by latency (table -> rows -> codes) for single tokens.
#include "fe_attention_cache.cuh"

namespace fe {
namespace {

// The largest |v| of 8 bf16 as bf16 bits: they order like the values, infinities and NaN (0x7f80
// and above) last.
constexpr uint32_t kBf16Inf = 0x7f80u;
__device__ __forceinline__ uint32_t amax8(const uint4 &u)
{
    const uint32_t m = __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu), __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16);
}

// zeros in place of non-finite elements
__device__ __forceinline__ uint4 finite_only(uint4 u)
{
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & kBf16Inf) == kBf16Inf) w[i] &= 0xffff0000u;
        if ((w[i] & (kBf16Inf << 16)) == kBf16Inf << 16) w[i] &= 0x0000ffffu;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The smallest power of two 2^e with amax <= 448 * 2^e, e >= kMinScaleExp; 0 for amax = 0.
// amax comes as bf16 bits (1.f * 2^E, or subnormal, far below the smallest scale); 448 = 1.75 * 2^8.
constexpr int kMinScaleExp = -80;
__device__ __forceinline__ float block_scale(uint32_t amax)
{
    if (amax == 0) return 0.f;
    const int e = static_cast<int>(amax >> 7) - 127 - 8 + ((amax & 0x7fu) > 0x60u ? 1 : 0);  // mantissa above 1.75
    return __uint_as_float(static_cast<uint32_t>(max(e, kMinScaleExp) + 127) << 23);
}

__device__ __forceinline__ uint32_t encode4(uint32_t x, uint32_t y, float inv)
{
    float2 a = unpack_bf16x2(x), b = unpack_bf16x2(y);
    mul_f32x2(a.x, a.y, inv, inv);
    mul_f32x2(b.x, b.y, inv, inv);
    return pack_e4m3x4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ uint2 encode8(const uint4 &u, float inv)
{
    return make_uint2(encode4(u.x, u.y, inv), encode4(u.z, u.w, inv));
}

__device__ __forceinline__ uint32_t rescale4(uint32_t codes, float ratio)
{
    const float2 a = e4m3x2_to_f32x2(codes & 0xffffu), b = e4m3x2_to_f32x2(codes >> 16);
    return pack_e4m3x4(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
}

// The block's largest k and v (every thread gets both).
template <int WARPS>
__device__ __forceinline__ void block_max(uint32_t &k, uint32_t &v, uint32_t (&red)[2][WARPS])
{
    k = __reduce_max_sync(0xffffffffu, k);
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) {
        red[0][threadIdx.x >> 5] = k;
        red[1][threadIdx.x >> 5] = v;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
        k = max(k, red[0][i]);
        v = max(v, red[1][i]);
    }
}

struct AppendArgs {
    const __nv_bfloat16 *qkv;
    const int32_t *cu, *past, *table;
    uint8_t *k, *v;
    float *ks, *vs;
    int64_t total, row;  // tokens and elements per row of qkv
    int batch, max_len, width, pages, page, kv_heads, k_col0, v_col0;
};

// THREADS threads hold CH 16-byte chunks of K and of V each: CH * THREADS * 8 >= page * HD.
template <int HD, int CH, int THREADS>
__global__ void __launch_bounds__(THREADS) kv_append(const AppendArgs a, int reach, int *status)
{
    constexpr int LPT = HD / 8;  // lanes of a token: 8, 16 or 32, aligned within a warp
    __shared__ uint32_t red[2][2][THREADS / 32];
    const int b = blockIdx.x / reach, nth = blockIdx.x % reach, head = blockIdx.y;
    grid_dep_wait();
    grid_dep_launch();
    const int t0 = a.cu[b], t1 = a.cu[b + 1], past = a.past[b];
    if (t1 == t0) return;
    const int64_t len = static_cast<int64_t>(t1) - t0, end = past + len;
    if (t0 < 0 || len < 0 || t1 > a.total || len > a.max_len || past < 0 || end > kMaxCacheTokens ||
        end > static_cast<int64_t>(a.width) * a.page) {  // offsets that do not describe the batch: nothing is touched
        if (threadIdx.x == 0) report(status, DEV_BAD_INPUT);
        return;
    }
    const int64_t ordinal = past / a.page + nth;
    const int64_t base = ordinal * a.page;  // first token of the page
    if (base >= end) return;
    const int lo = past > base ? static_cast<int>(past - base) : 0;              // first new slot
    const int hi = end - base < a.page ? static_cast<int>(end - base) : a.page;  // past the last

    // the rows are on their way before the page is looked up
    uint4 kr[CH], vr[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int chunk = c * THREADS + threadIdx.x, slot = chunk / LPT, col = chunk % LPT * 8;
        kr[c] = vr[c] = make_uint4(0, 0, 0, 0);
        if (slot >= lo && slot < hi) {
            const __nv_bfloat16 *p = a.qkv + (t0 + (base + slot - past)) * a.row + static_cast<int64_t>(head) * HD + col;
            kr[c] = *reinterpret_cast<const uint4 *>(p + a.k_col0);
            vr[c] = *reinterpret_cast<const uint4 *>(p + a.v_col0);
        }
    }
    const int id = a.table[static_cast<int64_t>(b) * a.width + ordinal];
    if (id < 0 || id >= a.pages) {
        if (threadIdx.x == 0) report(status, DEV_BAD_INPUT);
        return;
    }
    const int64_t si = static_cast<int64_t>(id) * a.kv_heads + head;
    const int64_t block = si * a.page * HD;  // codes of this (page, head)
    const float k_old = lo > 0 ? a.ks[si] : 0.f, v_old = lo > 0 ? a.vs[si] : 0.f;

    uint32_t km = 0, vm = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        km = max(km, amax8(kr[c]));
        vm = max(vm, amax8(vr[c]));
    }
    block_max<THREADS / 32>(km, vm, red[0]);  // its barrier: every thread has read the old scales
    uint32_t poisoned = 0;                    // bit c: this thread's token of chunk c holds something non-finite
    if (max(km, vm) >= kBf16Inf) {            // rare: find those tokens, and the maxima without them
        km = vm = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const uint32_t mk = amax8(kr[c]);
            const uint32_t any = __ballot_sync(0xffffffffu, max(mk, amax8(vr[c])) >= kBf16Inf);
            const uint32_t group = LPT == 32 ? 0xffffffffu : ((1u << (LPT & 31)) - 1u) << ((threadIdx.x & 31) / LPT * LPT);
            if (any & group) poisoned |= 1u << c;
            else km = max(km, mk);  // a poisoned token's key is stored as NaN and sets no scale
            vr[c] = finite_only(vr[c]);
            vm = max(vm, amax8(vr[c]));
        }
        block_max<THREADS / 32>(km, vm, red[1]);
    }
    const float k_new = fmaxf(k_old, block_scale(km)), v_new = fmaxf(v_old, block_scale(vm));
    const float k_inv = k_new > 0.f ? 1.0f / k_new : 0.f, v_inv = v_new > 0.f ? 1.0f / v_new : 0.f;
    if (threadIdx.x == 0) {
        a.ks[si] = k_new;
        a.vs[si] = v_new;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int chunk = c * THREADS + threadIdx.x, slot = chunk / LPT;
        if (slot >= lo && slot < hi) {
            *reinterpret_cast<uint2 *>(a.k + block + chunk * 8) =
                (poisoned >> c) & 1u ? make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu) : encode8(kr[c], k_inv);
            *reinterpret_cast<uint2 *>(a.v + block + chunk * 8) = encode8(vr[c], v_inv);
        }
    }
    // older tokens of the page follow a scale that grew
    for (int which = 0; which < 2; ++which) {
        const float was = which ? v_old : k_old, now = which ? v_new : k_new;
        if (lo == 0 || !(now > was)) continue;
        uint8_t *codes = (which ? a.v : a.k) + block;
        const float ratio = was / now;
        for (int chunk = threadIdx.x; chunk < lo * LPT; chunk += THREADS) {
            uint2 *p = reinterpret_cast<uint2 *>(codes + chunk * 8);
            const uint2 u = *p;
            *p = make_uint2(rescale4(u.x, ratio), rescale4(u.y, ratio));
        }
    }
}

template <int HD>
cudaError_t append(const AppendArgs &a, cudaStream_t s)
{
    const int reach = (a.page - 1 + a.max_len - 1) / a.page + 1;  // pages that max_len tokens at any offset can touch
    const dim3 grid(static_cast<unsigned>(a.batch) * reach, a.kv_heads);
    int *status = current_device_status_word();
    const int chunks = a.page * HD / 8;  // 128 (page 16, head_dim 64) to 4096 (128, 256)
    if (chunks <= 128) return launch_k(kv_append<HD, 1, 128>, grid, dim3(128), 0, s, a, reach, status);
    if (chunks <= 256) return launch_k(kv_append<HD, 1, 256>, grid, dim3(256), 0, s, a, reach, status);
    if (chunks <= 512) return launch_k(kv_append<HD, 2, 256>, grid, dim3(256), 0, s, a, reach, status);
    if (chunks <= 1024) return launch_k(kv_append<HD, 4, 256>, grid, dim3(256), 0, s, a, reach, status);
    if (chunks <= 2048) return launch_k(kv_append<HD, 4, 512>, grid, dim3(512), 0, s, a, reach, status);
    return launch_k(kv_append<HD, 8, 512>, grid, dim3(512), 0, s, a, reach, status);
}

}  // namespace

cudaError_t launch_kv_cache_append_e4m3(const void *qkv, const int32_t *cu, int batch, int max_len, int64_t total,
                                        int q_heads, int kv_heads, int head_dim, const int32_t *past, const int32_t *table,
                                        int width, void *k, void *v, float *ks, float *vs, int pages, int page,
                                        cudaStream_t s)
{
    AppendArgs a;
    a.qkv = static_cast<const __nv_bfloat16 *>(qkv);
    a.cu = cu, a.past = past, a.table = table;
    a.k = static_cast<uint8_t *>(k), a.v = static_cast<uint8_t *>(v);
    a.ks = ks, a.vs = vs;
    a.total = total;
    a.row = static_cast<int64_t>(q_heads + 2 * kv_heads) * head_dim;
    a.batch = batch, a.max_len = max_len, a.width = width, a.pages = pages, a.page = page, a.kv_heads = kv_heads;
    a.k_col0 = q_heads * head_dim;
    a.v_col0 = (q_heads + kv_heads) * head_dim;
    if (head_dim == 64) return append<64>(a, s);
    if (head_dim == 128) return append<128>(a, s);
    return append<256>(a, s);
}

}  // namespace fe

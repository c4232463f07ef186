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
#include "fe_e4m3.cuh"
#include "fe_internal.h"

namespace fe {
namespace {

// max |v| of 8 bf16 as the bits of an fp32 value, non-finite ones left out; bad: any of those
__device__ __forceinline__ float amax8(const uint4 &u, bool &bad)
{
    float m = 0.f;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_bf16x2(w[i]);
        bad |= !(fabsf(f.x) <= 3.402823466e38f) || !(fabsf(f.y) <= 3.402823466e38f);
        m = fmaxf(m, fmaxf(finite_abs(f.x), finite_abs(f.y)));
    }
    return m;
}

// The smallest power of two 2^e with amax <= 448 * 2^e, e >= kMinScaleExp; 0 for amax = 0.
// amax widened from bf16 is 1.f * 2^E or subnormal (far below the smallest scale).
constexpr int kMinScaleExp = -80;
__device__ __forceinline__ float block_scale(float amax)
{
    if (amax == 0.f) return 0.f;
    const uint32_t b = __float_as_uint(amax);
    int e = static_cast<int>(b >> 23) - 127 - 8;                  // 448 = 1.75 * 2^8
    if ((b & 0x7fffffu) > 0x600000u) ++e;                         // mantissa above 1.75
    e = e < kMinScaleExp ? kMinScaleExp : e;
    return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

__device__ __forceinline__ uint2 encode8(const uint4 &u, float inv, bool nan_all)
{
    if (nan_all) return make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
    const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), c = unpack_bf16x2(u.z), d = unpack_bf16x2(u.w);
    return make_uint2(pack_e4m3x4(a.x * inv, a.y * inv, b.x * inv, b.y * inv),
                      pack_e4m3x4(c.x * inv, c.y * inv, d.x * inv, d.y * inv));
}

// zeros in place of non-finite elements (values of a poisoned token)
__device__ __forceinline__ uint4 finite_only(uint4 u)
{
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & 0x7f80u) == 0x7f80u) w[i] &= 0xffff0000u;
        if ((w[i] & 0x7f800000u) == 0x7f800000u) w[i] &= 0x0000ffffu;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint32_t rescale4(uint32_t codes, float ratio)
{
    const float2 a = e4m3x2_to_f32x2(codes & 0xffffu), b = e4m3x2_to_f32x2(codes >> 16);
    return pack_e4m3x4(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
}

struct AppendArgs {
    const __nv_bfloat16 *qkv;
    const int32_t *cu, *past, *table;
    uint8_t *k, *v;
    float *ks, *vs;
    int64_t total, row;  // tokens and elements per row of qkv
    int batch, width, pages, page, kv_heads, k_col0, v_col0;
};

// THREADS threads hold CH 16-byte chunks of K and of V each: CH * THREADS * 8 >= page * HD.
template <int HD, int CH, int THREADS>
__global__ void __launch_bounds__(THREADS) kv_append(const AppendArgs a, int reach, int *status)
{
    constexpr int LPT = HD / 8;  // lanes of a token: 8, 16 or 32, aligned within a warp
    __shared__ float red[2][THREADS / 32];
    const int b = blockIdx.x / reach, nth = blockIdx.x % reach, head = blockIdx.y;
    grid_dep_wait();
    grid_dep_launch();
    const int t0 = a.cu[b], t1 = a.cu[b + 1], past = a.past[b];
    if (t1 <= t0) return;
    if (t0 < 0 || t1 > a.total || past < 0) {  // offsets that do not describe the batch: nothing is touched
        if (threadIdx.x == 0) report(status, DEV_BAD_INPUT);
        return;
    }
    const int64_t end = static_cast<int64_t>(past) + (t1 - t0);
    const int64_t ordinal = past / a.page + nth;
    const int64_t base = ordinal * a.page;  // first token of the page
    if (base >= end) return;
    if (nth == reach - 1 && base + a.page < end && threadIdx.x == 0) report(status, DEV_BAD_INPUT);  // longer than max_len
    const int id = ordinal < a.width ? a.table[static_cast<int64_t>(b) * a.width + ordinal] : -1;
    if (id < 0 || id >= a.pages) {
        if (threadIdx.x == 0) report(status, DEV_BAD_INPUT);
        return;
    }
    const int lo = past > base ? static_cast<int>(past - base) : 0;                       // first new slot
    const int hi = end - base < a.page ? static_cast<int>(end - base) : a.page;           // past the last
    const int64_t block = (static_cast<int64_t>(id) * a.kv_heads + head) * a.page * HD;  // codes of this (page, head)
    const int64_t si = static_cast<int64_t>(id) * a.kv_heads + head;
    const float k_old = lo > 0 ? a.ks[si] : 0.f, v_old = lo > 0 ? a.vs[si] : 0.f;

    uint4 kr[CH], vr[CH];
    float km = 0.f, vm = 0.f;
    uint32_t poisoned = 0;  // bit c: this thread's token of chunk c holds something non-finite
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
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        bool bad = false;
        const float mk = amax8(kr[c], bad);
        vm = fmaxf(vm, amax8(vr[c], bad));
        const uint32_t any = __ballot_sync(0xffffffffu, bad);
        const uint32_t group = (LPT == 32 ? 0xffffffffu : ((1u << LPT) - 1u) << ((threadIdx.x & 31) / LPT * LPT));
        if (any & group) poisoned |= 1u << c;
        else km = fmaxf(km, mk);  // a poisoned token's key is stored as NaN and sets no scale
    }
    km = warp_max(km);
    vm = warp_max(vm);
    if ((threadIdx.x & 31) == 0) {
        red[0][threadIdx.x >> 5] = km;
        red[1][threadIdx.x >> 5] = vm;
    }
    __syncthreads();  // also: every thread has read the old scales
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
        km = fmaxf(km, red[0][i]);
        vm = fmaxf(vm, red[1][i]);
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
            const bool nan = (poisoned >> c) & 1u;
            *reinterpret_cast<uint2 *>(a.k + block + chunk * 8) = encode8(kr[c], k_inv, nan);
            *reinterpret_cast<uint2 *>(a.v + block + chunk * 8) = encode8(nan ? finite_only(vr[c]) : vr[c], v_inv, false);
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
cudaError_t append(const AppendArgs &a, int max_len, cudaStream_t s)
{
    const int reach = (a.page - 1 + max_len - 1) / a.page + 1;  // pages that max_len tokens at any offset can touch
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
    a.batch = batch, a.width = width, a.pages = pages, a.page = page, a.kv_heads = kv_heads;
    a.k_col0 = q_heads * head_dim;
    a.v_col0 = (q_heads + kv_heads) * head_dim;
    if (head_dim == 64) return append<64>(a, max_len, s);
    if (head_dim == 128) return append<128>(a, max_len, s);
    return append<256>(a, max_len, s);
}

}  // namespace fe

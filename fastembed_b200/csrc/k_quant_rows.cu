// k_quant_rows.cu — rows to e4m3 codes with one fp32 scale each, and the residual add +
// RMSNorm whose output is such a row: the 8-bit counterparts of the bf16 row kernels that
// feed the projections.
//
//     s_i = max(max_j |v_ij|, 2^-110) / 448,   q_ij = e4m3(v_ij / s_i)
//
// with v the input row, or v = h / sqrt(mean(h^2) + eps) * w after h += y.  The maximum is
// over the finite values; what is not finite takes the NaN code, so it poisons its own row of
// the product that reads the codes and leaves the row's other codes as they would be.
//
// The maximum is known only after the whole row, so the row stays in registers between the
// reads and the writes: every input byte is read once and every output byte written once, and
// the kernels are bound by HBM.  A row of at most 2048 values is one warp's (up to eight
// 8-value chunks a lane); wider rows, and launches of so few rows that one warp each would
// leave most of the SMs idle, take a block of 256 threads a row.  Rows that are wider than
// 16384 or whose width is not a multiple of 8 (or unaligned) take a scalar kernel that reads
// the row again (from L2) in place of keeping it.
#include "fe_e4m3.cuh"
#include "fe_internal.h"

namespace fe {
namespace {

constexpr int kRowThreads = 256;
constexpr int kWarpRowThreads = 128;  // of a block of warps with a row each: 26,508 x 1,024 and 71,550 x 2,048 within 2 % of 256

__device__ __forceinline__ void load8(const float *p, float (&v)[8])
{
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&v)[8])
{
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), c = unpack_bf16x2(u.z), d = unpack_bf16x2(u.w);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// Reduction over the threads of a row: the warp's lanes, or the whole block (every thread gets
// the result; `red` is one float per warp, free to be written again after the call).
template <bool BLOCK, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float *red)
{
    v = MAX ? warp_max(v) : warp_sum(v);
    if constexpr (BLOCK) {
        constexpr int W = kRowThreads / 32;
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < W; ++i) v = MAX ? fmaxf(v, red[i]) : v + red[i];
        __syncthreads();
    }
    return v;
}

// IT: the input (quantiser) or the residual branch y (norm) element; BLOCK: a block per row,
// else a warp; CH: 8-value chunks per thread.
template <class IT, bool NORM, bool BLOCK, int CH>
__global__ void __launch_bounds__(BLOCK ? kRowThreads : kWarpRowThreads)
    rows_to_e4m3(const IT *__restrict__ x, float *h32, const float *__restrict__ w, float wadd, float eps, int64_t rows,
                 int dim, uint8_t *__restrict__ q, float *__restrict__ scale)
{
    constexpr int T = BLOCK ? kRowThreads : 32;
    __shared__ float red[kRowThreads / 32];
    const int t = BLOCK ? threadIdx.x : threadIdx.x & 31;
    const int64_t r = BLOCK ? static_cast<int64_t>(blockIdx.x)
                            : static_cast<int64_t>(blockIdx.x) * (kWarpRowThreads / 32) + (threadIdx.x >> 5);
    grid_dep_wait();
    grid_dep_launch();
    if (r >= rows) return;  // whole warps only: a block-per-row launch has exactly `rows` blocks
    float v[CH][8];
    if constexpr (NORM) {
        float *hr = h32 + r * dim;
        const IT *yr = x ? x + r * dim : nullptr;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * T + t) * 8;
            if (col < dim) load8(hr + col, v[c]);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] = 0.f;
        }
        if (yr) {
            float y[CH][8];
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (c * T + t) * 8;
                if (col < dim) load8(yr + col, y[c]);
                else
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[c][j] = 0.f;
            }
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (c * T + t) * 8;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] += y[c][j];
                if (col < dim) {
                    *reinterpret_cast<float4 *>(hr + col) = make_float4(v[c][0], v[c][1], v[c][2], v[c][3]);
                    *reinterpret_cast<float4 *>(hr + col + 4) = make_float4(v[c][4], v[c][5], v[c][6], v[c][7]);
                }
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                s0 = fmaf(v[c][j], v[c][j], s0);
                s1 = fmaf(v[c][j + 1], v[c][j + 1], s1);
            }
            ss += s0 + s1;
        }
        const float rms = 1.0f / sqrtf(row_reduce<BLOCK, false>(ss, red) / static_cast<float>(dim) + eps);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * T + t) * 8;
            if (col < dim) {
                float g[8];
                load8(w + col, g);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] *= rms * (g[j] + wadd);
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * T + t) * 8;
            if (col < dim) load8(x + r * dim + col, v[c]);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] = 0.f;
        }
    }
    float m = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[c][j]));
    m = fmaxf(row_reduce<BLOCK, true>(m, red), kTinyAmax);
    const float s = m / kE4m3Max, inv = 1.0f / s;
    if (t == 0) scale[r] = s;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * T + t) * 8;
        if (col < dim) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                v[c][j] = finite_or_nan(v[c][j]);
                v[c][j + 1] = finite_or_nan(v[c][j + 1]);
                div_by2(v[c][j], v[c][j + 1], s, inv);
            }
            *reinterpret_cast<uint2 *>(q + r * dim + col) =
                make_uint2(pack_e4m3x4(v[c][0], v[c][1], v[c][2], v[c][3]), pack_e4m3x4(v[c][4], v[c][5], v[c][6], v[c][7]));
        }
    }
}

// The quantiser of bf16 rows, a warp each: the row waits for its maximum as it came, half the
// registers of its fp32 values (71,550 x 2,048: 76 us with those, 65 so), and the maximum
// is taken on the bits, which order like the values, infinities and NaN last.
template <int CH>
__global__ void __launch_bounds__(kWarpRowThreads)
    bf16_rows_to_e4m3(const __nv_bfloat16 *__restrict__ x, int64_t rows, int dim, uint8_t *__restrict__ q,
                      float *__restrict__ scale)
{
    constexpr uint32_t inf = 0x7f80u;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * (kWarpRowThreads / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    grid_dep_wait();
    grid_dep_launch();
    if (r >= rows) return;
    uint4 u[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * 32 + lane) * 8;
        u[c] = col < dim ? *reinterpret_cast<const uint4 *>(x + r * dim + col) : make_uint4(0, 0, 0, 0);
    }
    uint32_t m2 = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c)
        m2 = __vmaxu2(m2, __vmaxu2(__vmaxu2(u[c].x & 0x7fff7fffu, u[c].y & 0x7fff7fffu),
                                   __vmaxu2(u[c].z & 0x7fff7fffu, u[c].w & 0x7fff7fffu)));
    uint32_t m = __reduce_max_sync(0xffffffffu, max(m2 & 0xffffu, m2 >> 16));
    if (m >= inf) {  // rare: the maximum without what is not finite, and NaN in its place
        m = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            uint32_t w[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if ((w[i] & inf) == inf) w[i] |= 0x7fffu;
                else m = max(m, w[i] & 0x7fffu);
                if ((w[i] & (inf << 16)) == inf << 16) w[i] |= 0x7fff0000u;
                else m = max(m, (w[i] >> 16) & 0x7fffu);
            }
            u[c] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        m = __reduce_max_sync(0xffffffffu, m);
    }
    const float s = fmaxf(__uint_as_float(m << 16), kTinyAmax) / kE4m3Max, inv = 1.0f / s;
    if (lane == 0) scale[r] = s;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * 32 + lane) * 8;
        float2 a = unpack_bf16x2(u[c].x), b = unpack_bf16x2(u[c].y), d = unpack_bf16x2(u[c].z), e = unpack_bf16x2(u[c].w);
        div_by2(a.x, a.y, s, inv);
        div_by2(b.x, b.y, s, inv);
        div_by2(d.x, d.y, s, inv);
        div_by2(e.x, e.y, s, inv);
        if (col < dim)
            *reinterpret_cast<uint2 *>(q + r * dim + col) =
                make_uint2(pack_e4m3x4(a.x, a.y, b.x, b.y), pack_e4m3x4(d.x, d.y, e.x, e.y));
    }
}

// Any width and alignment: a block per row, the row read again for each pass.
template <class IT, bool NORM>
__global__ void __launch_bounds__(kRowThreads)
    rows_to_e4m3_any(const IT *__restrict__ x, float *h32, const float *__restrict__ w, float wadd, float eps, int dim,
                     uint8_t *__restrict__ q, float *__restrict__ scale)
{
    __shared__ float red[kRowThreads / 32];
    const int64_t r = blockIdx.x;
    grid_dep_wait();
    grid_dep_launch();
    float rms = 1.f;
    float *hr = NORM ? h32 + r * dim : nullptr;
    const IT *xr = x ? x + r * dim : nullptr;
    if constexpr (NORM) {
        float ss = 0.f;
        for (int c = threadIdx.x; c < dim; c += kRowThreads) {
            float h = hr[c];
            if (xr) {
                h += widen(xr[c]);
                hr[c] = h;
            }
            ss = fmaf(h, h, ss);
        }
        rms = 1.0f / sqrtf(row_reduce<true, false>(ss, red) / static_cast<float>(dim) + eps);
    }
    // a thread reads back only what it wrote itself
    auto value = [&](int c) { return NORM ? hr[c] * (rms * (w[c] + wadd)) : widen(xr[c]); };
    float m = 0.f;
    for (int c = threadIdx.x; c < dim; c += kRowThreads) m = fmaxf(m, finite_abs(value(c)));
    m = fmaxf(row_reduce<true, true>(m, red), kTinyAmax);
    const float s = m / kE4m3Max, inv = 1.0f / s;
    if (threadIdx.x == 0) scale[r] = s;
    for (int c = threadIdx.x; c < dim; c += kRowThreads)
        q[r * dim + c] = static_cast<uint8_t>(cvt_e4m3x2(div_by(finite_or_nan(value(c)), s, inv), 0.f));
}

struct RowArgs {
    const void *x;
    float *h32;
    const float *w;
    float wadd, eps;
    int64_t rows;
    int dim;
    void *q;
    float *scale;
};

template <class IT, bool NORM, bool BLOCK, int CH>
cudaError_t go(const RowArgs &a, cudaStream_t s)
{
    constexpr int per = kWarpRowThreads / 32;
    const int64_t grid = BLOCK ? a.rows : (a.rows + per - 1) / per;
    if constexpr (!NORM && !BLOCK && sizeof(IT) == 2)
        return launch_k(bf16_rows_to_e4m3<CH>, dim3(static_cast<unsigned>(grid)), dim3(kWarpRowThreads), 0, s,
                        static_cast<const IT *>(a.x), a.rows, a.dim, static_cast<uint8_t *>(a.q), a.scale);
    else
        return launch_k(rows_to_e4m3<IT, NORM, BLOCK, CH>, dim3(static_cast<unsigned>(grid)),
                        dim3(BLOCK ? kRowThreads : kWarpRowThreads), 0, s, static_cast<const IT *>(a.x), a.h32, a.w, a.wadd,
                        a.eps, a.rows, a.dim, static_cast<uint8_t *>(a.q), a.scale);
}

template <class IT, bool NORM>
cudaError_t pick(const RowArgs &a, cudaStream_t s)
{
    auto aligned = [](const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
    const int chunks = a.dim / 8;  // 8-value chunks of a row
    if (a.dim % 8 != 0 || chunks > 8 * kRowThreads || !aligned(a.x, 16) || !aligned(a.h32, 16) || !aligned(a.w, 16) ||
        !aligned(a.q, 8))
        return launch_k(rows_to_e4m3_any<IT, NORM>, dim3(static_cast<unsigned>(a.rows)), dim3(kRowThreads), 0, s,
                        static_cast<const IT *>(a.x), a.h32, a.w, a.wadd, a.eps, a.dim, static_cast<uint8_t *>(a.q),
                        a.scale);
    // fewer rows than SMs: a block a row puts a row's loads in flight at once
    const bool few = a.rows <= current_sm_count() && chunks > 32;
    if (chunks <= 8 * 32 && !few) {
        if (chunks <= 32) return go<IT, NORM, false, 1>(a, s);
        if (chunks <= 64) return go<IT, NORM, false, 2>(a, s);
        if (chunks <= 128) return go<IT, NORM, false, 4>(a, s);
        return go<IT, NORM, false, 8>(a, s);
    }
    if (chunks <= kRowThreads) return go<IT, NORM, true, 1>(a, s);
    if (chunks <= 2 * kRowThreads) return go<IT, NORM, true, 2>(a, s);
    if (chunks <= 4 * kRowThreads) return go<IT, NORM, true, 4>(a, s);
    return go<IT, NORM, true, 8>(a, s);
}

}  // namespace

cudaError_t launch_quantize_rows_e4m3(const void *x, int x_dtype, int64_t rows, int dim, void *q, float *scale,
                                      cudaStream_t s)
{
    const RowArgs a{x, nullptr, nullptr, 0.f, 0.f, rows, dim, q, scale};
    return x_dtype == FE_DTYPE_BF16 ? pick<__nv_bfloat16, false>(a, s) : pick<float, false>(a, s);
}

cudaError_t launch_add_rmsnorm_e4m3(const void *y, int y_dtype, float *h32, const float *w, bool one_plus, float eps,
                                    int64_t rows, int dim, void *q, float *scale, cudaStream_t s)
{
    const RowArgs a{y, h32, w, one_plus ? 1.f : 0.f, eps, rows, dim, q, scale};
    return y_dtype == FE_DTYPE_BF16 ? pick<__nv_bfloat16, true>(a, s) : pick<float, true>(a, s);
}

}  // namespace fe

// k_attention_cache.cu — attention of new tokens over the paged 8-bit key-value cache.
//
//     out_i = sum_j p_ij v_j,   p_ij = softmax_j(scale * q_i . k_j),   j <= past + i (causal)
//                                                                  or j < past + len
// with k_j = kc_j sk(page), v_j = vc_j sv(page): e4m3 codes times the scale of their page and
// head.  The scales leave the products:
//     s_ij = (scale log2 e) sk q_i . kc_j          (base-2 logits)
//     t_ij = s_ij + log2 sv,   P_ij = 2^(t_ij - m_i),   m_i = max_j t_ij - 15
//     out_i = 2^(m_i - n_i) (sum_j P_ij vc_j) / (sum_j 2^(s_ij - n_i)),   n_i = max_j s_ij
// so the value scale moves into the exponent, the running maximum m is that of the weights as they
// meet the codes, and P (at most 2^15) keeps 11 bits in f16 with nothing above 2^-39 of the
// largest weight lost, whatever the pages' scales are.  A page of zero values (sv = 0: t = -inf) takes part
// in the sum of weights only, and that sum has a reference of its own, which no value scale moves.
// Statistics and sums are fp32.
//
// attn_cache_stream: the form for few rows (single tokens).  A key-value head's rows are its
// query heads' new tokens together, r = token * group + head, 8 NR of them to a CTA.  Nothing is
// shared between warps but the final sum: each warp takes every WARPS-th run of 32 tokens (16 at
// head_dim 256) of its CTA's part of the sequence, through a cp.async ring of its own, into the
// fragments of mma.m16n8k16.
//   S^T [tokens x rows] = K Q^T: A is K.  A thread's 16 consecutive bytes of a token (one shared-
//     memory load) are the four k-pairs of four k-steps: the order of k inside the sum is free, so
//     Q's fragments are loaded in that order once.
//   O^T [hd x rows] = V^T P^T: A is V^T.  A thread reads 16 consecutive codes of four tokens and
//     pairs them up by byte permutes; which hd row a fragment row stands for is free too (row g
//     of m-tile i is hd 16 g + 2 i).  P^T in B-fragment form is the 8x8 transpose of S^T's
//     accumulator.
// Each e4m3 pair becomes f16x2 in one conversion (exact).  The sequence is split over CTAs when
// there are too few to fill the GPU.  Up to eight parts are the CTAs of a cluster, which sum them
// through distributed shared memory; more (one long sequence) go through the workspace and
// attn_cache_join, a launch later.
//
// Pages beyond the sequence are never read; slots past its end are masked before they are used
// (values zeroed: a slot never written may hold any code).  A page id outside the pool sets
// FE_ERR_INVALID_ARGUMENT in the device status word and its tokens are left out.
#include <algorithm>

#include "fe_attention_cache.cuh"

namespace fe {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBoost = 15.f;  // P is at most 2^15
constexpr int kSms = 148;

// D += A B, m16n8k16, f16 inputs, fp32 accumulator
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds16(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ uint2 lds8(uint32_t addr)
{
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}

template <int HD, int NR, int WARPS>
struct StreamCfg {
    static constexpr int ROWS = 8 * NR;
    static constexpr int U = HD == 256 ? 1 : 2;          // 16-token tiles of a run
    static constexpr int RUN = 16 * U;                   // tokens of a run
    static constexpr int STAGES = 2;
    static constexpr uint32_t TILE = 16 * HD;            // bytes of a tile's K or V
    static constexpr uint32_t STAGE = U * 2 * TILE + 16; // K, V of each tile, then sk, sv of both
    static constexpr uint32_t RING = STAGES * STAGE;     // of a warp
    static constexpr int LD = HD + 4;                    // floats per row of the joining buffer
    static constexpr uint32_t JOIN = (WARPS * ROWS * (LD + 4) + ROWS * 4) * 4;
    static constexpr uint32_t SMEM = WARPS * RING > JOIN ? WARPS * RING : JOIN;
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

// Byte offset of 16-byte chunk `ch` of token `row` in a staged tile.  Chunks are permuted within
// 128 bytes so that the eight lanes of a phase meet eight different ones, reading K (a row's
// chunks 4 j + c, two rows a phase) as well as V (chunk g or g / 2 of four rows).
template <int HD>
__device__ __forceinline__ uint32_t staged(int row, int ch)
{
    if constexpr (HD == 64) {
        const int line = row >> 1;
        return line * 128 + (((((row & 1) << 2) | ch) ^ ((2 * line) & 7)) << 4);
    } else {
        return row * HD + ((ch ^ (row & 7)) << 4);
    }
}

// The token of a 16-token tile that row g (0..7; g + 8: token + 8) of an MMA fragment stands for:
// any order does, and this one keeps K's rows of a phase (g, g + 1) in different 64-byte halves
// and V's (even or odd g) in different chunks.
template <int HD>
__device__ __forceinline__ int token_of(int g)
{
    if constexpr (HD == 64) return g;
    else return (g & 2) | (g >> 2) | (((g ^ (g >> 2)) & 1) << 2);
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// CLUSTER: the launch's parts (gridDim.z of them) are one cluster along z.
template <int HD, int NR, int WARPS, bool CLUSTER>
__global__ void __launch_bounds__(32 * WARPS) attn_cache_stream(const CacheArgs a, int row_tiles, int *status)
{
    using C = StreamCfg<HD, NR, WARPS>;
    constexpr int KC = HD / 64;            // 16-byte chunks of a token's key per thread
    constexpr int VB = HD >= 128 ? 16 : 8; // bytes of a token's value per thread and 128 (64) codes
    constexpr int VC = HD >= 128 ? HD / 128 : 1;
    constexpr int VW = VB / 4;             // words of those
    constexpr int MT = HD / 16;            // m-tiles of O^T
    // the warps' rings; at the end [WARPS][ROWS][LD], then [WARPS][ROWS][4], then [ROWS][4] floats
    extern __shared__ __align__(16) float join[];

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, c = lane & 3;
    const int split = blockIdx.z, kvh = blockIdx.y;
    const int b = blockIdx.x / row_tiles, tile = blockIdx.x % row_tiles;
    grid_dep_wait();
    grid_dep_launch();
    CacheSeq sq;
    if (!load_seq(a, b, sq, status)) return;
    const int rows = sq.len * a.group, r0 = tile * C::ROWS;
    if (r0 >= rows) return;

    // Q fragments (column n = g of each 8-row tile), each row brought to [1, 2) at its maximum by
    // a power of two so that f16 holds every bf16 of it
    uint32_t qf[NR][KC][4][2];
    float qs[NR][2];   // base-2 logit factor of rows 2c, 2c + 1
    int lim[NR][2];    // last visible token of rows 2c, 2c + 1 (-1: no such row)
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int r = r0 + 8 * n + g;
        float f[KC][16];
        float m = 0.f;
        if (r < rows) {
            const __nv_bfloat16 *p =
                a.qkv + (sq.t0 + r / a.group) * a.row + static_cast<int64_t>(kvh * a.group + r % a.group) * HD + 16 * c;
#pragma unroll
            for (int j = 0; j < KC; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 u = *reinterpret_cast<const uint4 *>(p + 64 * j + 8 * h);
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 x = unpack_bf16x2(w[i]);
                        // an infinity becomes NaN (0 * inf): its products could all be -inf, a row that sees nothing
                        f[j][8 * h + 2 * i] = fmaf(x.x, 0.f, x.x);
                        f[j][8 * h + 2 * i + 1] = fmaf(x.y, 0.f, x.y);
                        m = fmaxf(m, fmaxf(finite_abs(x.x), finite_abs(x.y)));
                    }
                }
        } else {
#pragma unroll
            for (int j = 0; j < KC; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) f[j][i] = 0.f;
        }
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        // 2^-e and 2^e of the row's exponent, e in [-126, 127] (subnormal rows stay below 1, well above f16's steps)
        int e = static_cast<int>(__float_as_uint(m) >> 23) - 127;
        e = e < -126 ? -126 : e;
        const float down = __uint_as_float(static_cast<uint32_t>(127 - (e > 126 ? 126 : e)) << 23);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + (e > 126 ? 126 : e)) << 23);
#pragma unroll
        for (int j = 0; j < KC; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                qf[n][j][q][0] = pack_f16x2(f[j][4 * q] * down, f[j][4 * q + 1] * down);
                qf[n][j][q][1] = pack_f16x2(f[j][4 * q + 2] * down, f[j][4 * q + 3] * down);
            }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int rr = r0 + 8 * n + 2 * c + h;
            qs[n][h] = __shfl_sync(0xffffffffu, up, (2 * c + h) * 4) * a.scale_log2;
            lim[n][h] = rr >= rows ? -1 : a.causal ? sq.past + rr / a.group : sq.kv - 1;
        }
    }
    // tokens this CTA reads: its part of those its last row sees
    const int last_row = min(r0 + C::ROWS, rows) - 1;
    const int end_all = a.causal ? sq.past + last_row / a.group + 1 : sq.kv;
    const int runs = (end_all + C::RUN - 1) / C::RUN;
    const int per = (runs + a.splits - 1) / a.splits;
    const int run0 = split * per, run1 = min(run0 + per, runs);

    float o[NR][MT][4];
    float mx[NR][2];            // the row's reference for O
    float nx[NR][2], l[NR][2];  // the lane's own for its part of the sum
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[n][i][j] = 0.f;
        mx[n][0] = mx[n][1] = nx[n][0] = nx[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
    }

    // A run is C::U 16-token tiles, each inside one page (pages are 16 tokens or more).  Each warp
    // streams its runs through a ring of its own, two runs on their way while it works, with no
    // registers held for them.  32 sequences of 16,000 tokens: 184 us (87 % of the copy bandwidth),
    // loaded straight into fragments one run ahead 197; three stages, and so two CTAs an SM in place
    // of three, 208: the warps matter more than the depth.
    const int32_t *tab = a.table + static_cast<int64_t>(b) * a.width;
    const int page_mask = (1 << a.page_log2) - 1;
    const uint32_t ring = smem_u32(join) + warp * C::RING;
    auto look_up = [&](int run, int (&id)[C::U]) {  // the run's pages, -1: none
#pragma unroll
        for (int u = 0; u < C::U; ++u) {
            const int tok = run * C::RUN + 16 * u;
            id[u] = -1;
            if (run < run1 && tok < end_all) {
                id[u] = __ldg(tab + (tok >> a.page_log2));
                if (id[u] < 0) id[u] = a.pages;  // as bad as any id past the pool
            }
        }
    };
    auto request = [&](int run, int (&id)[C::U], uint32_t st) {
#pragma unroll
        for (int u = 0; u < C::U; ++u) {
            if (id[u] >= a.pages) {
                if (lane == 0) report(status, DEV_BAD_INPUT);
                id[u] = -1;
            }
            const uint32_t e = st + C::U * 2 * C::TILE + 4 * u;
            if (id[u] >= 0) {
                const int64_t ph = static_cast<int64_t>(id[u]) * a.kv_heads + kvh;
                const int64_t at = ((ph << a.page_log2) + ((run * C::RUN + 16 * u) & page_mask)) * HD + 16 * lane;
                const uint32_t k = st + u * 2 * C::TILE;
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) {  // 32 chunks at a time
                    const int x = 32 * i + lane;
                    const uint32_t to = staged<HD>(x / (HD / 16), x % (HD / 16));
                    cp_async16(k + to, a.k + at + 512 * i);
                    cp_async16(k + C::TILE + to, a.v + at + 512 * i);
                }
                if (lane < 2) cp_async4(e + 8 * lane, (lane ? a.vs : a.ks) + ph);
            } else if (lane < 2) {  // a value scale below 0: no page
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(e + 8 * lane), "f"(lane ? -1.f : 0.f) : "memory");
            }
        }
        cp_async_commit();
    };
    int ahead = run0 + warp, id[C::U];  // the next run to be requested and its pages
    {
        int first[C::STAGES][C::U];
#pragma unroll
        for (int i = 0; i < C::STAGES; ++i) look_up(ahead + i * WARPS, first[i]);
        look_up(ahead + C::STAGES * WARPS, id);
#pragma unroll
        for (int i = 0; i < C::STAGES; ++i, ahead += WARPS) request(ahead, first[i], ring + i * C::STAGE);
    }
    const int tg = token_of<HD>(g), tv[2] = {token_of<HD>(2 * c), token_of<HD>(2 * c + 1)};
    uint32_t st = ring;
    for (int run = run0 + warp; run < run1; run += WARPS) {
        cp_async_wait<C::STAGES - 1>();
        __syncwarp();  // every lane's part of the run has arrived
        float sk[2], sv[2];
        {
            const uint4 e = lds16(st + C::U * 2 * C::TILE);
            sk[0] = __uint_as_float(e.x), sk[1] = __uint_as_float(e.y);
            sv[0] = __uint_as_float(e.z), sv[1] = __uint_as_float(e.w);
        }
        // S^T: accumulator (token g, row 2c), (g, 2c + 1), (g + 8, 2c), (g + 8, 2c + 1)
        float s[NR][C::U][4];
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int u = 0; u < C::U; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][u][i] = 0.f;
#pragma unroll
        for (int u = 0; u < C::U; ++u)
#pragma unroll
            for (int j = 0; j < KC; ++j) {
                const uint32_t at = st + u * 2 * C::TILE + staged<HD>(tg, 4 * j + c);
                const uint4 x = lds16(at), y = lds16(at + 8 * HD);
                const uint32_t lo[4] = {x.x, x.y, x.z, x.w}, hi[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t a0 = e4m3x2_to_f16x2(lo[q]), a1 = e4m3x2_to_f16x2(hi[q]);
                    const uint32_t a2 = e4m3x2_to_f16x2(lo[q] >> 16), a3 = e4m3x2_to_f16x2(hi[q] >> 16);
#pragma unroll
                    for (int n = 0; n < NR; ++n) mma_f16(s[n][u], a0, a1, a2, a3, qf[n][j][q][0], qf[n][j][q][1]);
                }
            }
        // base-2 logits, masked; t = s + log2 sv (-inf for a page of zero values: it adds to the sum alone)
        float ev[2];
#pragma unroll
        for (int u = 0; u < C::U; ++u) ev[u] = sv[u] > 0.f ? log2f(sv[u]) : -INFINITY;
        uint32_t pt[NR][C::U][2];  // P^T fragments [tile][tokens 2c.. / 2c + 8..]
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            float top[2] = {mx[n][0], mx[n][1]}, sum_top[2] = {nx[n][0], nx[n][1]};
#pragma unroll
            for (int u = 0; u < C::U; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = run * C::RUN + 16 * u + tg + 8 * (i >> 1);
                    const bool on = sv[u] >= 0.f && tok <= lim[n][i & 1];
                    s[n][u][i] = on ? s[n][u][i] * (sk[u] * qs[n][i & 1]) : -INFINITY;
                    top[i & 1] = fmaxf(top[i & 1], s[n][u][i] + ev[u]);
                    sum_top[i & 1] = fmaxf(sum_top[i & 1], s[n][u][i]);
                }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], d));
            }
            const bool grew = top[0] > mx[n][0] || top[1] > mx[n][1];
            if (__any_sync(0xffffffffu, grew)) {
                float f[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f[h] = mx[n][h] == -INFINITY ? 0.f : exp2_fast(mx[n][h] - top[h]);
                    mx[n][h] = top[h];
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    o[n][i][0] *= f[0];
                    o[n][i][1] *= f[1];
                    o[n][i][2] *= f[0];
                    o[n][i][3] *= f[1];
                }
            }
            const float ref[2] = {mx[n][0] == -INFINITY ? 0.f : mx[n][0] - kBoost,
                                  mx[n][1] == -INFINITY ? 0.f : mx[n][1] - kBoost};
            float sum_ref[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                sum_ref[h] = sum_top[h] == -INFINITY ? 0.f : sum_top[h];
                l[n][h] *= exp2_fast(nx[n][h] - sum_ref[h]);
                nx[n][h] = sum_top[h];
            }
#pragma unroll
            for (int u = 0; u < C::U; ++u) {
                float p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[i] = exp2_fast(s[n][u][i] + ev[u] - ref[i & 1]);
                    l[n][i & 1] += exp2_fast(s[n][u][i] - sum_ref[i & 1]);
                }
                pt[n][u][0] = transpose8x8(pack_f16x2(p[0], p[1]));
                pt[n][u][1] = transpose8x8(pack_f16x2(p[2], p[3]));
            }
        }
        // O^T: m-tile (j, 2 w) holds codes 4 w, 4 w + 1 of a thread's run of 16 (8), (j, 2 w + 1) the next two
#pragma unroll
        for (int u = 0; u < C::U; ++u) {
            const uint32_t vt = st + u * 2 * C::TILE + C::TILE;
            const int tok0 = run * C::RUN + 16 * u;
            // slots past the sequence's end hold anything, a NaN code among it, and a page that is not
            // there leaves the stage as it was: 0 * NaN would be NaN
            const bool check = tok0 + 16 > sq.kv || sv[u] < 0.f;
#pragma unroll
            for (int j = 0; j < VC; ++j) {
                uint32_t vf[4][VW];  // [token 2c, 2c + 1, 2c + 8, 2c + 9][word]
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = tv[i & 1];
                    if constexpr (VB == 16) {
                        const uint4 x = lds16(vt + staged<HD>(row, 8 * j + g) + (i >> 1) * 8 * HD);
                        vf[i][0] = x.x, vf[i][1] = x.y, vf[i][2] = x.z, vf[i][3] = x.w;
                    } else {
                        const uint2 x = lds8(vt + staged<HD>(row, g >> 1) + 8 * (g & 1) + (i >> 1) * 8 * HD);
                        vf[i][0] = x.x, vf[i][1] = x.y;
                    }
                    if (check)
                        if (sv[u] < 0.f || tok0 + row + 8 * (i >> 1) >= sq.kv)
#pragma unroll
                            for (int w = 0; w < VW; ++w) vf[i][w] = 0;
                }
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    const uint32_t x0 = __byte_perm(vf[0][w], vf[1][w], 0x5140);
                    const uint32_t x1 = __byte_perm(vf[0][w], vf[1][w], 0x7362);
                    const uint32_t y0 = __byte_perm(vf[2][w], vf[3][w], 0x5140);
                    const uint32_t y1 = __byte_perm(vf[2][w], vf[3][w], 0x7362);
                    const uint32_t a0 = e4m3x2_to_f16x2(x0), a1 = e4m3x2_to_f16x2(x0 >> 16);
                    const uint32_t a2 = e4m3x2_to_f16x2(y0), a3 = e4m3x2_to_f16x2(y0 >> 16);
                    const uint32_t b0 = e4m3x2_to_f16x2(x1), b1 = e4m3x2_to_f16x2(x1 >> 16);
                    const uint32_t b2 = e4m3x2_to_f16x2(y1), b3 = e4m3x2_to_f16x2(y1 >> 16);
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        mma_f16(o[n][2 * VW * j + 2 * w], a0, a1, a2, a3, pt[n][u][0], pt[n][u][1]);
                        mma_f16(o[n][2 * VW * j + 2 * w + 1], b0, b1, b2, b3, pt[n][u][0], pt[n][u][1]);
                    }
                }
            }
        }
        __syncwarp();  // the stage is read: the run STAGES on takes it
        request(ahead, id, st);
        ahead += WARPS;
        look_up(ahead, id);
        st += C::STAGE;
        if (st == ring + C::RING) st = ring;
    }
    cp_async_wait<0>();
    __syncthreads();  // the rings become the joining buffer

    // join the warps: each leaves its rows' references, sum and O, then the CTA adds them up
    float4 *mn = reinterpret_cast<float4 *>(join + WARPS * C::ROWS * C::LD), *cmn = mn + WARPS * C::ROWS;
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float top = nx[n][h];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            float t = l[n][h] * part_weight(nx[n][h], top);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
            const int r = 8 * n + 2 * c + h;
            if (g == 0) mn[warp * C::ROWS + r] = make_float4(mx[n][h] - kBoost, top, t, 0.f);
            float *dst = join + (warp * C::ROWS + r) * C::LD;
#pragma unroll
            for (int j = 0; j < VC; ++j)
#pragma unroll
                for (int i = 0; i < 2 * VW; ++i) {
                    const int mt = 2 * VW * j + i, hd = 128 * j + VB * g + 2 * i;
                    *reinterpret_cast<float2 *>(dst + hd) = make_float2(o[n][mt][h], o[n][mt][2 + h]);
                }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < C::ROWS * HD / 4; i += 32 * WARPS) {
        const int r = i / (HD / 4), hd = i % (HD / 4) * 4;
        if (r0 + r >= rows) break;
        RowPart sum{-INFINITY, -INFINITY, 0.f};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float4 p = mn[w * C::ROWS + r];
            sum.m = fmaxf(sum.m, p.x);
            sum.n = fmaxf(sum.n, p.y);
        }
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float4 p = mn[w * C::ROWS + r];
            const float4 x = *reinterpret_cast<const float4 *>(join + (w * C::ROWS + r) * C::LD + hd);
            const float k = part_weight(p.x, sum.m);
            sum.l += p.z * part_weight(p.y, sum.n);
            acc.x += x.x * k, acc.y += x.y * k, acc.z += x.z * k, acc.w += x.w * k;
        }
        if constexpr (CLUSTER) {  // this CTA's part, for the cluster to read
            *reinterpret_cast<float4 *>(join + r * C::LD + hd) = acc;  // only this thread has read it
            if (hd == 0) cmn[r] = make_float4(sum.m, sum.n, sum.l, 0.f);
            continue;
        }
        const int64_t orow = (sq.t0 + (r0 + r) / a.group) * static_cast<int64_t>(a.q_heads) + kvh * a.group + (r0 + r) % a.group;
        if (a.splits == 1) {
            const RowFactor f = row_factor(sum.m, sum.n, sum.l);
            *reinterpret_cast<uint2 *>(a.out + orow * HD + hd) =
                make_uint2(pack_bf16x2(f(acc.x), f(acc.y)), pack_bf16x2(f(acc.z), f(acc.w)));
        } else {
            const int64_t at = orow * a.splits + split;
            *reinterpret_cast<float4 *>(a.part_o + at * HD + hd) = acc;
            if (hd == 0) *reinterpret_cast<float4 *>(a.part_mn + at * 4) = make_float4(sum.m, sum.n, sum.l, 0.f);
        }
    }
    if constexpr (CLUSTER) {
        const int parts = gridDim.z;
        __syncthreads();
        cluster_sync();  // every part is in its CTA's shared memory
        for (int i = split + parts * threadIdx.x; i < C::ROWS * HD / 4; i += parts * 32 * WARPS) {
            const int r = i / (HD / 4), hd = i % (HD / 4) * 4;
            if (r0 + r >= rows) break;
            RowPart sum{-INFINITY, -INFINITY, 0.f};
            for (int k = 0; k < parts; ++k) {
                const float4 p = ld_cluster4(map_to_rank(cmn + r, k));
                sum.m = fmaxf(sum.m, p.x);
                sum.n = fmaxf(sum.n, p.y);
            }
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = 0; k < parts; ++k) {
                const float4 p = ld_cluster4(map_to_rank(cmn + r, k));
                const float4 x = ld_cluster4(map_to_rank(join + r * C::LD + hd, k));
                const float f = part_weight(p.x, sum.m);
                sum.l += p.z * part_weight(p.y, sum.n);
                acc.x += x.x * f, acc.y += x.y * f, acc.z += x.z * f, acc.w += x.w * f;
            }
            const RowFactor f = row_factor(sum.m, sum.n, sum.l);
            const int64_t orow =
                (sq.t0 + (r0 + r) / a.group) * static_cast<int64_t>(a.q_heads) + kvh * a.group + (r0 + r) % a.group;
            *reinterpret_cast<uint2 *>(a.out + orow * HD + hd) =
                make_uint2(pack_bf16x2(f(acc.x), f(acc.y)), pack_bf16x2(f(acc.z), f(acc.w)));
        }
        __syncthreads();
        cluster_sync();  // no CTA leaves while another reads its part
    }
}

// Sums the parts of each (token, query head) row of a sequence, WPR warps a row: every lane has the weight
// of two parts (there are at most 64), each warp adds up every WPR-th.
template <int HD, int WPR>
__global__ void __launch_bounds__(128) attn_cache_join(const CacheArgs a, int *status)
{
    constexpr int V = HD / 32;
    __shared__ float rest[3][HD];  // sums of the row's warps but the first
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % WPR;
    grid_dep_wait();
    grid_dep_launch();
    CacheSeq sq;
    if (!load_seq(a, blockIdx.y, sq, status)) return;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * (4 / WPR) + warp / WPR;
    if (i >= static_cast<int64_t>(sq.len) * a.q_heads) return;  // whole rows
    const int64_t r = static_cast<int64_t>(sq.t0) * a.q_heads + i;
    RowPart p2[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        p2[h] = {-INFINITY, -INFINITY, 0.f};
        if (lane + 32 * h < a.splits) {
            const float4 p = *reinterpret_cast<const float4 *>(a.part_mn + (r * a.splits + lane + 32 * h) * 4);
            p2[h] = {p.x, p.y, p.z};
        }
    }
    RowPart sum{warp_max(fmaxf(p2[0].m, p2[1].m)), warp_max(fmaxf(p2[0].n, p2[1].n)), 0.f};
    float k[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        k[h] = part_weight(p2[h].m, sum.m);
        sum.l += p2[h].l * part_weight(p2[h].n, sum.n);
    }
    sum.l = warp_sum(sum.l);
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    const float *p = a.part_o + r * a.splits * HD + lane * V;
#pragma unroll 4
    for (int s = part; s < a.splits; s += WPR) {
        const float w = __shfl_sync(0xffffffffu, s < 32 ? k[0] : k[1], s & 31);
        float x[V];
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float2 f = *reinterpret_cast<const float2 *>(p + s * HD + i);
            x[i] = f.x, x[i + 1] = f.y;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(x[i], w, acc[i]);
    }
    if constexpr (WPR > 1) {
        if (part > 0)
#pragma unroll
            for (int i = 0; i < V; ++i) rest[part - 1][lane * V + i] = acc[i];
        __syncthreads();
        if (part > 0) return;
#pragma unroll
        for (int w = 0; w < WPR - 1; ++w)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += rest[w][lane * V + i];
    }
    const RowFactor f = row_factor(sum.m, sum.n, sum.l);
    __nv_bfloat16 *dst = a.out + r * HD + lane * V;
#pragma unroll
    for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t *>(dst + i) = pack_bf16x2(f(acc[i]), f(acc[i + 1]));
}

template <int HD>
cudaError_t launch_join(const CacheArgs &a, int *status, cudaStream_t s)
{
    const unsigned rows = static_cast<unsigned>(a.max_len) * a.q_heads;
    if (a.splits > 4) return launch_k(attn_cache_join<HD, 4>, dim3(rows, a.batch), dim3(128), 0, s, a, status);
    return launch_k(attn_cache_join<HD, 1>, dim3((rows + 3) / 4, a.batch), dim3(128), 0, s, a, status);
}

cudaError_t launch_join(const CacheArgs &a, int head_dim, int *status, cudaStream_t s)
{
    return head_dim == 64 ? launch_join<64>(a, status, s) : head_dim == 128 ? launch_join<128>(a, status, s) : launch_join<256>(a, status, s);
}

constexpr int kStreamRows = 32;    // rows of a key-value head up to which the streaming kernel runs at any size
constexpr int kStreamCtas = 2 * kSms;            // ... and with more rows up to so many CTAs, one part each, which
constexpr int64_t kStreamTokens = int64_t{1} << 18;  // read so many tokens together
constexpr int kClusterParts = 8;   // portable cluster size
constexpr int kMaxParts = 64;      // two a lane where they are joined
constexpr int kPartTokens = 128;   // a part has a run for each of four warps

// 8-row tiles of a CTA: 16 rows where the registers allow it and there are more than 8
int row_tile_count(int64_t rows, int head_dim) { return rows > 8 && head_dim < 256 ? 2 : 1; }

// Which kernel runs and into how many parts the sequences are split.  A matter of the arguments
// alone (a B200 has kSms multiprocessors), so that a workspace sized on one device serves on any.
struct CachePlan {
    bool tiles, cluster, wide;  // cluster: the parts are a cluster; wide: eight warps a CTA
    int splits;
    bool workspace() const { return splits > 1 && !cluster; }
};
CachePlan plan_attention_cache(int batch, int max_len, int max_kv, int q_heads, int kv_heads, int head_dim)
{
    const int64_t rows = static_cast<int64_t>(max_len) * (q_heads / kv_heads);
    const int per = 8 * row_tile_count(rows, head_dim);
    const int64_t ctas = std::max<int64_t>(1, (rows + per - 1) / per * batch * kv_heads);
    // The streaming kernel reads the cache once per 8 or 16 rows, the tiles once per 128 or 256, but a tile
    // CTA costs 7 to 25 us before its matrix products fill.  Streamed against tiles, heads 16 to 8 of 128:
    // 1 sequence of 4,000 tokens, 30 new ones, 19 and 27 us, 60 new ones (64 CTAs, 260,000 tokens) 25 and 29;
    // 8 of 500, 30 new ones (256 CTAs), 16 and 21; past the limits 4 of 4,000, 20 new ones, 40 and 34,
    // 16 prompts of 30 (512 CTAs) 14 and 11.
    CachePlan p{rows > kStreamRows && (ctas > kStreamCtas || ctas * max_kv > kStreamTokens), false, false, 1};
    if (p.tiles) {
        const int64_t tiles = (rows + attention_cache_tile_rows(head_dim) - 1) / attention_cache_tile_rows(head_dim);
        // one CTA an SM: split until they have one each, 512 tokens or more a part
        const int64_t want = std::min<int64_t>(kSms / std::max<int64_t>(1, tiles * batch * kv_heads), 65535 / tiles);
        p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, max_kv / 512, kMaxParts})));
        return p;
    }
    const int64_t resident = (head_dim == 128 && per == 16 ? 2 : 3) * kSms;  // what registers allow
    const int64_t room = std::min<int64_t>(resident / ctas, kClusterParts);
    if (room > 1 && max_kv <= 512 * room) {
        // As many parts as all fit at once, and those short; a power of two, since clusters of 3 or 6 leave SMs of
        // their group idle.  (Clusters that do not fit wait for room: 7 parts of 32 sequences x 8 heads
        // took 186 us as clusters and 158 with the second launch; 16 sequences of 500, 5 new tokens, 3 parts
        // for 2 CTAs an SM 21.8 us, 2 parts 12.8.  1 x 2,000 tokens 8.7 us, with the second launch 14.9.)
        while (2 * p.splits <= std::min<int64_t>(room, max_kv / kPartTokens)) p.splits *= 2;
        p.cluster = p.splits > 1;
    }
    if (p.splits == 1) {
        // Few CTAs: one round of the resident ones, 256 tokens or more a part.  1 x 16,000 tokens: 8 heads 16.7 us (8
        // parts in a cluster 21.5), 2 heads 12.8 (21.4), head_dim 256 and 1 head 16.5 (41.5).  Else about four
        // rounds, since sequences differ in length, of 1,024 tokens or more (a CTA costs 2.7 us beside its
        // reading).  32 sequences of 8,000 to 16,000 tokens, 8 heads: 2 rounds 159 us, 3 152, 4 150,
        // 6 152, 8 157; 16 of 8,000: parts of 512 tokens 67 us, of 1,024 62.
        const int64_t fill = resident / ctas;
        const int64_t want = fill >= 8 ? std::min(fill, max_kv / int64_t{256})
                                       : std::min((4 * resident + ctas - 1) / ctas, max_kv / int64_t{1024});
        p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, kMaxParts)));
    }
    // A CTA that has its SM to itself takes twice the warps; not in clusters that fill more than half of the
    // SMs, which would wait for eight of a group (2 x 2,000 tokens, 8 heads: 15.7 us, with four warps 10.4).
    p.wide = head_dim < 256 && ctas * p.splits <= (p.cluster ? kSms / 2 : kSms);
    return p;
}

template <int HD, int NR, int WARPS, bool CLUSTER>
cudaError_t stream(const CacheArgs &a, int *status, cudaStream_t s)
{
    using C = StreamCfg<HD, NR, WARPS>;
    auto kern = attn_cache_stream<HD, NR, WARPS, CLUSTER>;
    {
        static uint64_t configured[64] = {};  // context the attribute was set in
        int dev = 0;
        cudaGetDevice(&dev);
        const uint64_t ctx = current_context_id();
        if (dev >= 64 || configured[dev] != ctx) {
            cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
            if (e != cudaSuccess) return e;
            if (dev < 64) configured[dev] = ctx;
        }
    }
    const int row_tiles = (a.max_len * a.group + C::ROWS - 1) / C::ROWS;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = a.splits;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.batch) * row_tiles, a.kv_heads, a.splits);
    cfg.blockDim = dim3(32 * WARPS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = CLUSTER ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, row_tiles, status);
    return e != cudaSuccess || CLUSTER || a.splits == 1 ? e : launch_join<HD>(a, status, s);
}

template <int HD, int NR>
cudaError_t stream_as(const CacheArgs &a, const CachePlan &p, int *status, cudaStream_t s)
{
    if constexpr (HD < 256) {
        if (p.wide) return p.cluster ? stream<HD, NR, 8, true>(a, status, s) : stream<HD, NR, 8, false>(a, status, s);
    }
    return p.cluster ? stream<HD, NR, 4, true>(a, status, s) : stream<HD, NR, 4, false>(a, status, s);
}

template <int HD>
cudaError_t stream_any(const CacheArgs &a, const CachePlan &p, int *status, cudaStream_t s)
{
    if constexpr (HD < 256)
        if (row_tile_count(static_cast<int64_t>(a.max_len) * a.group, HD) == 2) return stream_as<HD, 2>(a, p, status, s);
    return stream_as<HD, 1>(a, p, status, s);
}

}  // namespace

size_t attention_cache_workspace_bytes(int batch, int max_len, int64_t total, int max_kv, int q_heads, int kv_heads,
                                       int head_dim)
{
    const CachePlan p = plan_attention_cache(batch, max_len, max_kv, q_heads, kv_heads, head_dim);
    return p.workspace() ? static_cast<size_t>(total) * q_heads * p.splits * (head_dim + 4) * sizeof(float) : 0;
}

cudaError_t launch_attention_cache_e4m3(const void *qkv, const int32_t *cu, int batch, int max_len, int64_t total,
                                        int q_heads, int kv_heads, int head_dim, const int32_t *past, int max_kv,
                                        const int32_t *table, int width, const void *k, const void *v, const float *ks,
                                        const float *vs, int pages, int page, bool causal, float scale, void *out,
                                        void *workspace, cudaStream_t s, fe_status *st)
{
    *st = FE_OK;
    CacheArgs a;
    a.qkv = static_cast<const __nv_bfloat16 *>(qkv);
    a.cu = cu, a.past = past, a.table = table;
    a.k = static_cast<const uint8_t *>(k), a.v = static_cast<const uint8_t *>(v);
    a.ks = ks, a.vs = vs;
    a.out = static_cast<__nv_bfloat16 *>(out);
    a.total = total;
    a.row = static_cast<int64_t>(q_heads + 2 * kv_heads) * head_dim;
    a.batch = batch, a.max_len = max_len, a.width = width, a.pages = pages;
    a.page_log2 = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
    a.q_heads = q_heads, a.kv_heads = kv_heads, a.group = q_heads / kv_heads, a.causal = causal;
    a.scale_log2 = scale * kLog2e;
    const CachePlan plan = plan_attention_cache(batch, max_len, max_kv, q_heads, kv_heads, head_dim);
    a.splits = plan.splits;
    a.part_o = static_cast<float *>(workspace);
    a.part_mn = a.part_o + total * q_heads * a.splits * head_dim;
    int *status = current_device_status_word();
    if (plan.tiles) {
        cudaError_t e = launch_attention_cache_tiles(a, head_dim, status, s, st);
        return e != cudaSuccess || *st != FE_OK || a.splits == 1 ? e : launch_join(a, head_dim, status, s);
    }
    if (head_dim == 64) return stream_any<64>(a, plan, status, s);
    if (head_dim == 128) return stream_any<128>(a, plan, status, s);
    return stream_any<256>(a, plan, status, s);
}

}  // namespace fe

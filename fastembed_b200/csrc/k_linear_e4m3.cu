// k_linear_e4m3.cu — tcgen05 linear layer on 8-bit operands:
//
//     y = epilogue(sx_i * sw_j * sum_k xq_ik wq_jk)
//
// with xq [m, k] and wq [n, k] e4m3 codes, one fp32 scale per row of x (token) and per row of
// w (output channel), FP32 accumulation in TMEM.  Both scales are constant along k, so they
// leave the sum: the mainloop multiplies bare codes (tcgen05.mma kind::f8f6f4, twice the bf16
// rate) and the epilogue applies sx_i * sw_j to the accumulator before bias / activation /
// residual / gating, in fp32, with one rounding where y is bf16.
//
// A k-block is 128 codes = one 128-byte swizzled row, so shared-memory stages, descriptors and
// TMA boxes have the bf16 linear layer's geometry with half as many k-blocks: the mainloop of a
// tile takes half as long while its epilogue costs the same, and below K = 2048 the epilogue
// decides.  Hence eight epilogue warps in the pair kernel.
//   linear_e4m3_pair  a cluster pair computes a 256 x 256 tile (cta_group::2); m >= 512.
//   linear_e4m3_cta   one CTA, 128 x BN tiles; BN shrinks (256, 128, 64) until there are as
//                     many tiles as SMs: few rows mean reading the weight, and that wants every
//                     SM's loads in flight.
// Warps: 0 TMA producer, 1 TMEM owner and MMA issuer (an elected lane), then the epilogue.
// Every mbarrier wait is bounded; on timeout the CTA records FE_ERR_DEVICE_TIMEOUT in the device
// status word, lets its own copies and MMAs land, frees its TMEM and exits.
#include <cuda.h>

#include <algorithm>

#include "fe_e4m3.cuh"
#include "fe_internal.h"

namespace fe {
namespace {

constexpr int BK = 128;  // codes per k-block: one 128-byte swizzled row
constexpr uint32_t kSlab = 32 * 128;  // one warp's 32-row x 128-byte store slab

enum Epi : int { E_NONE = 0, E_BIAS = 1, E_GELU = 2, E_RELU = 3, E_SWISH = 4, E_RESID = 5, E_SWIGLU = 6, E_GEGLU = 7 };

// Instruction descriptor of kind::f8f6f4 with e4m3 A and B (format 0), fp32 D, both K-major:
// [4,6) D format (1 = f32), [7,10) A format, [10,13) B format, [17,23) N >> 3, [24,29) M >> 4.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int M, int N)
{
    return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void umma_f8_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void umma_f8_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

struct EpiArgs {
    const float *sx;        // [M]
    const float *sw;        // [N]
    const float *bias;      // [N] or null
    const float *residual;  // [M, N] or null
    int epi;
};

// v[j] *= p[j] (or v[j] += p[j]) over W columns from col0, of which the last may lie past N
template <int W, bool MUL>
__device__ __forceinline__ void apply_cols(float (&v)[W], const float *__restrict__ p, int col0, int N)
{
    if (col0 + W <= N) {
#pragma unroll
        for (int j = 0; j < W; j += 4) {
            const float4 b = __ldg(reinterpret_cast<const float4 *>(p + col0 + j));
            if constexpr (MUL) {
                mul_f32x2(v[j], v[j + 1], b.x, b.y);
                mul_f32x2(v[j + 2], v[j + 3], b.z, b.w);
            } else {
                add_f32x2(v[j], v[j + 1], b.x, b.y);
                add_f32x2(v[j + 2], v[j + 3], b.z, b.w);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (col0 + j < N) v[j] = MUL ? v[j] * __ldg(p + col0 + j) : v[j] + __ldg(p + col0 + j);
    }
}

// 32 accumulator columns of this thread's row, scaled: acc * sx_i * sw_j
__device__ __forceinline__ void load_scaled(uint32_t taddr, float (&v)[32], const EpiArgs &ea, float sx, int col0, int N)
{
    uint32_t u[32];
    tmem_ld_x32(taddr, u);
    tmem_wait_ld_regs(u);
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        v[j] = __uint_as_float(u[j]);
        v[j + 1] = __uint_as_float(u[j + 1]);
        mul_f32x2(v[j], v[j + 1], sx, sx);
    }
    apply_cols<32, true>(v, ea.sw, col0, N);
}

__device__ __forceinline__ uint4 pack8(const float *f)
{
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// Drains COLS columns of one warp's 32 accumulator rows: 32-row x 128-byte slabs (two per
// warp) staged in 128B-swizzled shared memory and stored by TMA, which clips rows >= M and
// columns >= N.  `row` is this thread's output row, `store_row` the warp's first.
template <int COLS, bool OUT_BF16>
__device__ __forceinline__ void drain(uint32_t t_row, int row, int store_row, int n0, int M, int N, const EpiArgs &ea,
                                      float sx, const CUtensorMap *tm_y, uint8_t *bufs, int &pp, int lane)
{
    const int epi = ea.epi;
    constexpr int CHUNK = OUT_BF16 ? 64 : 32;  // y columns per slab
    const bool glu = OUT_BF16 && COLS >= 128 && epi >= E_SWIGLU;
    const int step = glu ? 2 * CHUNK : CHUNK;  // accumulator columns per slab
#pragma unroll 1
    for (int c = 0; c < COLS; c += step) {
        float f[CHUNK];
        if constexpr (OUT_BF16) {
#pragma unroll
            for (int hb = 0; hb < 2; ++hb) {
                float v[32];
                if (glu) {  // 32 gate columns, then their 32 inputs
                    float u[32];
                    const int a = c + 64 * hb;
                    load_scaled(t_row + a, v, ea, sx, n0 + a, N);
                    load_scaled(t_row + a + 32, u, ea, sx, n0 + a + 32, N);
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        if (epi == E_SWIGLU) silu_fast2(v[j], v[j + 1]);
                        else gelu_tanh_fast2(v[j], v[j + 1]);
                        mul_f32x2(v[j], v[j + 1], u[j], u[j + 1]);
                    }
                } else {
                    const int col0 = n0 + c + 32 * hb;
                    load_scaled(t_row + c + 32 * hb, v, ea, sx, col0, N);
                    if (epi != E_NONE) apply_cols<32, false>(v, ea.bias, col0, N);
                    if (epi == E_GELU) {
#pragma unroll
                        for (int j = 0; j < 32; j += 2) gelu_tanh_fast2(v[j], v[j + 1]);
                    } else if (epi == E_SWISH) {
#pragma unroll
                        for (int j = 0; j < 32; j += 2) silu_fast2(v[j], v[j + 1]);
                    } else if (epi == E_RELU) {  // as a comparison: NaN stays NaN
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];
                    }
                }
#pragma unroll
                for (int j = 0; j < 32; ++j) f[32 * hb + j] = v[j];
            }
        } else {
            const int col0 = n0 + c;
            load_scaled(t_row + c, f, ea, sx, col0, N);
            if (epi != E_NONE) apply_cols<32, false>(f, ea.bias, col0, N);
            if (epi == E_RESID && row < M) {
                const float *rp = ea.residual + static_cast<size_t>(row) * N;
                apply_cols<32, false>(f, rp, col0, N);
            }
        }
        uint8_t *buf = bufs + pp * kSlab;
        if (lane == 0) bulk_wait_read<1>();  // the store that last used `buf` has read it
        __syncwarp();
        uint8_t *rowp = buf + lane * 128;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            uint4 w;
            if constexpr (OUT_BF16) w = pack8(f + 8 * u);
            else w = make_uint4(__float_as_uint(f[4 * u]), __float_as_uint(f[4 * u + 1]), __float_as_uint(f[4 * u + 2]),
                                __float_as_uint(f[4 * u + 3]));
            *reinterpret_cast<uint4 *>(rowp + ((u ^ (lane & 7)) << 4)) = w;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(tm_y, buf, glu ? (n0 + c) / 2 : n0 + c, store_row);
            bulk_commit();
        }
        pp ^= 1;
    }
}

// ------------------------------------------------------------------ one CTA
template <int BN>
struct CtaCfg {
    static constexpr int EPI_WARPS = 4;
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr uint32_t A_BYTES = 128 * BK;
    static constexpr uint32_t B_BYTES = BN * BK;
    static constexpr uint32_t STAGE = A_BYTES + B_BYTES;
    static constexpr uint32_t RING = STAGES * STAGE;
    static constexpr uint32_t EPI = EPI_WARPS * 2 * kSlab;
    static constexpr uint32_t SMEM = 1024 + RING + EPI + 256;
    static constexpr uint32_t TMEM_COLS = 2 * BN;
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

template <int BN, bool OUT_BF16>
__global__ void __launch_bounds__(CtaCfg<BN>::THREADS, 1)
    linear_e4m3_cta(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                    const __grid_constant__ CUtensorMap tm_y, int M, int N, int K, const EpiArgs ea, int *status)
{
    using C = CtaCfg<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = smem;
    uint8_t *epi_buf = smem + C::RING;
    uint64_t *full = reinterpret_cast<uint64_t *>(epi_buf + C::EPI);
    uint64_t *empty = full + C::STAGES;
    uint64_t *acc_full = empty + C::STAGES;  // [2]
    uint64_t *acc_empty = acc_full + 2;      // [2]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int n_tiles = (N + BN - 1) / BN;
    const int num_tiles = (M + 127) / 128 * n_tiles;
    const int k_iters = (K + BK - 1) / BK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], C::EPI_WARPS);
        }
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tm_x);
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_y);
    }
    grid_dep_wait();
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dep_launch();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0, armed = 0, armed_parity = 0;  // per stage: armed at least once / parity of the last arm
            for (int tile = blockIdx.x; tile < num_tiles && !*abort_flag; tile += gridDim.x) {
                const int m0 = tile / n_tiles * 128, n0 = tile % n_tiles * BN;
                for (int kb = 0; kb < k_iters; ++kb) {
                    if (!mbar_wait(&empty[stage], phase ^ 1)) {
                        report(status, DEV_TIMEOUT);
                        *abort_flag = 1;
                        break;
                    }
                    uint8_t *a_dst = ring + stage * C::STAGE;
                    mbar_arrive_expect_tx(&full[stage], C::STAGE);
                    tma_load_2d(a_dst, &tm_x, &full[stage], kb * BK, m0);
                    tma_load_2d(a_dst + C::A_BYTES, &tm_w, &full[stage], kb * BK, n0);
                    armed |= 1u << stage;
                    armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            for (int s = 0; s < C::STAGES; ++s)  // every load this thread started lands before the CTA exits
                if (armed & (1u << s))
                    if (!mbar_wait_drain(&full[s], (armed_parity >> s) & 1u)) report(status, DEV_TIMEOUT);
        }
    } else if (warp == 1) {
        const bool leader = elect_lane();  // the whole warp waits; this lane issues
        constexpr uint32_t idesc = idesc_e4m3_f32(128, BN);
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool issued = false;
        for (int tile = blockIdx.x; tile < num_tiles && !*abort_flag; tile += gridDim.x) {
            if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1)) {
                report(status, DEV_TIMEOUT);
                *abort_flag = 1;
                break;
            }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + acc * BN;
            for (int kb = 0; kb < k_iters; ++kb) {
                if (!mbar_wait(&full[stage], phase)) {
                    report(status, DEV_TIMEOUT);
                    *abort_flag = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t a_addr = smem_u32(ring + stage * C::STAGE);
                const uint64_t ad = sdesc_sw128(a_addr, 16, 1024), bd = sdesc_sw128(a_addr + C::A_BYTES, 16, 1024);
#pragma unroll
                for (int k = 0; k < BK / 32; ++k)  // +32 bytes per K step inside the swizzle atom
                    if (leader) umma_f8_ss(d_tmem, ad + 2 * k, bd + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
                issued = true;
                if (leader) umma_commit(&empty[stage]);
                if (++stage == C::STAGES) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (*abort_flag) break;
            if (leader) umma_commit(&acc_full[acc]);
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1;
        }
        if (*abort_flag && issued) {  // outstanding MMAs retire before TMEM is released
            if (leader) umma_commit(&acc_full[acc]);
            if (!mbar_wait_drain(&acc_full[acc], acc_phase)) report(status, DEV_TIMEOUT);
        }
    } else {
        const int q = warp & 3;  // TMEM lane quarter this warp may access
        uint8_t *bufs = epi_buf + q * 2 * kSlab;
        int acc = 0, pp = 0;
        uint32_t acc_phase = 0;
        for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x) {
            if (*abort_flag) break;
            const int m0 = tile / n_tiles * 128, n0 = tile % n_tiles * BN;
            const int row = m0 + q * 32 + lane;
            const float sx = row < M ? __ldg(ea.sx + row) : 0.f;  // overlaps the wait for the accumulator
            if (!mbar_wait(&acc_full[acc], acc_phase)) {
                report(status, DEV_TIMEOUT);
                *abort_flag = 1;
                break;
            }
            tc_fence_after();
            if (m0 + q * 32 < M)  // a warp whose rows all lie past M has nothing to store
                drain<BN, OUT_BF16>(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN, row, m0 + q * 32, n0, M, N,
                                    ea, sx, &tm_y, bufs, pp, lane);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[acc]);
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1;
        }
        if (lane == 0) bulk_wait_all<0>();
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
}

// ------------------------------------------------------------------ CTA pair
// The leader (cluster rank 0) issues M = 256 MMAs over both CTAs' stages: each CTA stages its
// own 128 rows of x and of w.  Both CTAs' loads complete on the leader's stage barrier, commits
// are multicast to both CTAs' barriers, and each epilogue warp reports back to the leader.
struct PairCfg {
    static constexpr int STAGES = 5;
    static constexpr int EPI_WARPS = 8;  // two per TMEM lane quarter, 128 columns each
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static constexpr int BN = 256;
    static constexpr int COLS = BN / (EPI_WARPS / 4);
    static constexpr uint32_t HALF = 128 * BK;     // 16 KB: 128 rows
    static constexpr uint32_t STAGE = 2 * HALF;    // this CTA's x rows + w rows
    static constexpr uint32_t RING = STAGES * STAGE;
    static constexpr uint32_t EPI = EPI_WARPS * 2 * kSlab;
    static constexpr uint32_t SMEM = 1024 + RING + EPI + 256;
    static constexpr uint32_t TMEM_COLS = 2 * BN;
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

template <bool OUT_BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg::THREADS, 1)
    linear_e4m3_pair(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_y, int M, int N, int K, const EpiArgs ea, int *status)
{
    using C = PairCfg;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = smem;
    uint8_t *epi_buf = smem + C::RING;
    uint64_t *full = reinterpret_cast<uint64_t *>(epi_buf + C::EPI);  // used in the leader
    uint64_t *empty = full + C::STAGES;                               // both CTAs
    uint64_t *acc_full = empty + C::STAGES;                           // both CTAs [2]
    uint64_t *acc_empty = acc_full + 2;                               // used in the leader [2]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1;
    const int npairs = gridDim.x >> 1;
    const int n_tiles = (N + C::BN - 1) / C::BN;
    const int num_tiles = (M + 255) / 256 * n_tiles;
    const int k_iters = (K + BK - 1) / BK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 2 * C::EPI_WARPS);  // one arrival per epilogue warp of either CTA
        }
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tm_x);
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_y);
    }
    grid_dep_wait();
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, C::TMEM_COLS);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers exist before any cross-CTA signal
    tc_fence_after();
    grid_dep_launch();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0, armed = 0, armed_parity = 0;
            for (int tile = pair; tile < num_tiles && !*abort_flag; tile += npairs) {
                const int m0 = tile / n_tiles * 256 + static_cast<int>(rank) * 128;
                const int n0 = tile % n_tiles * C::BN + static_cast<int>(rank) * 128;
                for (int kb = 0; kb < k_iters; ++kb) {
                    if (!mbar_wait(&empty[stage], phase ^ 1)) {
                        report(status, DEV_TIMEOUT);
                        *abort_flag = 1;
                        break;
                    }
                    uint8_t *a_dst = ring + stage * C::STAGE;
                    const uint32_t leader_full = map_to_rank(&full[stage], 0);
                    if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * C::STAGE);
                    tma_load_2d_pair(a_dst, &tm_x, leader_full, kb * BK, m0);
                    tma_load_2d_pair(a_dst + C::HALF, &tm_w, leader_full, kb * BK, n0);
                    armed |= 1u << stage;
                    armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // The leader's stage barriers count both CTAs' bytes: it drains the pair's loads.
            if (rank == 0)
                for (int s = 0; s < C::STAGES; ++s)
                    if (armed & (1u << s))
                        if (!mbar_wait_drain(&full[s], (armed_parity >> s) & 1u)) report(status, DEV_TIMEOUT);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const bool leader = elect_lane();
            constexpr uint32_t idesc = idesc_e4m3_f32(256, C::BN);
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool issued = false;
            for (int tile = pair; tile < num_tiles && !*abort_flag; tile += npairs) {
                if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1)) {
                    report(status, DEV_TIMEOUT);
                    *abort_flag = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * C::BN;
                for (int kb = 0; kb < k_iters; ++kb) {
                    if (!mbar_wait(&full[stage], phase)) {
                        report(status, DEV_TIMEOUT);
                        *abort_flag = 1;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(ring + stage * C::STAGE);
                    const uint64_t ad = sdesc_sw128(a_addr, 16, 1024), bd = sdesc_sw128(a_addr + C::HALF, 16, 1024);
#pragma unroll
                    for (int k = 0; k < BK / 32; ++k)
                        if (leader) umma_f8_ss_pair(d_tmem, ad + 2 * k, bd + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
                    issued = true;
                    if (leader) umma_commit_pair_both(&empty[stage]);
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (*abort_flag) break;
                if (leader) umma_commit_pair_both(&acc_full[acc]);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
            }
            if (*abort_flag && issued) {
                if (leader) umma_commit_pair_both(&acc_full[acc]);
                if (!mbar_wait_drain(&acc_full[acc], acc_phase)) report(status, DEV_TIMEOUT);
            }
        }
    } else {
        const int q = warp & 3;            // TMEM lane quarter
        const int h = (warp - 2) >> 2;     // column half
        uint8_t *bufs = epi_buf + (warp - 2) * 2 * kSlab;
        const uint32_t leader_acc_empty[2] = {map_to_rank(&acc_empty[0], 0), map_to_rank(&acc_empty[1], 0)};
        int acc = 0, pp = 0;
        uint32_t acc_phase = 0;
        for (int tile = pair; tile < num_tiles; tile += npairs) {
            if (*abort_flag) break;
            const int m0 = tile / n_tiles * 256 + static_cast<int>(rank) * 128;
            const int n0 = tile % n_tiles * C::BN + h * C::COLS;
            const int row = m0 + q * 32 + lane;
            const float sx = row < M ? __ldg(ea.sx + row) : 0.f;
            if (!mbar_wait(&acc_full[acc], acc_phase)) {
                report(status, DEV_TIMEOUT);
                *abort_flag = 1;
                break;
            }
            tc_fence_after();
            if (m0 + q * 32 < M && n0 < N)
                drain<C::COLS, OUT_BF16>(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * C::BN + h * C::COLS, row,
                                         m0 + q * 32, n0, M, N, ea, sx, &tm_y, bufs, pp, lane);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(leader_acc_empty[acc]);
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1;
        }
        if (lane == 0) bulk_wait_all<0>();
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();  // no CTA leaves while its peer may still signal it or read its smem
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
    }
}

// Sets a kernel's shared-memory size once per device and context.
template <class Kern>
cudaError_t allow_smem(Kern kern, uint32_t bytes, uint64_t (&configured)[64])
{
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t ctx = current_context_id();
    if (dev < 64 && configured[dev] == ctx) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e == cudaSuccess && dev < 64) configured[dev] = ctx;
    return e;
}

struct Maps {
    CUtensorMap x, w, y;
};

template <int BN, bool OUT_BF16>
cudaError_t launch_cta(const Maps &t, int M, int N, int K, const EpiArgs &ea, cudaStream_t s)
{
    using C = CtaCfg<BN>;
    static uint64_t configured[64] = {};
    cudaError_t e = allow_smem(linear_e4m3_cta<BN, OUT_BF16>, C::SMEM, configured);
    if (e != cudaSuccess) return e;
    const int tiles = (M + 127) / 128 * ((N + BN - 1) / BN);
    return launch_k(linear_e4m3_cta<BN, OUT_BF16>, dim3(std::min(current_sm_count(), tiles)), dim3(C::THREADS), C::SMEM, s,
                    t.x, t.w, t.y, M, N, K, ea, current_device_status_word());
}

template <bool OUT_BF16>
cudaError_t launch_pair(const Maps &t, int M, int N, int K, const EpiArgs &ea, cudaStream_t s)
{
    using C = PairCfg;
    static uint64_t configured[64] = {};
    cudaError_t e = allow_smem(linear_e4m3_pair<OUT_BF16>, C::SMEM, configured);
    if (e != cudaSuccess) return e;
    const int tiles = (M + 255) / 256 * ((N + C::BN - 1) / C::BN);
    const int pairs = std::max(1, std::min(current_sm_count() / 2, tiles));
    return launch_k(linear_e4m3_pair<OUT_BF16>, dim3(2 * pairs), dim3(C::THREADS), C::SMEM, s, t.x, t.w, t.y, M, N, K, ea,
                    current_device_status_word());
}

}  // namespace

cudaError_t launch_linear_e4m3(const void *x, const float *sx, const void *w, const float *sw, const float *bias,
                               const float *residual, void *y, int64_t m, int64_t n, int64_t k, int epilogue, int y_dtype,
                               cudaStream_t s, fe_status *st)
{
    *st = FE_OK;
    const bool bf16 = y_dtype == FE_DTYPE_BF16;
    const bool glu = epilogue == E_SWIGLU || epilogue == E_GEGLU;
    const int64_t ny = glu ? n / 2 : n;
    const int sms = current_sm_count();
    auto tiles = [&](int64_t bn) { return (m + 127) / 128 * ((n + bn - 1) / bn); };
    const bool pair = m >= 512 && n >= 256;
    // the gated epilogues pair 32 gate with 32 input columns and fill a slab from 128
    const int bn = pair ? 128 : n > 128 && tiles(256) >= sms ? 256 : glu || tiles(128) >= sms ? 128 : 64;
    Maps t;
    fe_status r = make_tmap_2d(&t.x, x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, m, k, k, 128, BK);
    if (r == FE_OK) r = make_tmap_2d(&t.w, w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, n, k, k, bn, BK);
    if (r == FE_OK)
        r = bf16 ? make_tmap_2d(&t.y, y, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, m, ny, ny, 32, 64)
                 : make_tmap_2d(&t.y, y, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, m, n, n, 32, 32);
    if (r != FE_OK) {
        *st = r;
        return cudaSuccess;
    }
    const EpiArgs ea{sx, sw, bias, residual, epilogue};
    const int M = static_cast<int>(m), N = static_cast<int>(n), K = static_cast<int>(k);
    if (pair) return bf16 ? launch_pair<true>(t, M, N, K, ea, s) : launch_pair<false>(t, M, N, K, ea, s);
    if (bn == 256) return bf16 ? launch_cta<256, true>(t, M, N, K, ea, s) : launch_cta<256, false>(t, M, N, K, ea, s);
    if (bn == 128) return bf16 ? launch_cta<128, true>(t, M, N, K, ea, s) : launch_cta<128, false>(t, M, N, K, ea, s);
    return bf16 ? launch_cta<64, true>(t, M, N, K, ea, s) : launch_cta<64, false>(t, M, N, K, ea, s);
}

cudaError_t set_wait_limit_linear_e4m3(uint64_t ns) { return set_wait_limit_this_file(ns); }

}  // namespace fe

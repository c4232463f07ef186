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
//   linear_e4m3_pair  a cluster pair computes a 256 x 256 tile (cta_group::2); calls of more than
//                     a round of the SMs' tiles.
//   linear_e4m3_cta   one CTA, 128 x BN tiles; few rows mean reading the weight, and that wants
//                     many SMs' loads in flight, so BN is the smallest of 64, 128 and 256 that is one round
//                     of them (at 64 columns 4,096 channels are 64 SMs).
// K is never split: a row's result has the same bits in whatever batch, and so kernel, it comes.
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

// Commit of the pair's MMAs arriving at the leader (rank 0) alone.
__device__ __forceinline__ void umma_commit_pair_leader(uint64_t *bar)
{
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(1))
        : "memory");
}

// A whole warp's wait: its lanes go on, or give up, together.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

// A warp leaves its loop as one, whichever of its lanes read the flag before it was set
__device__ __forceinline__ bool given_up(const volatile int *flag) { return __any_sync(0xffffffffu, *flag != 0); }

struct EpiArgs {
    const float *sx;        // [M]
    const float *sw;        // [N]
    const float *bias;      // [N]; null for the epilogues without one
    int epi;
};

// A warp's columns' scales and biases, for the tile at hand, in its own shared memory: every lane
// needs every column's (lane = row).  Taken before the wait for the accumulator.
template <int COLS>
__device__ __forceinline__ void stage_cols(float *cols, const float *__restrict__ sw, const float *__restrict__ bias, int n0,
                                           int N, int lane)
{
    __syncwarp();  // the previous tile's have been read
    float s[COLS / 32], b[COLS / 32];
#pragma unroll
    for (int i = 0; i < COLS / 32; ++i) {
        const int col = n0 + 32 * i + lane;
        s[i] = col < N ? __ldg(sw + col) : 0.f;
        b[i] = col < N && bias != nullptr ? __ldg(bias + col) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < COLS / 32; ++i) {
        cols[32 * i + lane] = s[i];
        cols[COLS + 32 * i + lane] = b[i];
    }
    __syncwarp();
}

// The accumulator's columns go back to the issuer, maybe in the other CTA.  What the arrival hands
// over has been read into registers before (tcgen05.wait::ld), so it need not wait, as a release to the
// cluster does, for this thread's stores: 26,508 x 4,096 x 1,024 with gelu 120 us, with release 132.
__device__ __forceinline__ void arrive_acc_empty(uint32_t cluster_addr)
{
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// z_j = acc_j * (sx_i sw_j) + b_j for 32 accumulator columns, sw and b in shared memory
__device__ __forceinline__ void scale_bias(float (&z)[32], const uint32_t (&u)[32], float sx, const float *sw, const float *b)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float4 s = *reinterpret_cast<const float4 *>(sw + 4 * j);
        const float4 c = *reinterpret_cast<const float4 *>(b + 4 * j);
        mul_f32x2(s.x, s.y, sx, sx);
        mul_f32x2(s.z, s.w, sx, sx);
        fma_f32x2v(z[4 * j], z[4 * j + 1], __uint_as_float(u[4 * j]), __uint_as_float(u[4 * j + 1]), s.x, s.y, c.x, c.y);
        fma_f32x2v(z[4 * j + 2], z[4 * j + 3], __uint_as_float(u[4 * j + 2]), __uint_as_float(u[4 * j + 3]), s.z, s.w, c.z,
                   c.w);
    }
}

__device__ __forceinline__ void activate(float (&z)[32], int epi)
{
    if (epi == E_GELU) {
#pragma unroll
        for (int j = 0; j < 32; j += 2) gelu_tanh_fast2(z[j], z[j + 1]);
    } else if (epi == E_SWISH) {
#pragma unroll
        for (int j = 0; j < 32; j += 2) silu_fast2(z[j], z[j + 1]);
    } else if (epi == E_RELU) {  // as a comparison: NaN stays NaN
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] = z[j] < 0.f ? 0.f : z[j];
    }
}

__device__ __forceinline__ uint4 pack8(const float *f)
{
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// 32 finished columns of this thread's row into its slab row: 16-byte chunks from `first` on
template <bool OUT_BF16>
__device__ __forceinline__ void to_slab(uint8_t *slab, const float (&z)[32], int first, int lane)
{
    uint8_t *rowp = slab + lane * 128;
#pragma unroll
    for (int u = 0; u < (OUT_BF16 ? 4 : 8); ++u) {
        uint4 w;
        if constexpr (OUT_BF16) w = pack8(z + 8 * u);
        else w = make_uint4(__float_as_uint(z[4 * u]), __float_as_uint(z[4 * u + 1]), __float_as_uint(z[4 * u + 2]),
                            __float_as_uint(z[4 * u + 3]));
        *reinterpret_cast<uint4 *>(rowp + (((first + u) ^ (lane & 7)) << 4)) = w;
    }
}

// What an epilogue warp carries from tile to tile: its two 32-row x 128-byte slabs (128B-swizzled),
// its columns' vectors and, for the residual, a barrier each whose phase is the parity bit of `phase`.
struct Slabs {
    uint8_t *buf;
    uint64_t *bar;
    float *cols;  // scales, then biases, of the tile's columns
    uint32_t phase, armed;
    int pp;
};

__device__ __forceinline__ void store_slab(const CUtensorMap *tm_y, Slabs &sl, int x, int y, int lane)
{
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
        tma_store_2d(tm_y, sl.buf + sl.pp * kSlab, x, y);
        bulk_commit();
    }
    sl.pp ^= 1;
}

// Drains COLS columns of one warp's 32 accumulator rows; rows >= M and columns >= N are clipped
// by the tensor map.  The next 32 columns' TMEM load is in flight during the arithmetic of these.
// At K = 1024 this bounds the kernel: 26,508 x 4,096 with gelu takes 108 us (121 in a long run, under the
// power cap), 73 of it without draining; with the column vectors read from global memory where they
// are used 8 us more.
template <int COLS, bool OUT_BF16>
__device__ __forceinline__ void drain(uint32_t t_row, int store_row, int n0, int N, const EpiArgs &ea, float sx,
                                      const CUtensorMap *tm_y, Slabs &sl, int lane)
{
    const int epi = ea.epi;
    uint32_t u[2][32];
    tmem_ld_x32(t_row, u[0]);
#pragma unroll 4
    for (int c = 0; c < COLS; c += 32) {
        uint32_t(&v)[32] = u[(c >> 5) & 1];
        tmem_wait_ld_regs(v);
        if (c + 32 < COLS) tmem_ld_x32(t_row + c + 32, u[((c >> 5) & 1) ^ 1]);
        float z[32];
        scale_bias(z, v, sx, sl.cols + c, sl.cols + COLS + c);
        if constexpr (OUT_BF16) activate(z, epi);
        const bool begins = !OUT_BF16 || (c & 32) == 0, ends = !OUT_BF16 || (c & 32) != 0;
        if (begins) {
            if (lane == 0) bulk_wait_read<1>();  // the store that last used the slab has read it
            __syncwarp();
        }
        to_slab<OUT_BF16>(sl.buf + sl.pp * kSlab, z, OUT_BF16 ? (c & 32) / 8 : 0, lane);
        if (ends) store_slab(tm_y, sl, n0 + (OUT_BF16 ? c & ~63 : c), store_row, lane);
    }
}

// Gated epilogues: 32 gate columns, then their 32 inputs; 128 accumulator columns fill a slab.
template <int COLS>
__device__ __forceinline__ void drain_glu(uint32_t t_row, int store_row, int n0, int N, const EpiArgs &ea, float sx,
                                          const CUtensorMap *tm_y, Slabs &sl, int lane)
{
    uint32_t g[32], u[32];
    tmem_ld_x32(t_row, g);
    tmem_ld_x32(t_row + 32, u);
#pragma unroll 2
    for (int c = 0; c < COLS; c += 64) {
        tmem_wait_ld_regs(g);
        tmem_wait_ld_regs(u);
        float a[32], b[32];
        scale_bias(a, g, sx, sl.cols + c, sl.cols + COLS + c);  // no bias: zeros
        scale_bias(b, u, sx, sl.cols + c + 32, sl.cols + COLS + c + 32);
        if (c + 64 < COLS) {
            tmem_ld_x32(t_row + c + 64, g);
            tmem_ld_x32(t_row + c + 96, u);
        }
        activate(a, ea.epi == E_SWIGLU ? E_SWISH : E_GELU);
#pragma unroll
        for (int j = 0; j < 32; j += 2) mul_f32x2(a[j], a[j + 1], b[j], b[j + 1]);
        if ((c & 64) == 0) {
            if (lane == 0) bulk_wait_read<1>();
            __syncwarp();
        }
        to_slab<true>(sl.buf + sl.pp * kSlab, a, (c & 64) / 16, lane);
        if ((c & 64) != 0) store_slab(tm_y, sl, (n0 + c - 64) / 2, store_row, lane);
    }
}

// The residual's first two 32-column chunks of a tile into the two slabs, once their last
// stores have read them: called before the wait for the accumulator.
__device__ __forceinline__ void load_residual(const CUtensorMap *tm_r, Slabs &sl, int slab, int x, int y, int lane)
{
    if (lane == 0) {
        mbar_arrive_expect_tx(&sl.bar[slab], kSlab);
        tma_load_2d(sl.buf + slab * kSlab, tm_r, &sl.bar[slab], x, y);
    }
    sl.armed |= 1u << slab;
}

template <int COLS>
__device__ __forceinline__ void start_residual(const CUtensorMap *tm_r, Slabs &sl, int n0, int store_row, int lane)
{
    if (lane == 0) bulk_wait_read<0>();
    __syncwarp();
    sl.pp = 0;
    load_residual(tm_r, sl, 0, n0, store_row, lane);
    load_residual(tm_r, sl, 1, n0 + 32, store_row, lane);
    // the rest on their way to L2
    if (lane == 0)
        for (int c = 64; c < COLS; c += 32) tma_prefetch_l2_2d(tm_r, n0 + c, store_row);
}

// y = acc sx sw + b + residual in fp32: the residual arrives in the slab that the result leaves
// from (read by rows it would be 16 bytes of a different line per lane).  False on a timeout.
template <int COLS>
__device__ __forceinline__ bool drain_residual(uint32_t t_row, int store_row, int n0, int N, const EpiArgs &ea, float sx,
                                               const CUtensorMap *tm_y, const CUtensorMap *tm_r, Slabs &sl, int lane)
{
    uint32_t u[2][32];
    tmem_ld_x32(t_row, u[0]);
#pragma unroll 2
    for (int c = 0; c < COLS; c += 32) {
        uint32_t(&v)[32] = u[(c >> 5) & 1];
        tmem_wait_ld_regs(v);
        if (c + 32 < COLS) tmem_ld_x32(t_row + c + 32, u[((c >> 5) & 1) ^ 1]);
        float z[32];
        scale_bias(z, v, sx, sl.cols + c, sl.cols + COLS + c);
        const int slab = sl.pp;
        if (!warp_wait(&sl.bar[slab], (sl.phase >> slab) & 1u)) {
            tmem_wait_ld();
            return false;
        }
        sl.phase ^= 1u << slab;
        sl.armed &= ~(1u << slab);
        const uint8_t *rowp = sl.buf + slab * kSlab + lane * 128;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float4 r = *reinterpret_cast<const float4 *>(rowp + ((k ^ (lane & 7)) << 4));
            add_f32x2(z[4 * k], z[4 * k + 1], r.x, r.y);
            add_f32x2(z[4 * k + 2], z[4 * k + 3], r.z, r.w);
        }
        to_slab<false>(sl.buf + slab * kSlab, z, 0, lane);
        store_slab(tm_y, sl, n0 + c, store_row, lane);
        if (c + 64 < COLS) {
            if (lane == 0) bulk_wait_read<0>();  // this chunk's store has read the slab
            __syncwarp();
            load_residual(tm_r, sl, slab, n0 + c + 64, store_row, lane);
        }
    }
    return true;
}

// One tile of an epilogue warp, from the wait for its accumulator on.
template <int COLS, bool OUT_BF16>
__device__ __forceinline__ bool finish_tile(uint64_t *acc_full, uint32_t parity, uint32_t t_row, int row, int store_row, int n0,
                                            int M, int N, const EpiArgs &ea, const CUtensorMap *tm_y, const CUtensorMap *tm_r,
                                            Slabs &sl, int lane)
{
    const float sx = row < M ? __ldg(ea.sx + row) : 0.f;  // these loads overlap the wait for the accumulator
    const bool any = store_row < M && n0 < N;             // else nothing to store
    if (any) stage_cols<COLS>(sl.cols, ea.sw, ea.bias, n0, N, lane);
    if constexpr (!OUT_BF16)
        if (ea.epi == E_RESID && any) start_residual<COLS>(tm_r, sl, n0, store_row, lane);
    if (!warp_wait(acc_full, parity)) return false;
    tc_fence_after();
    if (!any) return true;
    if constexpr (OUT_BF16) {
        if constexpr (COLS >= 128)
            if (ea.epi >= E_SWIGLU) {
                drain_glu<COLS>(t_row, store_row, n0, N, ea, sx, tm_y, sl, lane);
                return true;
            }
    } else {
        if (ea.epi == E_RESID) return drain_residual<COLS>(t_row, store_row, n0, N, ea, sx, tm_y, tm_r, sl, lane);
    }
    drain<COLS, OUT_BF16>(t_row, store_row, n0, N, ea, sx, tm_y, sl, lane);
    return true;
}

// Before a warp leaves: residual loads still in flight land, stores complete.
__device__ __forceinline__ void leave(Slabs &sl, int *status, int lane)
{
    for (int i = 0; i < 2; ++i)
        if ((sl.armed >> i) & 1u)
            if (!mbar_wait_drain(&sl.bar[i], (sl.phase >> i) & 1u)) report(status, DEV_TIMEOUT);
    if (lane == 0) bulk_wait_all<0>();
    __syncwarp();
}

// ------------------------------------------------------------------ one CTA
// Rows of x that a tile loads: of a single one only those there are (in eights); the MMA multiplies
// whatever lies behind them, into rows that are not stored.  8 x 4,096 x 4,096 takes 8.9 us, with all
// 128 rows loaded, most of them zeros from outside the tensor, 11.8.
__host__ __device__ __forceinline__ int x_rows(int M) { return M < 128 ? (M + 7) & ~7 : 128; }

template <int BN>
struct CtaCfg {
    static constexpr int EPI_WARPS = 4;
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static constexpr int STAGES = BN == 128 ? 5 : 3;
    // Blocks of BK a stage.  One wait, commit and release each take longer than a block's four MMAs at 64
    // columns: 8 x 1,024 x 4,096 takes 8.6 us with two blocks a stage, 9.6 with one (and seven stages).
    static constexpr int GROUP = BN == 64 ? 2 : 1;
    static constexpr uint32_t A_BYTES = 128 * BK;
    static constexpr uint32_t B_BYTES = BN * BK;
    static constexpr uint32_t BLOCK = A_BYTES + B_BYTES;
    static constexpr uint32_t STAGE = GROUP * BLOCK;
    static constexpr uint32_t RING = STAGES * STAGE;
    static constexpr uint32_t EPI = EPI_WARPS * 2 * kSlab;
    static constexpr uint32_t COLV = EPI_WARPS * 2 * BN * 4;  // column vectors
    static constexpr uint32_t SMEM = 1024 + RING + EPI + COLV + 384;
    static constexpr uint32_t TMEM_COLS = 2 * BN;
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

template <int BN, bool OUT_BF16>
__global__ void __launch_bounds__(CtaCfg<BN>::THREADS, 1)
    linear_e4m3_cta(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                    const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_r, int M, int N, int K,
                    const EpiArgs ea, int *status)
{
    using C = CtaCfg<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = smem;
    uint8_t *epi_buf = smem + C::RING;
    float *colv = reinterpret_cast<float *>(epi_buf + C::EPI);
    uint64_t *full = reinterpret_cast<uint64_t *>(epi_buf + C::EPI + C::COLV);
    uint64_t *empty = full + C::STAGES;
    uint64_t *acc_full = empty + C::STAGES;  // [2]
    uint64_t *acc_empty = acc_full + 2;      // [2]
    uint64_t *res_bar = acc_empty + 2;       // [EPI_WARPS][2]
    uint64_t *probe = res_bar + 2 * C::EPI_WARPS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(probe + 1);
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
        for (int b = 0; b < 2 * C::EPI_WARPS; ++b) mbar_init(&res_bar[b], 1);
        mbar_init(probe, 1);
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
                for (int kb = 0; kb < k_iters; kb += C::GROUP) {
                    if (!mbar_wait(&empty[stage], phase ^ 1)) {
                        report(status, DEV_TIMEOUT);
                        *abort_flag = 1;
                        break;
                    }
                    const int blocks = min(C::GROUP, k_iters - kb);
                    mbar_arrive_expect_tx(&full[stage], blocks * (x_rows(M) * BK + C::B_BYTES));
#pragma unroll
                    for (int g = 0; g < C::GROUP; ++g)
                        if (g < blocks) {
                            uint8_t *a_dst = ring + stage * C::STAGE + g * C::BLOCK;
                            tma_load_2d(a_dst, &tm_x, &full[stage], (kb + g) * BK, m0);
                            tma_load_2d(a_dst + C::A_BYTES, &tm_w, &full[stage], (kb + g) * BK, n0);
                        }
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
        for (int tile = blockIdx.x; tile < num_tiles && !given_up(abort_flag); tile += gridDim.x) {
            if (!warp_wait(&acc_empty[acc], acc_phase ^ 1)) {
                report(status, DEV_TIMEOUT);
                *abort_flag = 1;
                break;
            }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + acc * BN;
            for (int kb = 0; kb < k_iters; kb += C::GROUP) {
                if (!warp_wait(&full[stage], phase)) {
                    report(status, DEV_TIMEOUT);
                    *abort_flag = 1;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int g = 0; g < C::GROUP; ++g) {
                    const uint32_t a_addr = smem_u32(ring + stage * C::STAGE + g * C::BLOCK);
                    const uint64_t ad = sdesc_sw128(a_addr, 16, 1024), bd = sdesc_sw128(a_addr + C::A_BYTES, 16, 1024);
                    if (leader && kb + g < k_iters)
#pragma unroll
                        for (int k = 0; k < BK / 32; ++k)  // +32 bytes per K step inside the swizzle atom
                            umma_f8_ss(d_tmem, ad + 2 * k, bd + 2 * k, idesc, (kb | g | k) != 0 ? 1u : 0u);
                }
                issued = true;
                if (leader) umma_commit(&empty[stage]);
                if (++stage == C::STAGES) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (given_up(abort_flag)) break;
            if (leader) umma_commit(&acc_full[acc]);
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1;
        }
        if (issued) {  // MMAs retire before TMEM is released, also where the epilogue gave up on them
            if (leader) umma_commit(probe);
            if (!mbar_wait_drain(probe, 0)) report(status, DEV_TIMEOUT);
        }
    } else {
        const int q = warp & 3;  // TMEM lane quarter this warp may access
        Slabs sl{epi_buf + q * 2 * kSlab, res_bar + 2 * q, colv + q * 2 * BN, 0, 0, 0};
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x) {
            if (given_up(abort_flag)) break;
            const int m0 = tile / n_tiles * 128 + q * 32, n0 = tile % n_tiles * BN;
            const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN;
            if (!finish_tile<BN, OUT_BF16>(&acc_full[acc], acc_phase, t_row, m0 + lane, m0, n0, M, N, ea, &tm_y, &tm_r, sl,
                                           lane)) {
                report(status, DEV_TIMEOUT);
                *abort_flag = 1;
                break;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[acc]);
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1;
        }
        leave(sl, status, lane);
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
    static constexpr int STAGES = 4;
    static constexpr int EPI_WARPS = 8;  // two per TMEM lane quarter, 128 columns each
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static constexpr int BN = 256;
    static constexpr int COLS = BN / (EPI_WARPS / 4);
    static constexpr uint32_t HALF = 128 * BK;     // 16 KB: 128 rows
    static constexpr uint32_t STAGE = 2 * HALF;    // this CTA's x rows + w rows
    static constexpr uint32_t RING = STAGES * STAGE;
    static constexpr uint32_t EPI = EPI_WARPS * 2 * kSlab;
    static constexpr uint32_t COLV = EPI_WARPS * 2 * COLS * 4;  // column vectors
    static constexpr uint32_t SMEM = 1024 + RING + EPI + COLV + 384;
    static constexpr uint32_t TMEM_COLS = 2 * BN;
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

template <bool OUT_BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg::THREADS, 1)
    linear_e4m3_pair(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_r, int M, int N, int K,
                     const EpiArgs ea, int *status)
{
    using C = PairCfg;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = smem;
    uint8_t *epi_buf = smem + C::RING;
    float *colv = reinterpret_cast<float *>(epi_buf + C::EPI);
    uint64_t *full = reinterpret_cast<uint64_t *>(epi_buf + C::EPI + C::COLV);  // used in the leader
    uint64_t *empty = full + C::STAGES;                               // both CTAs
    uint64_t *acc_full = empty + C::STAGES;                           // both CTAs [2]
    uint64_t *acc_empty = acc_full + 2;                               // used in the leader [2]
    uint64_t *res_bar = acc_empty + 2;       // [EPI_WARPS][2]
    uint64_t *probe = res_bar + 2 * C::EPI_WARPS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(probe + 1);
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
        for (int b = 0; b < 2 * C::EPI_WARPS; ++b) mbar_init(&res_bar[b], 1);
        mbar_init(probe, 1);
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
            for (int tile = pair; tile < num_tiles && !given_up(abort_flag); tile += npairs) {
                if (!warp_wait(&acc_empty[acc], acc_phase ^ 1)) {
                    report(status, DEV_TIMEOUT);
                    *abort_flag = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * C::BN;
                for (int kb = 0; kb < k_iters; ++kb) {
                    if (!warp_wait(&full[stage], phase)) {
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
                if (given_up(abort_flag)) break;
                if (leader) umma_commit_pair_both(&acc_full[acc]);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
            }
            if (issued) {  // as above
                if (leader) umma_commit_pair_leader(probe);
                if (!mbar_wait_drain(probe, 0)) report(status, DEV_TIMEOUT);
            }
        }
    } else {
        const int q = warp & 3;            // TMEM lane quarter
        const int h = (warp - 2) >> 2;     // column half
        Slabs sl{epi_buf + (warp - 2) * 2 * kSlab, res_bar + 2 * (warp - 2), colv + (warp - 2) * 2 * C::COLS, 0, 0, 0};
        const uint32_t leader_acc_empty[2] = {map_to_rank(&acc_empty[0], 0), map_to_rank(&acc_empty[1], 0)};
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int tile = pair; tile < num_tiles; tile += npairs) {
            if (given_up(abort_flag)) break;
            const int m0 = tile / n_tiles * 256 + static_cast<int>(rank) * 128 + q * 32;
            const int n0 = tile % n_tiles * C::BN + h * C::COLS;
            const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * C::BN + h * C::COLS;
            if (!finish_tile<C::COLS, OUT_BF16>(&acc_full[acc], acc_phase, t_row, m0 + lane, m0, n0, M, N, ea, &tm_y, &tm_r, sl,
                                                lane)) {
                report(status, DEV_TIMEOUT);
                *abort_flag = 1;
                break;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_acc_empty(leader_acc_empty[acc]);
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1;
        }
        leave(sl, status, lane);
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
    CUtensorMap x, w, y, r;
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
                    t.x, t.w, t.y, t.r, M, N, K, ea, current_device_status_word());
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
    return launch_k(linear_e4m3_pair<OUT_BF16>, dim3(2 * pairs), dim3(C::THREADS), C::SMEM, s, t.x, t.w, t.y, t.r, M, N, K, ea,
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
    // The narrowest tiles of 64 and 128 columns that are one round of the SMs, else pairs; without the rows
    // for those (or the columns), 256 columns where that is no more work per SM than 128.  At K =
    // 4,096: 1,024 x 1,024 is 128 tiles of 64, 9.6 us (of 128 11.2, 16 pairs 15.6); 2,048 x 1,024 128 of
    // 128, 12.1 (pairs 15.9, two rounds of 64 17.5); 4,099 x 1,024 68 pairs, 16.8 (two rounds of 128 19.4);
    // 300 x 8,192 96 of 256, 16.7 (192 of 128 18.7); 300 x 16,384 384 of 128, 27.8 (192 of 256 34.0).
    auto tiles = [&](int64_t bn) { return (m + 127) / 128 * ((n + bn - 1) / bn); };
    auto rounds = [&](int64_t bn) { return (tiles(bn) + sms - 1) / sms; };
    const bool pair = m >= 512 && n >= 256 && tiles(128) > sms;
    // the gated epilogues pair 32 gate with 32 input columns and fill a slab from 128
    const int bn = pair ? 128 : !glu && tiles(64) <= sms ? 64 : n > 128 && tiles(128) > sms && 2 * rounds(256) <= rounds(128) ? 256 : 128;
    Maps t;
    fe_status r = make_tmap_2d(&t.x, x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, m, k, k, x_rows(static_cast<int>(m)), BK);
    if (r == FE_OK) r = make_tmap_2d(&t.w, w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, n, k, k, bn, BK);
    if (r == FE_OK)
        r = bf16 ? make_tmap_2d(&t.y, y, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, m, ny, ny, 32, 64)
                 : make_tmap_2d(&t.y, y, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, m, n, n, 32, 32);
    t.r = t.y;  // not read without a residual
    if (r == FE_OK && residual) r = make_tmap_2d(&t.r, residual, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, m, n, n, 32, 32);
    if (r != FE_OK) {
        *st = r;
        return cudaSuccess;
    }
    const EpiArgs ea{sx, sw, epilogue == E_NONE || glu ? nullptr : bias, epilogue};
    const int M = static_cast<int>(m), N = static_cast<int>(n), K = static_cast<int>(k);
    if (pair) return bf16 ? launch_pair<true>(t, M, N, K, ea, s) : launch_pair<false>(t, M, N, K, ea, s);
    if (bn == 256) return bf16 ? launch_cta<256, true>(t, M, N, K, ea, s) : launch_cta<256, false>(t, M, N, K, ea, s);
    if (bn == 128) return bf16 ? launch_cta<128, true>(t, M, N, K, ea, s) : launch_cta<128, false>(t, M, N, K, ea, s);
    return bf16 ? launch_cta<64, true>(t, M, N, K, ea, s) : launch_cta<64, false>(t, M, N, K, ea, s);
}

cudaError_t set_wait_limit_linear_e4m3(uint64_t ns) { return set_wait_limit_this_file(ns); }

}  // namespace fe

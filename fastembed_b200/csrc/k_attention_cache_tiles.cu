// k_attention_cache_tiles.cu — attention over the paged 8-bit key-value cache on tcgen05, for
// prompts (many rows per key-value head).  The mathematics is that of k_attention_cache.cu:
//     s_ij = qf_i sk(j) (q_i . kc_j),  t_ij = s_ij + log2 sv(j),  P_ij = 2^(t_ij - m_i)
//     out_i = sum_j P_ij vc_j / sum_j P_ij / sv(j)
//
// A unit is (sequence, key-value head, ROWS rows), the rows being the new tokens times the
// query heads of the group, r = token * group + head, so one pass over the cache serves every
// query head that shares it.  A unit is one CTA: NS streams of 128 rows (two for head_dim 64
// and 128) over the same 128-token items, each with its own S, O and softmax warpgroup, so that
// one stream's softmax runs under the other's MMAs.  Units go out longest first (a causal
// prompt's last tile sees the most tokens); a unit's items may be split over CTAs.
//
//   K stays in 8 bits: S = Q K^T as kind::f8f6f4 with Q in two e4m3 parts, q = hi + lo.  A bf16
//     has 8 significant bits and each part holds 4, so after a power-of-two scaling of the row
//     (maximum in [128, 256)) the split is exact down to 2^-10 of the row's largest element and
//     off by at most 2^-18 of it below.  Two 8-bit products cost what one f16 product does and
//     the codes are multiplied as they lie in memory: nothing converts K.
//   V becomes f16 (exact) on four converter warps, which also zero the slots past the
//     sequence's end; O += P V as kind::f16 with P (f16) in TMEM over S.
//   Scales: an item's 16-token groups (a page holds at least one) each have (sk, log2 sv,
//     1 / sv) in a small ring that the producer fills.  P's reference moves only when a tile's
//     maximum exceeds it by 2^8, so P lies below 2^15.  The sum of P / sv underflows only where
//     the scales of a sequence's pages differ by more than 2^30: from the first such item on the
//     exponentials of the sum are taken apart from those of P.
//
//   warp 0       TMA producer: K and V pages of each item (a box is a page; a page that is not
//                there, or past the end, is read as zeros from outside the tensor)
//   warp 1       TMEM owner and MMA issuer (an elected lane), in the fixed order
//                PV0(n), S0(n+1), PV1(n), S1(n+1)
//   next 4 NS    softmax (thread = row); they also quantise Q into shared memory
//   last 4       V converters
// Waits are bounded; on timeout the CTA records FE_ERR_DEVICE_TIMEOUT and leaves.
#include <cuda.h>

#include <algorithm>

#include "fe_attention_cache.cuh"

namespace fe {
namespace {

constexpr int TK = 128;  // tokens per item
constexpr int kEnt = 8;  // ring of the items' scales; see the producer for why 8 is enough
constexpr float kBoost = 7.f;   // P is 2^7 at the reference maximum, below 2^15 before it moves
constexpr float kLazy = 8.f;

template <int HD>
struct TileCfg {
    static constexpr int NS = HD == 256 ? 1 : 2;      // streams of 128 rows
    static constexpr int ROWS = 128 * NS;
    static constexpr uint32_t KT = TK * HD;           // bytes of a K or raw V tile, and of a part of Q
    static constexpr uint32_t VT = 2 * TK * HD;       // bytes of an f16 V tile
    static constexpr int KS = HD == 256 ? 2 : 3;      // K slots
    static constexpr int RS = HD == 256 ? 1 : 2;      // raw V slots
    static constexpr int VS = HD == 256 ? 1 : 2;      // f16 V slots
    static constexpr int SOFT = 4 * NS;               // softmax warps
    static constexpr int WARPS = 2 + SOFT + 4;
    static constexpr int THREADS = 32 * WARPS;
    static constexpr uint32_t USED = 1024 + NS * 2 * KT + KS * KT + RS * KT + VS * VT + kEnt * 8 * 16 + 512;
    // more than half of an SM's: a CTA takes all 512 TMEM columns, a second one would wait for them
    static constexpr uint32_t SMEM = USED < 120 * 1024 ? 120 * 1024 : USED;
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

// Byte offset of 16-byte chunk c of row r in a tile of HD-byte rows as TMA writes it: boxes of
// 128 bytes with the 128-byte swizzle, or (head_dim 64) rows of 64 bytes with the 64-byte one.
template <int HD>
__device__ __forceinline__ uint32_t tile_offset(int r, int c)
{
    if constexpr (HD == 64) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
    else return (c >> 3) * (TK * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// Shared-memory descriptor of such a tile (K-major), advanced by `kk` steps of 32 bytes.
template <int HD>
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, int kk)
{
    if constexpr (HD == 64) {
        uint64_t d = sdesc_sw128(addr + 32 * kk, 16, 512);
        d &= ~(static_cast<uint64_t>(7) << 61);
        return d | (static_cast<uint64_t>(4) << 61);  // 64-byte swizzle
    } else {
        return sdesc_sw128(addr + (kk >> 2) * (TK * 128) + (kk & 3) * 32, 16, 1024);
    }
}

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// kind::f8f6f4, e4m3 A and B, fp32 D, both K-major
__device__ __forceinline__ uint32_t idesc_f8(int M, int N)
{
    return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// kind::f16, f16 A and B (format 0), fp32 D, A K-major, B MN-major
__host__ __device__ constexpr uint32_t idesc_f16_bt(int M, int N)
{
    return (1u << 4) | (1u << 16) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// e4m3(a), e4m3(b) and what they leave: hi = e4m3(x), lo = e4m3(x - hi); NaN where x is not finite
__device__ __forceinline__ void split_e4m3x2(float a, float b, uint32_t &hi, uint32_t &lo)
{
    hi = cvt_e4m3x2(a, b);
    const float2 h = e4m3x2_to_f32x2(hi);
    lo = cvt_e4m3x2(a - h.x, b - h.y);
}

template <int HD>
__global__ void __launch_bounds__(TileCfg<HD>::THREADS, 1)
    attn_cache_tiles(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const CacheArgs a,
                     int *status)
{
    using C = TileCfg<HD>;
    constexpr int NS = C::NS, KS = C::KS, RS = C::RS, VS = C::VS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sQ = smem;                         // [NS][hi, lo]
    uint8_t *sK = sQ + NS * 2 * C::KT;          // [KS]
    uint8_t *sR = sK + KS * C::KT;              // [RS] raw V
    uint8_t *sV = sR + RS * C::KT;              // [VS] f16 V, HD / 64 boxes of 128 rows x 128 bytes
    float4 *ent = reinterpret_cast<float4 *>(sV + VS * C::VT);  // [kEnt][8]: sk, log2 sv, 1 / sv, (group 0) spread flag
    uint64_t *bars = reinterpret_cast<uint64_t *>(ent + kEnt * 8);
    uint64_t *q_full = bars;            // [NS] one arrival per softmax warp of the stream
    uint64_t *k_full = q_full + NS;     // [KS]
    uint64_t *k_empty = k_full + KS;    // [KS] a commit per stream
    uint64_t *r_full = k_empty + KS;    // [RS]
    uint64_t *r_empty = r_full + RS;    // [RS] one arrival per converter warp
    uint64_t *v_full = r_empty + RS;    // [VS] one arrival per converter warp
    uint64_t *v_empty = v_full + VS;    // [VS] a commit per stream
    uint64_t *e_full = v_empty + VS;    // [kEnt]
    uint64_t *s_full = e_full + kEnt;   // [2]
    uint64_t *p_full = s_full + 2;      // [2] one arrival per softmax warp
    uint64_t *pv_done = p_full + 2;     // [2]
    uint64_t *probe = pv_done + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(probe + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    static_assert((NS + 2 * KS + 2 * RS + 2 * VS + kEnt + 7) * 8 + 8 <= 512, "barrier space");

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int kvh = blockIdx.x, b = blockIdx.y;
    const int tiles = gridDim.z / a.splits;
    const int tile = tiles - 1 - static_cast<int>(blockIdx.z) / a.splits, split = blockIdx.z % a.splits;
    grid_dep_wait();
    CacheSeq sq;
    if (!load_seq(a, b, sq, status)) return;
    const int rows = sq.len * a.group, r0 = tile * C::ROWS;
    if (r0 >= rows) return;
    // items of this CTA: its part of those the unit's last row sees
    const int end = a.causal ? sq.past + (min(r0 + C::ROWS, rows) - 1) / a.group + 1 : sq.kv;
    const int all = (end + TK - 1) / TK, per = (all + a.splits - 1) / a.splits;
    const int j0 = split * per;
    const int items = max(0, min(per, all - j0));

    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) mbar_init(&q_full[i], 4);
        for (int i = 0; i < KS; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], NS);
        }
        for (int i = 0; i < RS; ++i) {
            mbar_init(&r_full[i], 1);
            mbar_init(&r_empty[i], 4);
        }
        for (int i = 0; i < VS; ++i) {
            mbar_init(&v_full[i], 4);
            mbar_init(&v_empty[i], NS);
        }
        for (int i = 0; i < kEnt; ++i) mbar_init(&e_full[i], 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&pv_done[i], 1);
        }
        mbar_init(probe, 1);
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dep_launch();
    const uint32_t tmem = *tmem_slot;  // S slots at 0 and 128, O of stream s at 256 + s * HD

    // S slot and phase of item n: two streams own a slot each, one stream alternates
    auto slot_of = [](int s, int n) { return NS == 2 ? s : n & 1; };
    auto phase_of = [](int n) -> uint32_t { return NS == 2 ? n & 1 : (n >> 1) & 1; };
    // whole warps wait, and give up together
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        if (__all_sync(0xffffffffu, mbar_wait(bar, parity))) return true;
        report(status, DEV_TIMEOUT);
        *abort_flag = 1;
        return false;
    };

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        // K(n) goes into its slot once S(n - KS) of every stream is done, and S(m) is issued only
        // after the softmax of item m - 1 (one stream: m - 2) has read its scales: when the scales of
        // item n are written, those of item n - KS - 2 and before have been read, so 8 entries do.
        const bool leader = elect_lane();
        const int page = 1 << a.page_log2, ppi = a.page_log2 >= 7 ? 1 : TK >> a.page_log2;  // pages per item
        const int64_t none = static_cast<int64_t>(a.pages) * a.kv_heads << a.page_log2;     // a row outside the pool
        const int32_t *tab = a.table + static_cast<int64_t>(b) * a.width;
        float ref = 0.f;
        bool have_ref = false, spread = false;
        bool ok = true;
        int kn = 0, vn = 0;
        // lane i < 8: the page of token group i of an item, its row in the pool (or `none`)
        auto page_row = [&](int j, int g) -> int64_t {
            const int tok = j * TK + 16 * g;
            if (tok >= end) return none;
            const int id = __ldg(tab + (tok >> a.page_log2));
            if (id < 0 || id >= a.pages) {
                report(status, DEV_BAD_INPUT);
                return none;
            }
            return (static_cast<int64_t>(id) * a.kv_heads + kvh) << a.page_log2;
        };
        auto load = [&](const CUtensorMap *map, uint8_t *dst, uint64_t *bar, int64_t row) {
            // row: this lane's group's page row; one box a page
            if (leader) mbar_arrive_expect_tx(bar, C::KT);
            for (int p = 0; p < ppi; ++p) {
                const int y = static_cast<int>(__shfl_sync(0xffffffffu, row, p << (a.page_log2 - 4)));
                if (leader) {
                    if constexpr (HD == 64) tma_load_2d(dst + p * page * 64, map, bar, 0, y);
                    else
#pragma unroll
                        for (int x = 0; x < HD / 128; ++x)
                            tma_load_2d(dst + x * (TK * 128) + p * page * 128, map, bar, 128 * x, y);
                }
            }
        };
        for (int n = 0; n < items && ok && !*abort_flag; ++n) {
            const int ks = n % KS, rs = n % RS;
            const int64_t row = lane < 8 ? page_row(j0 + n, lane) : none;
            float4 e = make_float4(0.f, -INFINITY, 0.f, 0.f);  // a group that is not there: weight 0
            if (row != none) {
                const int64_t ph = row >> a.page_log2;
                const float sv = __ldg(a.vs + ph);
                e.x = __ldg(a.ks + ph);
                e.y = sv > 0.f ? log2f(sv) : 0.f;  // a page of zero values adds nothing to O
                e.z = sv > 0.f ? 1.0f / sv : 1.f;
            }
            const uint32_t there = __ballot_sync(0xffffffffu, row != none);
            if (there && !have_ref) {
                ref = __shfl_sync(0xffffffffu, e.y, __ffs(there) - 1);
                have_ref = true;
            }
            spread |= __any_sync(0xffffffffu, row != none && fabsf(e.y - ref) > 30.f);
            if (!(ok = wait(&k_empty[ks], ((n / KS) & 1) ^ 1))) break;
            if (lane < 8) {
                e.w = spread ? 1.f : 0.f;
                ent[(n % kEnt) * 8 + lane] = e;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&e_full[n % kEnt]);
            load(&tm_k, sK + ks * C::KT, &k_full[ks], row);
            kn = n + 1;
            if (!(ok = wait(&r_empty[rs], ((n / RS) & 1) ^ 1))) break;
            load(&tm_v, sR + rs * C::KT, &r_full[rs], row);
            vn = n + 1;
        }
        // every load this warp started lands before the CTA exits
        for (int n = max(0, kn - KS); n < kn; ++n) (void)mbar_wait_drain(&k_full[n % KS], (n / KS) & 1);
        for (int n = max(0, vn - RS); n < vn; ++n) (void)mbar_wait_drain(&r_full[n % RS], (n / RS) & 1);
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        const bool leader = elect_lane();
        constexpr uint32_t idesc_o = idesc_f16_bt(128, HD);
        bool issued = false;
        auto issue_s = [&](int s, int n) -> bool {
            const int ks = n % KS, sl = slot_of(s, n);
            if (!wait(&k_full[ks], (n / KS) & 1)) return false;
            if (n == 0 && !wait(&q_full[s], 0)) return false;
            // P of the slot's previous item consumed
            if (n >= (NS == 2 ? 1 : 2) && !wait(&pv_done[sl], phase_of(n - (NS == 2 ? 1 : 2)))) return false;
            tc_fence_after();
            const int n16 = min(TK, (end - (j0 + n) * TK + 15) & ~15);
            const uint32_t idesc = idesc_f8(128, n16);
            const uint32_t qa = smem_u32(sQ + s * 2 * C::KT), ka = smem_u32(sK + ks * C::KT);
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
                for (int kk = 0; kk < HD / 32; ++kk)
                    if (leader)
                        umma_f8(tmem + sl * 128, tile_desc<HD>(qa + part * C::KT, kk), tile_desc<HD>(ka, kk), idesc,
                                (part | kk) != 0 ? 1u : 0u);
            issued = true;
            if (leader) {
                umma_commit(&s_full[sl]);
                umma_commit(&k_empty[ks]);
            }
            return true;
        };
        auto issue_pv = [&](int s, int n) -> bool {
            const int vs = n % VS, sl = slot_of(s, n);
            if (!wait(&p_full[sl], phase_of(n))) return false;
            if (!wait(&v_full[vs], (n / VS) & 1)) return false;
            tc_fence_after();
            const int steps = (min(TK, end - (j0 + n) * TK) + 15) >> 4;
            const uint64_t vd = sdesc_sw128(smem_u32(sV + vs * C::VT), TK * 128, 1024);
            for (int k = 0; k < steps; ++k)  // 16 tokens = 16 rows of 128 bytes
                if (leader)
                    umma_f16_ts(tmem + 256 + s * HD, tmem + sl * 128 + k * 8, vd + static_cast<uint64_t>(k * 128), idesc_o,
                                (n | k) != 0 ? 1u : 0u);
            if (leader) {
                umma_commit(&pv_done[sl]);
                umma_commit(&v_empty[vs]);
            }
            return true;
        };
        bool ok = items > 0;
        for (int s = 0; s < NS && ok; ++s) ok = issue_s(s, 0);
        for (int n = 0; n < items && ok && !*abort_flag; ++n) {
            const bool more = n + 1 < items;
            if constexpr (NS == 2)
                ok = issue_pv(0, n) && (!more || issue_s(0, n + 1)) && issue_pv(1, n) && (!more || issue_s(1, n + 1));
            else  // the next S fills the other slot while this item's softmax runs
                ok = (!more || issue_s(0, n + 1)) && issue_pv(0, n);
        }
        if (issued) {  // MMAs retire before TMEM is released
            if (leader) umma_commit(probe);
            (void)mbar_wait_drain(probe, 0);
        }
    } else if (warp < 2 + C::SOFT) {
        // ------------------------------------------------ softmax: thread = row
        const int s = (warp - 2) >> 2, q = warp & 3;
        const int r = q * 32 + lane;  // row within the stream == TMEM lane
        const int rr = r0 + 128 * s + r;
        const bool live = rr < rows, warp_live = r0 + 128 * s + q * 32 < rows;
        const int token = live ? rr / a.group : 0, head = kvh * a.group + (live ? rr - token * a.group : 0);
        const int vis = !live ? 0 : a.causal ? sq.past + token + 1 : sq.kv;  // tokens this row sees
        float qf = 0.f;
        {
            // Q: the row's maximum to [128, 256), split in two e4m3 parts
            const __nv_bfloat16 *p = a.qkv + (sq.t0 + token) * a.row + static_cast<int64_t>(head) * HD;
            uint32_t m = 0;  // of |q| as bf16 bits: their order is that of the values
            if (live)
#pragma unroll 4
                for (int c = 0; c < HD / 8; ++c) {
                    const uint4 u = *reinterpret_cast<const uint4 *>(p + 8 * c);
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t x = w[i] & 0x7fffu, y = (w[i] >> 16) & 0x7fffu;
                        m = max(m, max(x < 0x7f80u ? x : 0u, y < 0x7f80u ? y : 0u));
                    }
                }
            int e = static_cast<int>(m >> 7) - 127 - 7;  // q * 2^-e has its maximum in [128, 256)
            e = max(-100, e);
            const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            // a negative softmax scale turns Q's signs, so that the logit factor is never negative
            const float sign = a.scale_log2 < 0.f ? -down : down;
            qf = fabsf(a.scale_log2) * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            uint8_t *hi = sQ + s * 2 * C::KT, *lo = hi + C::KT;
#pragma unroll 2
            for (int c = 0; c < HD / 16; ++c) {
                uint4 u[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                if (live) {
                    u[0] = *reinterpret_cast<const uint4 *>(p + 16 * c);
                    u[1] = *reinterpret_cast<const uint4 *>(p + 16 * c + 8);
                }
                const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
                uint32_t h[4], l[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 x = unpack_bf16x2(w[2 * i]), y = unpack_bf16x2(w[2 * i + 1]);
                    uint32_t h0, l0, h1, l1;
                    split_e4m3x2(scaled_or_nan(x.x, sign), scaled_or_nan(x.y, sign), h0, l0);
                    split_e4m3x2(scaled_or_nan(y.x, sign), scaled_or_nan(y.y, sign), h1, l1);
                    h[i] = h0 | (h1 << 16);
                    l[i] = l0 | (l1 << 16);
                }
                const uint32_t at = tile_offset<HD>(r, c);
                *reinterpret_cast<uint4 *>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
                *reinterpret_cast<uint4 *>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[s]);
        }
        const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
        const uint32_t tO = tmem + lanes + 256 + s * HD;
        float m_run = -INFINITY, l_run = 0.f;
        bool ok = true;
        for (int n = 0; n < items; ++n) {
            const int sl = slot_of(s, n);
            const uint32_t tS = tmem + lanes + sl * 128;
            if (!(ok = wait(&e_full[n % kEnt], (n / kEnt) & 1) && wait(&s_full[sl], phase_of(n)))) break;
            tc_fence_after();
            const float4 *en = ent + (n % kEnt) * 8;
            const int base = (j0 + n) * TK, cols = min(TK, end - base), lim = vis - base;
            float alpha = 1.f;
            if (warp_live) {
                const bool spread = en[0].w != 0.f;
                float top = m_run;
                for (int c = 0; c < cols; c += 32) {
                    uint32_t v[32];
                    __syncwarp();
                    tmem_ld_x32(tS + c, v);
                    tmem_wait_ld_regs(v);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float m0 = -INFINITY, m1 = -INFINITY;
                        if (c + 32 <= lim) {  // nothing masked
#pragma unroll
                            for (int i = 0; i < 16; i += 4) {
                                m0 = max3f(m0, __uint_as_float(v[16 * h + i]), __uint_as_float(v[16 * h + i + 1]));
                                m1 = max3f(m1, __uint_as_float(v[16 * h + i + 2]), __uint_as_float(v[16 * h + i + 3]));
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (c + 16 * h + i < lim) m0 = fmaxf(m0, __uint_as_float(v[16 * h + i]));
                        }
                        m0 = fmaxf(m0, m1);
                        const float4 e = en[(c >> 4) + h];
                        if (m0 != -INFINITY) top = fmaxf(top, fmaf(m0, qf * e.x, e.y));
                    }
                }
                // the reference rises only when a tile exceeds it by more than 2^8
                if (top > m_run + kLazy || m_run == -INFINITY) {
                    alpha = m_run == -INFINITY ? 0.f : exp2_fast(m_run - top);
                    m_run = top;
                }
                const float shift = m_run == -INFINITY ? 0.f : kBoost - m_run;
                float sum = 0.f;
                __syncwarp();
                for (int c = 0; c < cols; c += 32) {
                    uint32_t v[32];
                    tmem_ld_x32(tS + c, v);
                    tmem_wait_ld_regs(v);
                    uint32_t pk[16];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float4 e = en[(c >> 4) + h];
                        const float f = qf * e.x, g = e.y + shift;
                        float s0 = 0.f, s1 = 0.f;
                        if (c + 16 * h >= lim) {  // all masked
#pragma unroll
                            for (int i = 0; i < 8; ++i) pk[8 * h + i] = 0;
                            continue;
                        }
                        const bool whole = c + 16 * h + 16 <= lim;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            float p0, p1;
                            fma_f32x2(p0, p1, __uint_as_float(v[16 * h + 2 * i]), __uint_as_float(v[16 * h + 2 * i + 1]), f, g);
                            p0 = exp2_fast(p0);
                            p1 = exp2_fast(p1);
                            if (!whole) {
                                if (c + 16 * h + 2 * i >= lim) p0 = 0.f;
                                if (c + 16 * h + 2 * i + 1 >= lim) p1 = 0.f;
                            }
                            add_f32x2(s0, s1, p0, p1);
                            pk[8 * h + i] = pack_f16x2(p0, p1);
                        }
                        if (!spread) {
                            sum = fmaf(s0 + s1, e.z, sum);
                        } else if (e.z != 0.f) {  // P / sv from its own exponentials
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (c + 16 * h + i < lim) sum += exp2_fast(fmaf(__uint_as_float(v[16 * h + i]), f, shift));
                        }
                    }
                    __syncwarp();
                    tmem_st_x16(tS + (c >> 1), pk);
                }
                l_run = fmaf(l_run, alpha, sum);
                tmem_wait_st();
            }
            // O *= alpha after the previous item's PV and before this one's
            if (n > 0 && warp_live && __any_sync(0xffffffffu, alpha != 1.f)) {
                if (!(ok = wait(&pv_done[slot_of(s, n - 1)], phase_of(n - 1)))) break;
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t v[32];
                    tmem_ld_x32(tO + c, v);
                    tmem_wait_ld_regs(v);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
                    tmem_st_x32(tO + c, v);
                }
                tmem_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[sl]);
        }
        if (ok && items > 0) ok = wait(&pv_done[slot_of(s, items - 1)], phase_of(items - 1));
        tc_fence_after();
        if (ok && warp_live) {
            const int64_t orow = (static_cast<int64_t>(sq.t0) + token) * a.q_heads + head;
            const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;  // a row that sees nothing is zero
            if (a.splits > 1 && live)
                *reinterpret_cast<float2 *>(a.part_ml + (orow * a.splits + split) * 2) = make_float2(m_run, l_run);
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                uint32_t v[32];
                if (items > 0) {
                    tmem_ld_x32(tO + c, v);
                    tmem_wait_ld_regs(v);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0;
                }
                if (live && a.splits > 1) {
                    float4 *dst = reinterpret_cast<float4 *>(a.part_o + (orow * a.splits + split) * HD + c);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        dst[i] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                             __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
                } else if (live) {
                    uint4 *dst = reinterpret_cast<uint4 *>(a.out + orow * HD + c);
                    uint32_t o[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        o[i] = pack_bf16x2(__uint_as_float(v[2 * i]) * inv, __uint_as_float(v[2 * i + 1]) * inv);
#pragma unroll
                    for (int i = 0; i < 4; ++i) dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
                __syncwarp();
            }
        }
    } else {
        // ------------------------------------------------ V converters
        const int t = threadIdx.x - 32 * (2 + C::SOFT);
        constexpr int CPR = HD / 16;  // 16-code chunks per row
        for (int n = 0; n < items && !*abort_flag; ++n) {
            const int rs = n % RS, vs = n % VS;
            if (!wait(&r_full[rs], (n / RS) & 1)) break;
            if (!wait(&v_empty[vs], ((n / VS) & 1) ^ 1)) break;
            const int valid = sq.kv - (j0 + n) * TK;  // slots past the sequence's end hold anything
            const uint8_t *src = sR + rs * C::KT;
            uint8_t *dst = sV + vs * C::VT;
#pragma unroll 4
            for (int i = t; i < TK * CPR; i += 128) {
                const int r = i / CPR, c = i % CPR;
                uint4 u = *reinterpret_cast<const uint4 *>(src + tile_offset<HD>(r, c));
                if (r >= valid) u = make_uint4(0, 0, 0, 0);
                const uint4 lo = make_uint4(e4m3x2_to_f16x2(u.x), e4m3x2_to_f16x2(u.x >> 16), e4m3x2_to_f16x2(u.y),
                                            e4m3x2_to_f16x2(u.y >> 16));
                const uint4 hi = make_uint4(e4m3x2_to_f16x2(u.z), e4m3x2_to_f16x2(u.z >> 16), e4m3x2_to_f16x2(u.w),
                                            e4m3x2_to_f16x2(u.w >> 16));
                // 16 codes = two 16-byte chunks of the 64-column box c / 4; the lanes of odd boxes
                // write their second chunk first, so that a row's eight lanes meet eight banks
                uint8_t *row = dst + (c >> 2) * (TK * 128) + r * 128;
                const int c0 = 2 * (c & 3), flip = (c >> 2) & 1;
                *reinterpret_cast<uint4 *>(row + (((c0 + flip) ^ (r & 7)) << 4)) = flip ? hi : lo;
                *reinterpret_cast<uint4 *>(row + (((c0 + 1 - flip) ^ (r & 7)) << 4)) = flip ? lo : hi;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&v_full[vs]);
                mbar_arrive(&r_empty[rs]);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int HD>
cudaError_t launch(const CacheArgs &a, int *status, cudaStream_t s, fe_status *st)
{
    using C = TileCfg<HD>;
    static uint64_t configured[64] = {};  // context the attribute was set in
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t ctx = current_context_id();
    if (dev >= 64 || configured[dev] != ctx) {
        cudaError_t e = cudaFuncSetAttribute(attn_cache_tiles<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured[dev] = ctx;
    }
    CUtensorMap tk, tv;
    const uint64_t n = static_cast<uint64_t>(a.pages) * a.kv_heads << a.page_log2;
    const uint32_t box = 1u << a.page_log2;
    const CUtensorMapSwizzle sw = HD == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    *st = make_tmap_2d(&tk, a.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, n, HD, HD, box, HD == 64 ? 64 : 128, sw);
    if (*st == FE_OK) *st = make_tmap_2d(&tv, a.v, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, n, HD, HD, box, HD == 64 ? 64 : 128, sw);
    if (*st != FE_OK) return cudaSuccess;
    const int tiles = static_cast<int>((static_cast<int64_t>(a.max_len) * a.group + C::ROWS - 1) / C::ROWS);
    return launch_k(attn_cache_tiles<HD>, dim3(a.kv_heads, a.batch, tiles * a.splits), dim3(C::THREADS), C::SMEM, s, tk, tv,
                    a, status);
}

}  // namespace

int attention_cache_tile_rows(int head_dim) { return head_dim == 256 ? TileCfg<256>::ROWS : TileCfg<128>::ROWS; }

cudaError_t launch_attention_cache_tiles(const CacheArgs &a, int head_dim, int *status, cudaStream_t s, fe_status *st)
{
    if (head_dim == 64) return launch<64>(a, status, s, st);
    if (head_dim == 128) return launch<128>(a, status, s, st);
    return launch<256>(a, status, s, st);
}

cudaError_t set_wait_limit_attention_cache(uint64_t ns) { return set_wait_limit_this_file(ns); }

}  // namespace fe

// k_attention_cache_tiles.cu — attention over the paged 8-bit key-value cache on tcgen05, for
// prompts (many rows per key-value head).  The mathematics is that of k_attention_cache.cu:
//     s_ij = qf_i sk(j) (q_i . kc_j),  t_ij = s_ij + log2 sv(j),  P_ij = 2^(t_ij - m_i)
//     out_i = 2^(m_i - n_i) sum_j P_ij vc_j / sum_j 2^(s_ij - n_i)
// While the pages' value scales lie within 2^30 of the first one's, sv0, the sum of weights comes from the same
// exponentials: 2^(s_ij - n_i) = P_ij sv0 / sv(j) with n_i = m_i - log2 sv0.  From the first page that is further
// off (or has nothing but zeros, sv = 0) on, it has exponentials and a running reference n_i of its own.
//
// A unit is (sequence, key-value head, ROWS rows), the rows being the new tokens times the
// query heads of the group, r = token * group + head, so one pass over the cache serves every
// query head that shares it.  A unit is one CTA: NS streams of 128 rows (two for head_dim 64
// and 128) over the same 128-token items, each with its own S, O and softmax warpgroup.  Units go
// out by tile, the last tile of every sequence first: longest first where the prompts are about as long as each
// other (a causal prompt's last tile sees the most tokens).  Beside a prompt, a single token over a long cache
// has its only tile at the end of that order.  A unit's items may be split over CTAs.
//
//   Steps of 64 tokens: a stream has two 64-column S slots in TMEM, S of a step goes into the
//     slot that the step before the last has left, and so S(k + 1) and PV(k - 1) run under the
//     softmax of step k.  (One 128-column slot per stream, where S had to wait for the previous
//     PV, took 250 us where this took 224: 8 prompts of 2,000 tokens after 1,000, 16 heads to 8, now 215.)
//   K stays in 8 bits: S = Q K^T as kind::f8f6f4 with Q in two e4m3 parts, q = hi + lo.  A bf16
//     has 8 significant bits and each part holds 4: hi is the upper four, lo the rest.  After a
//     power-of-two scaling of the row (maximum in [128, 256)) that is exact down to 2^-10 of the
//     row's largest element and off by at most 2^-16 of it below.  Two 8-bit products cost what one
//     f16 product does and the codes are multiplied as they lie in memory: nothing converts K.
//   V becomes f16 (exact) on four converter warps, which also zero the slots past the
//     sequence's end; O += P V as kind::f16 with P (f16) in TMEM over S.
//   Scales: an item's 16-token groups (a page holds at least one) each have (sk, log2 sv,
//     1 / sv) in a small ring that the producer fills.  P's reference moves only when a step's
//     maximum exceeds it by 2^8, so P lies below 2^15.  The sum of P / sv underflows only where
//     the scales of a sequence's pages differ by more than 2^30: from the first such item on the
//     exponentials of the sum are taken apart from those of P.
//
//   warp 0       TMA producer: K and V pages of each item (a box is a page; a page that is not
//                there, or past the end, is read as zeros from outside the tensor)
//   next NS      MMA issuers, one per stream (an elected lane each): PV(k), S(k + 2).  One warp for
//                both streams was what bounded the kernel: waits on barriers long complete, commits
//                and issue cost a warp some 600 clocks a product beside busy softmax warps, 2,500 a
//                step where the tensor cores need 1,290.
//   next 4 NS    softmax (thread = row); they also quantise Q into shared memory
//   last 4       V converters
// Waits are bounded; on timeout the CTA records FE_ERR_DEVICE_TIMEOUT and leaves.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

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
    static constexpr int WARPS = 1 + NS + SOFT + 4;
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

// Shared-memory descriptors as (address + LBO, SBO + version + layout) words: bits [0,14) address
// >> 4, [16,30) leading byte offset >> 4, [32,46) stride byte offset >> 4, [46,48) version 1,
// [61,64) layout (2 = 128-byte swizzle, 4 = 64-byte).
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return (addr >> 4) | (lbo >> 4 << 16); }
__host__ __device__ constexpr uint32_t desc_hi(uint32_t sbo, uint32_t layout) { return (sbo >> 4) | (1u << 14) | (layout << 29); }

// The MMAs of this kernel take their shared-memory descriptors as a low word (the address, which
// is all that changes) and a high word fixed per layout: the issuing warp shares its scheduler
// with softmax warps, and 64-bit address arithmetic is instructions that it waits for.
template <uint32_t HI_A, uint32_t HI_B, bool ACC>
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %4};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "n"(HI_A), "n"(HI_B), "n"(ACC ? 1 : 0)
        : "memory");
}

template <uint32_t HI_B>
__device__ __forceinline__ void umma_pv(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %4};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "r"(idesc), "n"(HI_B), "r"(accumulate)
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

// Two bf16 times a power of two as e4m3 codes
__device__ __forceinline__ uint32_t scaled_codes(uint32_t w, float f)
{
    float2 x = unpack_bf16x2(w);
    mul_f32x2(x.x, x.y, f, f);
    return cvt_e4m3x2(x.x, x.y);
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
    // [kEnt][8]: sk, log2 sv, sv0 / sv; then, in group 0, whether the scales are spread, in 1 log2 sv0, in 2 the first
    // token that is there
    float4 *ent = reinterpret_cast<float4 *>(sV + VS * C::VT);
    uint64_t *bars = reinterpret_cast<uint64_t *>(ent + kEnt * 8);
    uint64_t *k_full = bars;            // [KS]
    uint64_t *k_empty = k_full + KS;    // [KS] a commit per stream
    uint64_t *r_full = k_empty + KS;    // [RS]
    uint64_t *r_empty = r_full + RS;    // [RS] one arrival per converter warp
    uint64_t *v_full = r_empty + RS;    // [VS] one arrival per converter warp
    uint64_t *v_empty = v_full + VS;    // [VS] a commit per stream
    uint64_t *s_full = v_empty + VS;      // [NS][slot]
    uint64_t *p_full = s_full + 2 * NS;   // [NS][slot] one arrival per softmax warp
    uint64_t *pv_done = p_full + 2 * NS;  // [NS][slot]
    uint64_t *probe = pv_done + 2 * NS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(probe + NS);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    static_assert((7 * NS + 2 * KS + 2 * RS + 2 * VS) * 8 + 8 <= 512, "barrier space");

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
    const int streams = r0 + 128 < rows ? NS : 1;  // with a row; the second takes no part without

    if (threadIdx.x == 0) {
        for (int i = 0; i < KS; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], streams);
        }
        for (int i = 0; i < RS; ++i) {
            mbar_init(&r_full[i], 1);
            mbar_init(&r_empty[i], 4);
        }
        for (int i = 0; i < VS; ++i) {
            mbar_init(&v_full[i], 4);
            mbar_init(&v_empty[i], streams);
        }
        for (int i = 0; i < 2 * NS; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&pv_done[i], 1);
        }
        for (int i = 0; i < NS; ++i) mbar_init(&probe[i], 1);
        *abort_flag = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    __syncwarp();
    // Until here only warp 0 has anything of the CTA's state.  It starts the first item's loads while warp 1
    // allocates TMEM and the softmax warps quantise Q; then all meet (that after a common set-up:
    // 0.3 us more a unit of 7 in a row, 0.5 at head_dim 256).  S slot k & 1 of stream s is at
    // TMEM column 128 s + 64 (k & 1), O of stream s at 256 + s HD.
    auto meet = [&]() -> uint32_t {
        tc_fence_before();
        asm volatile("bar.sync 0;" ::: "memory");
        tc_fence_after();
        grid_dep_launch();
        return *reinterpret_cast<volatile uint32_t *>(tmem_slot);
    };
    uint32_t tmem;

    // step k is half k & 1 of item k / 2; a step that lies past the end is not there
    const int steps = items == 0 ? 0 : 2 * items - (end - (j0 + items - 1) * TK <= 64 ? 1 : 0);
    // a stream's barriers of step k: slot k & 1, in turn
    auto slot_of = [](int s, int k) { return 2 * s + (k & 1); };
    auto phase_of = [](int k) -> uint32_t { return (k >> 1) & 1; };
    // whole warps wait, and give up together
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        if (__all_sync(0xffffffffu, mbar_wait(bar, parity))) return true;
        report(status, DEV_TIMEOUT);
        *abort_flag = 1;
        return false;
    };
    auto given_up = [&]() -> bool { return __any_sync(0xffffffffu, *abort_flag != 0); };

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        // K(n) goes into its slot once every stream's S over item n - KS is done.  The second of those
        // is issued after the PV of the step two before it, the last of item n - KS - 1, so after
        // the softmax that read that item's scales: KS + 1 entries are in use, 8 do.
        const bool leader = elect_lane();
        const int page = 1 << a.page_log2, ppi = a.page_log2 >= 7 ? 1 : TK >> a.page_log2;  // pages per item
        const int64_t none = static_cast<int64_t>(a.pages) * a.kv_heads << a.page_log2;     // a row outside the pool
        const int32_t *tab = a.table + static_cast<int64_t>(b) * a.width;
        float ref = 0.f, ref_sv = 1.f;
        int first_there = 0x7fffffff;  // of this CTA's items so far
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
        auto fetch = [&](int n) -> bool {
            const int ks = n % KS, rs = n % RS;
            const int64_t row = lane < 8 ? page_row(j0 + n, lane) : none;
            float4 e = make_float4(0.f, -INFINITY, 0.f, 0.f);  // a group that is not there: weight 0
            if (row != none) {
                const int64_t ph = row >> a.page_log2;
                const float sv = __ldg(a.vs + ph);
                e.x = __ldg(a.ks + ph);
                if (sv > 0.f) e.y = log2f(sv);
                e.z = sv;
            }
            const uint32_t there = __ballot_sync(0xffffffffu, row != none);
            if (there) first_there = min(first_there, (j0 + n) * TK + 16 * (__ffs(there) - 1));
            const uint32_t valued = __ballot_sync(0xffffffffu, e.z > 0.f);
            if (valued && !have_ref) {
                ref = __shfl_sync(0xffffffffu, e.y, __ffs(valued) - 1);
                ref_sv = __shfl_sync(0xffffffffu, e.z, __ffs(valued) - 1);
                have_ref = true;
            }
            spread |= __any_sync(0xffffffffu, row != none && !(fabsf(e.y - ref) <= 30.f));
            if (row != none) e.z = spread ? 1.f : ref_sv / e.z;
            if (!wait(&k_empty[ks], ((n / KS) & 1) ^ 1)) return false;
            if (lane < 8) {
                e.w = lane == 0 ? (spread ? 1.f : 0.f) : lane == 1 ? ref : __int_as_float(first_there);
                ent[(n % kEnt) * 8 + lane] = e;
            }
            __syncwarp();  // the entries are written before the leader's arrival for K
            load(&tm_k, sK + ks * C::KT, &k_full[ks], row);
            kn = n + 1;
            if (!wait(&r_empty[rs], ((n / RS) & 1) ^ 1)) return false;
            load(&tm_v, sR + rs * C::KT, &r_full[rs], row);
            vn = n + 1;
            return true;
        };
        if (items > 0) ok = fetch(0);
        tmem = meet();
        for (int n = 1; n < items && ok && !given_up(); ++n) ok = fetch(n);
        // every load this warp started lands before the CTA exits
        for (int n = max(0, kn - KS); n < kn; ++n) (void)mbar_wait_drain(&k_full[n % KS], (n / KS) & 1);
        for (int n = max(0, vn - RS); n < vn; ++n) (void)mbar_wait_drain(&r_full[n % RS], (n / RS) & 1);
    } else if (warp <= NS) {
        // ------------------------------------------------ MMA issuer of a stream
        if (warp == 1) {
            tmem_alloc(tmem_slot, 512);
            tmem_relinquish();
        }
        tmem = meet();
        const int s = warp - 1;
        const bool leader = elect_lane();
        constexpr uint32_t idesc_o = idesc_f16_bt(128, HD);
        constexpr uint32_t kt = C::KT >> 4, vt = C::VT >> 4;  // in descriptor units of 16 bytes
        constexpr uint32_t half_k = (HD == 64 ? 64 * 64 : 64 * 128) >> 4, half_v = 64 * 128 >> 4, box = TK * 128 >> 4;
        constexpr uint32_t hi_k = HD == 64 ? desc_hi(512, 4) : desc_hi(1024, 2), hi_v = desc_hi(1024, 2);
        bool issued = false;
        const uint32_t qs = desc_lo(smem_u32(sQ) + s * 2 * C::KT, 16), kd0 = desc_lo(smem_u32(sK), 16);
        const uint32_t vd0 = desc_lo(smem_u32(sV), TK * 128);  // MN-major: LBO between 64-column boxes
        const uint32_t st = tmem + s * 128, od = tmem + 256 + s * HD;
        // the K ring's position of the next S, the V ring's of the next PV
        struct Ring {
            uint32_t slot, phase, at;
            __device__ __forceinline__ void next(uint32_t depth, uint32_t size)
            {
                ++slot;
                at += size;
                if (slot == depth) slot = 0, at = 0, phase ^= 1;
            }
        };
        Ring kr = {}, vr = {};
        // left: tokens from the step's first on (more than 0); par: the phase of the step's item
        auto issue_s = [&](auto hc, bool first, uint32_t par, int left) -> bool {
            constexpr int h = decltype(hc)::value;
            if (h == 0 && !wait(&k_full[kr.slot], kr.phase)) return false;
            if (!first && !wait(&pv_done[2 * s + h], par ^ 1)) return false;  // P of the slot's previous step consumed
            tc_fence_after();
            const uint32_t idesc = idesc_f8(128, min(64, (left + 15) & ~15));
            const uint32_t kd = kd0 + kr.at + h * half_k;
            if (leader) {
                umma_f8<hi_k, hi_k, false>(st + 64 * h, qs, kd, idesc);
#pragma unroll
                for (int i = 1; i < HD / 16; ++i) {  // the steps of 32 codes of both parts of Q
                    const int part = i / (HD / 32), kk = i % (HD / 32);
                    const uint32_t at = HD == 64 ? 2 * kk : (kk >> 2) * box + (kk & 3) * 2;
                    umma_f8<hi_k, hi_k, true>(st + 64 * h, qs + part * kt + at, kd + at, idesc);
                }
                umma_commit(&s_full[2 * s + h]);
                if (h) umma_commit(&k_empty[kr.slot]);
            }
            __syncwarp();  // no lane goes on to wait before the leader has issued
            issued = true;
            if (h) kr.next(KS, kt);
            return true;
        };
        auto issue_pv = [&](auto hc, bool first, uint32_t par, int left) -> bool {
            constexpr int h = decltype(hc)::value;
            if (h == 0 && !wait(&v_full[vr.slot], vr.phase)) return false;
            if (!wait(&p_full[2 * s + h], par)) return false;
            tc_fence_after();
            const uint32_t vd = vd0 + vr.at + h * half_v, pt = st + 64 * h;  // 16 tokens = 16 rows of 128 bytes
            if (leader) {
                umma_pv<hi_v>(od, pt, vd, idesc_o, h == 0 && first ? 0u : 1u);
                if (left > 48) {
#pragma unroll
                    for (int i = 1; i < 4; ++i) umma_pv<hi_v>(od, pt + 8 * i, vd + i * 128, idesc_o, 1u);
                } else {
                    for (int i = 1; 16 * i < left; ++i) umma_pv<hi_v>(od, pt + 8 * i, vd + i * 128, idesc_o, 1u);
                }
                umma_commit(&pv_done[2 * s + h]);
                if (h) umma_commit(&v_empty[vr.slot]);
            }
            __syncwarp();
            if (h) vr.next(VS, vt);
            return true;
        };
        constexpr std::integral_constant<int, 0> c0{};
        constexpr std::integral_constant<int, 1> c1{};
        int left = min(end - j0 * TK, items * TK);  // tokens of this CTA's part from this item's first on
        uint32_t par = 0;
        bool ok = items > 0 && s < streams && issue_s(c0, true, 0, left) && (left <= 64 || issue_s(c1, true, 0, left - 64));
        for (int n = 0; n < items && ok && !given_up(); ++n, left -= TK, par ^= 1) {
            const bool first = n == 0;
            ok = issue_pv(c0, first, par, left) && (left <= TK || issue_s(c0, false, par ^ 1, left - TK));
            if (left > 64)
                ok = ok && issue_pv(c1, first, par, left - 64) &&
                     (left <= TK + 64 || issue_s(c1, false, par ^ 1, left - TK - 64));
        }
        if (issued) {  // MMAs retire before TMEM is released
            if (leader) umma_commit(&probe[s]);
            (void)mbar_wait_drain(&probe[s], 0);
        }
    } else if (warp <= NS + C::SOFT) {
        // ------------------------------------------------ softmax: thread = row
        const int s = (warp - 1 - NS) >> 2, q = warp & 3;
        const int r = q * 32 + lane;  // row within the stream == TMEM lane
        const int rr = r0 + 128 * s + r;
        const bool live = rr < rows, warp_live = r0 + 128 * s + q * 32 < rows;
        const int token = live ? rr / a.group : 0, head = kvh * a.group + (live ? rr - token * a.group : 0);
        const int vis = !live ? 0 : a.causal ? sq.past + token + 1 : sq.kv;  // tokens this row sees
        bool ok = s < streams;
        float qf = 0.f;
        if (ok) {
            // Q: the row's maximum to [128, 256), split in two e4m3 parts.  HD / 16 lanes share a row (16
            // values each), RPI rows at a time, the loads of up to eight such rounds in flight together.
            constexpr int LPR = HD / 16, RPI = 32 / LPR, IT = 32 / RPI < 8 ? 32 / RPI : 8;
            const int c = lane % LPR;
            const int row0 = q * 32 + lane / LPR;  // of this lane in the first round, within the stream
            const int first = r0 + 128 * s + row0;
            int tk = first / a.group, hd = first - tk * a.group;  // of the round's row; RPI rows on each round
            const int tk_up = RPI / a.group, hd_up = RPI - tk_up * a.group;
            uint8_t *hi = sQ + s * 2 * C::KT, *lo = hi + C::KT;
#pragma unroll 1
            for (int i0 = 0; i0 < 32 / RPI; i0 += IT) {
                uint4 u[IT][2];
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    u[i][0] = u[i][1] = make_uint4(0, 0, 0, 0);
                    if (first + (i0 + i) * RPI < rows) {
                        const __nv_bfloat16 *p =
                            a.qkv + (sq.t0 + tk) * a.row + static_cast<int64_t>(kvh * a.group + hd) * HD + 16 * c;
                        u[i][0] = *reinterpret_cast<const uint4 *>(p);
                        u[i][1] = *reinterpret_cast<const uint4 *>(p + 8);
                    }
                    tk += tk_up;
                    hd += hd_up;
                    if (hd >= a.group) hd -= a.group, ++tk;
                }
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    uint32_t w[8] = {u[i][0].x, u[i][0].y, u[i][0].z, u[i][0].w, u[i][1].x, u[i][1].y, u[i][1].z, u[i][1].w};
                    uint32_t m2 = 0;  // of |q| as bf16 bits, both halves: their order is that of the values
#pragma unroll
                    for (int j = 0; j < 8; ++j) m2 = __vmaxu2(m2, w[j] & 0x7fff7fffu);
                    uint32_t m = max(m2 & 0xffffu, m2 >> 16);
#pragma unroll
                    for (int d = 1; d < LPR; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
                    if (__any_sync(0xffffffffu, m >= 0x7f80u)) {  // infinities and NaN: as NaN, the maximum without them
                        m = 0;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if ((w[j] & 0x7f80u) == 0x7f80u) w[j] |= 0x7fffu;
                            else m = max(m, w[j] & 0x7fffu);
                            if ((w[j] & 0x7f800000u) == 0x7f800000u) w[j] |= 0x7fff0000u;
                            else m = max(m, (w[j] >> 16) & 0x7fffu);
                        }
#pragma unroll
                        for (int d = 1; d < LPR; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
                    }
                    // q 2^-e has its maximum in [128, 256); 2^e is a normal number, so in less below 2^-119
                    const int e = max(-126, static_cast<int>(m >> 7) - 127 - 7);
                    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                    // a negative softmax scale turns Q's signs, so that the logit factor is never negative
                    const float sign = a.scale_log2 < 0.f ? -down : down;
                    const int mine = __shfl_sync(0xffffffffu, e, lane % RPI * LPR);  // row (i0 + i) RPI + lane % RPI
                    if (lane / RPI == i0 + i)
                        qf = fabsf(a.scale_log2) * __uint_as_float(static_cast<uint32_t>(127 + mine) << 23);
                    uint32_t h[4], l[4];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t top = w[j] & 0xfff0fff0u;  // sign, exponent, three mantissa bits
                        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&w[j]),
                                                         *reinterpret_cast<const __nv_bfloat162 *>(&top));  // exact
                        const uint32_t h2 = scaled_codes(top, sign);
                        const uint32_t l2 = scaled_codes(*reinterpret_cast<const uint32_t *>(&d), sign);
                        h[j >> 1] = j & 1 ? h[j >> 1] | (h2 << 16) : h2;
                        l[j >> 1] = j & 1 ? l[j >> 1] | (l2 << 16) : l2;
                    }
                    const uint32_t at = tile_offset<HD>(row0 + (i0 + i) * RPI, c);
                    *reinterpret_cast<uint4 *>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
                }
            }
            fence_proxy_async_smem();
        }
        tmem = meet();
        const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
        const uint32_t tO = tmem + lanes + 256 + s * HD;
        const int vis_all = __reduce_min_sync(0xffffffffu, vis);  // what every row of the warp sees
        float m_run = -INFINITY, l_run = 0.f;
        float n_run = -INFINITY;  // the sum's reference once the scales are spread, m_run - log2 sv0 before
        bool spread = false;
        for (int k = 0; k < steps && ok; ++k) {  // 64 tokens at a time, from registers
            const int n = k >> 1, h = k & 1, c0 = 64 * h;
            const uint32_t tS = tmem + lanes + s * 128 + 64 * h;
            if (!(ok = wait(&s_full[slot_of(s, k)], phase_of(k)))) break;
            tc_fence_after();
            // The item's scales need no barrier of their own (226 us with one, 220 without): the producer wrote
            // them before its arrival for K, which the issuer saw before it committed S.
            if (h == 0 && !spread && ent[(n % kEnt) * 8].w != 0.f) {
                spread = true;
                n_run = m_run - ent[(n % kEnt) * 8 + 1].w;
            }
            const float4 *en = ent + (n % kEnt) * 8 + (c0 >> 4);
            const int lim = vis - (j0 + n) * TK - c0;  // columns of the step that the row sees
            float alpha = 1.f;
            bool raised = false;  // by a row of the warp
            if (warp_live) {
                uint32_t v[64];
                tmem_ld_x32(tS, *reinterpret_cast<uint32_t(*)[32]>(v));
                tmem_ld_x32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(v + 32));
                tmem_wait_ld_regs(*reinterpret_cast<uint32_t(*)[32]>(v));
                tmem_wait_ld_regs(*reinterpret_cast<uint32_t(*)[32]>(v + 32));
                if (vis_all - (j0 + n) * TK - c0 < 64) {  // some row of the warp sees less
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (i >= lim) v[i] = 0xff800000u;  // -inf
                }
                float top = -INFINITY, f[4], g[4], z[4];
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    const float4 e = en[i4];
                    // never 0, so that masked logits stay -inf (page scales of 0 have codes of 0)
                    f[i4] = fmaxf(qf * e.x, 1e-30f);
                    g[i4] = e.y;
                    z[i4] = e.z;
                    const uint32_t *w = v + 16 * i4;
                    float m0 = __uint_as_float(w[0]), m1 = __uint_as_float(w[1]);
#pragma unroll
                    for (int i = 2; i < 14; i += 4) {
                        m0 = max3f(m0, __uint_as_float(w[i]), __uint_as_float(w[i + 1]));
                        m1 = max3f(m1, __uint_as_float(w[i + 2]), __uint_as_float(w[i + 3]));
                    }
                    m0 = max3f(m0, __uint_as_float(w[14]), __uint_as_float(w[15]));
                    top = fmaxf(top, fmaf(fmaxf(m0, m1), f[i4], g[i4]));
                }
                // The reference rises only when a step exceeds it by more than 2^8: from -inf with the first token
                // that the row sees.  (Rows that see none, behind the sequence's last, must not raise: the warp
                // would wait for PV and pass over O at every step.  16 prompts of 301 tokens after 700, 602 rows
                // a head: 77.7 us so, 82.6 when they did.)
                raised = __any_sync(0xffffffffu, top > m_run + kLazy);
                if (top > m_run + kLazy) {
                    alpha = exp2_fast(m_run - top);
                    m_run = top;
                }
                const float shift = m_run == -INFINITY ? 0.f : kBoost - m_run;
                float sum = 0.f, sum_alpha = alpha;
                if (spread) {  // the sum's terms from their own exponentials
                    float sum_top = -INFINITY;
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4)
                        if (z[i4] != 0.f)
#pragma unroll
                            for (int i = 0; i < 16; ++i) sum_top = fmaxf(sum_top, __uint_as_float(v[16 * i4 + i]) * f[i4]);
                    sum_alpha = 1.f;
                    if (sum_top > n_run + kLazy) {
                        sum_alpha = exp2_fast(n_run - sum_top);
                        n_run = sum_top;
                    }
                    const float sum_shift = n_run == -INFINITY ? 0.f : kBoost - n_run;
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4)
                        if (z[i4] != 0.f)
#pragma unroll
                            for (int i = 0; i < 16; ++i) sum += exp2_fast(fmaf(__uint_as_float(v[16 * i4 + i]), f[i4], sum_shift));
                }
                uint32_t pk[32];
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    const uint32_t *w = v + 16 * i4;
                    const float gk = g[i4] + shift;
                    float s0 = 0.f, s1 = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float p0, p1;
                        fma_f32x2(p0, p1, __uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]), f[i4], gk);
                        p0 = exp2_fast(p0);
                        p1 = exp2_fast(p1);
                        add_f32x2(s0, s1, p0, p1);
                        pk[8 * i4 + i] = pack_f16x2(p0, p1);
                    }
                    if (!spread) sum = fmaf(s0 + s1, z[i4], sum);
                }
                __syncwarp();
                tmem_st_x32(tS, pk);
                l_run = fmaf(l_run, sum_alpha, sum);
                tmem_wait_st();
            }
            // O *= alpha after the previous step's PV and before this one's
            if (raised && k > 0) {
                if (!(ok = wait(&pv_done[slot_of(s, k - 1)], phase_of(k - 1)))) break;
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
            if (lane == 0) mbar_arrive(&p_full[slot_of(s, k)]);
        }
        if (ok && steps > 0) ok = wait(&pv_done[slot_of(s, steps - 1)], phase_of(steps - 1));
        tc_fence_after();
        if (ok && warp_live) {
            // A row that sees no token of this part (its pages are out of the pool) has seen zeros, with a
            // non-finite query NaN: it ends as it began.
            bool sees = false;
            if (items > 0) {
                const float4 *last = ent + ((items - 1) % kEnt) * 8;
                sees = vis > __float_as_int(last[2].w);
                if (!spread) n_run = m_run - last[1].w;
            }
            if (!sees) m_run = n_run = -INFINITY, l_run = 0.f;
            if (a.splits > 1) {
                const int64_t at = ((static_cast<int64_t>(sq.t0) + token) * a.q_heads + head) * a.splits + split;
                if (live) *reinterpret_cast<float4 *>(a.part_mn + at * 4) = make_float4(m_run - kBoost, n_run - kBoost, l_run, 0.f);
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t v[32];
                    if (items > 0) {
                        tmem_ld_x32(tO + c, v);
                        tmem_wait_ld_regs(v);
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = sees ? v[i] : 0;
                    if (live) {
                        float4 *dst = reinterpret_cast<float4 *>(a.part_o + at * HD + c);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            dst[i] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                                 __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
                    }
                    __syncwarp();
                }
            } else {
                // Rows leave through this warp's share of Q's shared memory (every S that reads it is
                // done), so that whole rows are stored side by side: a lane a row would be 32 lines
                // an instruction.  16-byte chunks are permuted by the row against bank conflicts.
                const RowFactor f = row_factor(m_run, n_run, l_run);
                uint8_t *rowbuf = sQ + (s * 2 * C::KT) + q * (32 * HD * 2);
                constexpr int CH = HD / 8;  // 16-byte chunks of a row
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t v[32];
                    tmem_ld_x32(tO + c, v);
                    tmem_wait_ld_regs(v);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = sees ? v[i] : 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t o[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            o[j] = pack_bf16x2(f(__uint_as_float(v[8 * i + 2 * j])), f(__uint_as_float(v[8 * i + 2 * j + 1])));
                        *reinterpret_cast<uint4 *>(rowbuf + lane * (HD * 2) + (((c / 8 + i) ^ (lane & 7)) << 4)) =
                            make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
                __syncwarp();
                const int first = r0 + 128 * s + q * 32, count = min(32, rows - first);
                for (int x = lane; x < count * CH; x += 32) {
                    const int row = x / CH, ch = x % CH, tk = (first + row) / a.group;
                    const int64_t orow = (static_cast<int64_t>(sq.t0) + tk) * a.q_heads + kvh * a.group + first + row - tk * a.group;
                    *reinterpret_cast<uint4 *>(a.out + orow * HD + 8 * ch) =
                        *reinterpret_cast<const uint4 *>(rowbuf + row * (HD * 2) + ((ch ^ (row & 7)) << 4));
                }
            }
        }
    } else {
        // ------------------------------------------------ V converters
        tmem = meet();
        const int t = threadIdx.x - 32 * (1 + NS + C::SOFT);
        constexpr int CPR = HD / 16;  // 16-code chunks per row
        for (int n = 0; n < items && !given_up(); ++n) {
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

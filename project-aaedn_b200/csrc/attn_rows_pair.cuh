// attn_rows_pair.cuh — the attention of attn_rows_tc.cuh for head_dim 65..128
// with two SMs on a tile: a cluster of two CTAs, 256 query rows (128 each)
// against the same keys, tcgen05.mma over the pair (cta_group::2, M 256).
//
// What bounds the single-SM kernel at this head_dim is turning K and V from
// fp32 into their fp16 parts (and the shared memory traffic of that), once
// per 128 rows. Here each CTA converts half: the pair's MMA takes half of
// its B operand from either CTA's shared memory, so CTA r holds keys 32 r ..
// 32 r + 31 of K (B's rows for S = Q K^T) and dims 64 r .. 64 r + 63 of V
// (B's rows for O += P V), 16 KB a unit each. K and V have their own rings
// and their own converting warps, so the two conversions of a unit overlap.
// The scale of K is per 32 keys and that of V per 64 dims (the two O halves);
// the CTAs write them into each other's shared memory. Everything that
// belongs to rows (softmax, output sums, queries) is per CTA as before.
//
// The first CTA's warp 1 issues the MMAs of both; its barriers count the
// arrivals of both CTAs, and its commits arrive on both CTAs' barriers.
//
// On a B200, calls in a burst (at the 1000 W limit the long ones take up to 15 %
// more): one prompt of 4096 tokens, 64 query heads over 8, 816 us (three
// MMAs of full rate a product would be 490, one 163); eight sequences of 4120
// new tokens in all, 32 heads over 8, 198 us; 2048 tokens, 32 heads, 149 us; a
// tree of 16 nodes over 4001 cached tokens, 32 heads over 8, 34 us; sixteen
// trees of 1 to 63 nodes over 0 to 4032, 64 heads, 134 us. A unit takes about
// 3000 clocks, its MMAs 1536: P V waits for the weights of both CTAs, the
// output sums for P V, the next P V for them, and softmax and each conversion,
// one warp a scheduler, take about 2500 clocks of latencies a unit themselves
// (the ragged case: tensor pipe 40 % active, issue slots 49 %, HBM 13 %). With all
// of that arithmetic cut out the handshakes and MMAs alone took 573 us of what
// was 800 then. Tried and slower, from that 800: two units
// as one group through softmax, P V and sums (844 us: the conversions spill),
// the maximum kept from earlier units instead of a first pass over the scores
// (836), 64 scores in registers (900), one more pair of score buffers in the
// place of the second Q buffer (equal).
#pragma once

#include <cuda.h> // CUtensorMap

#include "attn_rows_tc.cuh"

namespace aaedn_dev
{

constexpr int RP_HDP = 128, RP_NS = 4;   // stages of K, and of V
constexpr uint32_t RP_STAGE = 16384;     // 32 keys x 128 dims, or 64 keys x 64 dims, of 4 bytes
constexpr uint32_t RP_Q_ROW = RP_HDP * 4u + 16u;
constexpr uint32_t RP_T_QLO = 64; // Q's low parts behind its high parts, in tensor memory columns
constexpr size_t RP_SMEM = 2 * RP_NS * (size_t)RP_STAGE + 128 * RP_Q_ROW + 1024; // + alignment slack

// What a CTA's converting warps say of their part of a unit; the other CTA's
// entry is written by it (rp_st_async).
struct RpKInfo
{
    float down;   // what undoes the scaling of K's 32 keys
    uint32_t bad; // keys with a non-finite value
};
struct RpVInfo
{
    float down; // of V's 64 dims
    int unused;
    uint32_t bad[2];
};
constexpr int RP_INFO = 8; // twice the stages: an entry is overwritten when its unit's sums are done

struct RpShared
{
    uint64_t raw[2][RP_NS], conv[2][RP_NS], free_[2][RP_NS]; // K, V stages: copied, converted, read by the MMAs
    uint64_t s_full[2], p_full[2], o_full, o_empty, q_raw[4], q_full[2], q_empty[2], done;
    uint32_t tmem, abort;
    RtStart start, end;
    int stage_valid[2][RP_NS];
    alignas(16) uint32_t wmax[2][2][4];
    uint32_t bad[2][2][2];
    uint64_t info[2][RP_INFO]; // the other CTA's entries have arrived
    alignas(16) RpKInfo kinfo[RP_INFO][2];
    RpVInfo vinfo[RP_INFO][2];
    int valid[RP_INFO]; // keys of the unit that exist
    float alpha[4][128];
    float q_down[4][128]; // what undoes an item's rows' scaling of Q
    uint64_t seen[4][128]; // which of a unit's keys a row attends
    float2 stats[4][128]; // (sum, offset) of an item's rows
    float lo[4][128]; // and the second part of a far offset
};

// ---- the pair -------------------------------------------------------------------
__device__ __forceinline__ uint32_t rp_cta_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
// the address of `laddr` (this CTA's shared memory) in CTA `rank`'s
__device__ __forceinline__ uint32_t rp_peer(uint32_t laddr, uint32_t rank)
{
    uint32_t ra;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(laddr), "r"(rank));
    return ra;
}
__device__ __forceinline__ void rp_st32(uint32_t addr, uint32_t v)
{
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void rp_arrive(uint32_t addr)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// 8 bytes into the other CTA's shared memory, counted on its barrier there
__device__ __forceinline__ void rp_st_async(uint32_t addr, uint32_t x, uint32_t y, uint32_t bar)
{
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.u32 [%0], {%1, %2}, [%3];" ::"r"(addr), "r"(x),
                 "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void rp_tma_2d(uint32_t dst, const void* map, int x, int y, uint32_t mbar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
                 "[%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(mbar)
                 : "memory");
}
__device__ __forceinline__ void rp_mma(uint32_t d, uint32_t a, uint32_t desc_lo, uint32_t desc_hi, uint32_t idesc,
                                       uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 desc;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 desc, {%2, %3};\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], desc, %4, p;\n\t}" ::"r"(d),
                 "r"(a), "r"(desc_lo), "r"(desc_hi), "r"(idesc), "r"(acc)
                 : "memory");
}
// arrives on the barrier at this offset in both CTAs
__device__ __forceinline__ void rp_commit(uint32_t mbar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     mbar),
                 "h"((uint16_t)3)
                 : "memory");
}
// rt_idesc with M = 256
__host__ __device__ constexpr uint32_t rp_idesc(int n, bool b_mn)
{
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((256u >> 4) << 24);
}

// ---------------------------------------------------------------------------
template <bool TREE>
__global__ void __launch_bounds__(RT_THREADS, 1)
    attn_rows_pair_kernel(const AttnRowsArgs a, unsigned* err, const __grid_constant__ CUtensorMap kmap,
                          const __grid_constant__ CUtensorMap vmap)
{
    constexpr int HDP = RP_HDP;
    extern __shared__ __align__(16) uint8_t rt_raw[];
    __shared__ RpShared sm;
    const uint32_t ring = (smem_addr(rt_raw) + 1023u) & ~1023u; // the swizzle works on address bits
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.n_heads / a.n_kv, R = 128 / G, R2 = 2 * R, hd = a.head_dim; // rows of both CTAs: 2 R tokens
    const uint32_t rank = rp_cta_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    volatile uint32_t* abort = &sm.abort;

    // stage s of kind 0 (K) or 1 (V)
    auto stage_at = [&](int kind, uint32_t s) { return ring + ((uint32_t)kind * RP_NS + s) * RP_STAGE; };
    auto fail = [&]() {
        *abort = 1u;
        rp_st32(rp_peer(smem_addr(&sm.abort), rank ^ 1u), 1u);
        atomicExch(err, 1u);
    };
    // false: the role ends (and says so in `failed`), and with it all others
    auto wait = [&](uint32_t bar, uint32_t parity) -> bool { return rt_wait(bar, parity, abort); };
    // the first CTA's barrier: its MMA warp waits for both CTAs
    auto lead = [&](const uint64_t* bar) { return rp_peer(smem_addr(bar), 0u); };
    bool failed = false;

    if (warp == 0)
    {
        const RtStart st = rt_locate<TREE>(a, R2, pair, pairs);
        if (lane == 0)
        {
            sm.start = st;
            if (rank == 0)
                reinterpret_cast<RtStart*>(a.workspace)[pair] = st;
        }
    }
    else if (warp == 3)
    {
        const RtStart en = rt_locate<TREE>(a, R2, pair + 1, pairs);
        if (lane == 0)
        {
            sm.end = en;
            if (rank == 0 && pair + 1 == pairs)
                reinterpret_cast<RtStart*>(a.workspace)[pairs] = en;
        }
    }
    else if (warp == 1)
    {
        if (lane == 0)
        {
            for (int k = 0; k < 2; ++k)
                for (int i = 0; i < RP_NS; ++i)
                {
                    mbar_init(smem_addr(&sm.raw[k][i]), 1);
                    mbar_init(smem_addr(&sm.conv[k][i]), 8); // four warps of each CTA
                    mbar_init(smem_addr(&sm.free_[k][i]), 1);
                }
            for (int i = 0; i < RP_INFO; ++i)
            {
                mbar_init(smem_addr(&sm.info[0][i]), 1);
                mbar_init(smem_addr(&sm.info[1][i]), 1);
            }
            for (int i = 0; i < 2; ++i)
            {
                mbar_init(smem_addr(&sm.s_full[i]), 1);
                mbar_init(smem_addr(&sm.p_full[i]), 8);
                mbar_init(smem_addr(&sm.q_full[i]), 8);
                mbar_init(smem_addr(&sm.q_empty[i]), 1);
            }
            for (int i = 0; i < 4; ++i)
                mbar_init(smem_addr(&sm.q_raw[i]), 1);
            mbar_init(smem_addr(&sm.o_full), 1);
            mbar_init(smem_addr(&sm.o_empty), 16);
            mbar_init(smem_addr(&sm.done), 1);
            mbar_init_fence();
            sm.abort = 0u;
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sm.tmem)),
                     "r"(RT_T_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    else if (warp == 2 && lane < 8)
        (&sm.bad[0][0][0])[lane] = 0u;
    rt_fence_before();
    __syncthreads();
    cluster_sync_all(); // the other CTA's barriers are ready
    rt_fence_after();
    constexpr uint32_t tmem = 0u; // all columns are the CTA's
    const RtStart st0 = sm.start;
    unsigned long long share = sm.end.begin - st0.begin;
    if (sm.tmem != tmem) // cannot be: nothing runs on other columns
    {
        share = 0;
        fail();
    }
    // wait() for a whole warp: its lanes go on, or give up, together
    auto wait_all = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait(bar, parity)); };

    if (warp < 4)
    {
        rt_regs_dec<RT_REGS_IO>();
        if (warp == 0 || warp == 2)
        {
            // ---- producers: warp 0 this CTA's keys of K, warp 2 its dims of V
            const int kind = warp >> 1;
            const CUtensorMap* map = kind ? &vmap : &kmap;
            uint32_t slot = 0, ph = 1, n = 0; // a new barrier's phase before the first counts as done
            bool ok = true;
            RtCursor<TREE> c;
            for (bool more = c.start(a, st0, share, R2); more && ok; more = c.next(a, R2))
            {
                const int* pt = rows_page_table(a, c.s);
                int mine = 0;
                for (int u = c.u0; u < c.u1 && ok; ++u, ++n)
                {
                    const int k = (u - c.u0) & 31;
                    if (k == 0) // the next 32 page numbers, one a lane
                        mine = u + lane < c.u1 ? __ldg(pt + u + lane) : 0;
                    const int page = __shfl_sync(0xffffffffu, mine, k);
                    ok = wait_all(smem_addr(&sm.free_[kind][slot]), ph);
                    if (ok && lane == 0)
                    {
                        // a page outside the pool is a unit without keys
                        const bool there = page >= 0 && page < a.n_pages;
                        const uint32_t bar = smem_addr(&sm.raw[kind][slot]);
                        sm.stage_valid[kind][slot] = there ? min(64, c.keys - u * 64) : 0;
                        if (there)
                        {
                            const int row = (page * a.n_kv + c.h) * ROWS_PAGE;
                            mbar_arrive_expect_tx(bar, RP_STAGE);
                            rp_tma_2d(stage_at(kind, slot), map, kind ? (int)rank * 64 : 0, kind ? row : row + (int)rank * 32,
                                      bar);
                        }
                        else
                            mbar_arrive(bar);
                    }
                    if (ok && ++slot == RP_NS)
                    {
                        slot = 0;
                        ph ^= 1u;
                    }
                }
            }
            failed = !ok;
            // the copies it issued have landed before the CTA may exit
            if (lane == 0)
                for (uint32_t p = n > RP_NS ? n - RP_NS : 0; p < n; ++p)
                    mbar_wait_bounded(smem_addr(&sm.raw[kind][p % RP_NS]), (p / RP_NS) & 1u, RT_WAIT_LIMIT_NS);
            __syncwarp();
        }
        else if (warp == 1 && rank == 0)
        {
            // ---- MMA issuer of both CTAs: the warp walks the units, one lane issues
            constexpr uint32_t id_qk = rp_idesc(64, false), id_pv = rp_idesc(HDP, true);
            uint32_t g = 0, item = 0, k_slot = 0, k_ph = 0, v_slot = 0, v_ph = 0;
            RtCursor<TREE> c;
            bool more = c.start(a, st0, share, R2), ok = true;
            int u = more ? c.u0 : 0;
            while (ok)
            {
                if (more)
                {
                    const uint32_t qb = item & 1u;
                    if ((u == c.u0 && !wait_all(smem_addr(&sm.q_full[qb]), (item >> 1) & 1u)) ||
                        !wait_all(smem_addr(&sm.conv[0][k_slot]), k_ph))
                    {
                        ok = false;
                        break;
                    }
                    rt_fence_after();
                    const uint32_t k_hi = rt_desc_lo(stage_at(0, k_slot), 16u), d = RT_T_S + (g & 1u) * 64u;
                    const bool last = u + 1 == c.u1;
                    if (rt_elect())
                    {
#pragma unroll 1
                        for (uint32_t p = 0; p < 3; ++p) // q_hi k_lo, q_lo k_hi, q_hi k_hi
                        {
                            const uint32_t q = RT_T_Q + qb * 128u + (p == 1 ? RP_T_QLO : 0u), k = k_hi + (p == 0 ? 512u : 0u);
#pragma unroll
                            for (uint32_t n = 0; n < HDP / 16; ++n)
                                rp_mma(d, q + n * 8u, k + (n >> 2) * 256u + (n & 3u) * 2u, RT_DESC_HI, id_qk, p | n);
                        }
                        rp_commit(smem_addr(&sm.s_full[g & 1u]));
                        rp_commit(smem_addr(&sm.free_[0][k_slot]));
                        if (last)
                            rp_commit(smem_addr(&sm.q_empty[qb]));
                    }
                    __syncwarp();
                    if (++k_slot == RP_NS)
                    {
                        k_slot = 0;
                        k_ph ^= 1u;
                    }
                }
                if (g > 0) // P V of the unit before
                {
                    const uint32_t j = g - 1u;
                    if (!wait_all(smem_addr(&sm.conv[1][v_slot]), v_ph) ||
                        !wait_all(smem_addr(&sm.p_full[j & 1u]), (j >> 1) & 1u) ||
                        (j >= 1u && !wait_all(smem_addr(&sm.o_empty), (j - 1u) & 1u)))
                    {
                        ok = false;
                        break;
                    }
                    rt_fence_after();
                    const uint32_t v_hi = rt_desc_lo(stage_at(1, v_slot), 8192u), ph = RT_T_S + (j & 1u) * 64u;
                    if (rt_elect())
                    {
#pragma unroll 1
                        for (uint32_t p = 0; p < 3; ++p) // p_hi v_lo, p_lo v_hi, p_hi v_hi
                        {
                            const uint32_t w = ph + (p == 1 ? 8u : 0u), v = v_hi + (p == 0 ? 512u : 0u);
#pragma unroll
                            for (uint32_t n = 0; n < 4; ++n)
                                rp_mma(RT_T_O, w + n * 16u, v + n * 128u, RT_DESC_HI, id_pv, p | n);
                        }
                        rp_commit(smem_addr(&sm.o_full));
                        rp_commit(smem_addr(&sm.free_[1][v_slot]));
                    }
                    __syncwarp();
                    if (++v_slot == RP_NS)
                    {
                        v_slot = 0;
                        v_ph ^= 1u;
                    }
                }
                if (!more)
                    break;
                ++g;
                if (++u >= c.u1)
                {
                    more = c.next(a, R2);
                    u = c.u0;
                    ++item;
                }
            }
            failed = !ok;
            if (rt_elect())
                rp_commit(smem_addr(&sm.done)); // every MMA issued, whatever happened
            __syncwarp();
        }
    }
    else if (warp < RT_W_O)
    {
        // ---- softmax: thread = row
        rt_regs_inc<RT_REGS_SM>();
        const int i = (warp & 3) * 32 + lane, ti = i / G;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        constexpr float LOG2E = 1.4426950408889634f;
        const float qs = fabsf(a.scale) * LOG2E;
        uint32_t g = 0, item = 0;
        bool ok = true;
        RtCursor<TREE> c;
        for (bool more = c.start(a, st0, share, R2); more && ok; more = c.next(a, R2), ++item)
        {
            const int r = (2 * c.t + (int)rank) * R + ti;
            const bool live = ti < R && r < c.q.n;
            const bool any = __any_sync(0xffffffffu, live); // a warp without rows computes nothing
            float qf = 0.0f;
            const int limit = TREE ? c.q.past : min(c.q.past, INT_MAX - c.q.n) + r; // past + r: far behind cap when clamped
            const uint64_t* mask = TREE ? a.mask + (size_t)(c.q.begin + (live ? r : 0)) * a.mask_words : nullptr;
            // weights are held as exp2(s + off) = 2^14 exp(score - max); a far offset
            // has a second part in sm.lo
            float off = INFINITY, l = 0.0f;
            bool bad = false;
            for (int u = c.u0; u < c.u1; ++u, ++g)
            {
                const uint32_t b = g & 1u;
                if (!wait_all(smem_addr(&sm.s_full[b]), (g >> 1) & 1u) ||
                    !wait_all(smem_addr(&sm.info[0][g % RP_INFO]), (g / RP_INFO) & 1u))
                {
                    ok = false;
                    break;
                }
                if (!any)
                {
                    if (lane == 0)
                        rp_arrive(lead(&sm.p_full[b]));
                    continue;
                }
                rt_fence_after();
                const uint32_t ts = tmem + lanes + RT_T_S + b * 64u;
                if (u == c.u0)
                    qf = qs * sm.q_down[item & 3u][i];
                // keys 0..31 and 32..63 were scaled by the two CTAs
                const uint4 in = *reinterpret_cast<const uint4*>(sm.kinfo[g % RP_INFO]); // (down, bad) twice
                float fa = rt_score_scale(qf * __uint_as_float(in.x));
                float fb = rt_score_scale(qf * __uint_as_float(in.z));
                const uint64_t seen = live ? rt_seen<TREE>(u, sm.valid[g % RP_INFO], limit, mask, a.mask_words) : 0ull;
                sm.seen[g & 3u][i] = seen;
                if ((in.y | in.w) != 0u && (seen & ((uint64_t)in.y | (uint64_t)in.w << 32)) != 0ull)
                    bad = true;
                const bool all = __all_sync(0xffffffffu, seen == ~0ull);
                // 16 keys at a time, twice: the largest score, then the weights (P takes
                // the place of S). Rolled loops over tensor memory: with all 64
                // scores in registers a unit alone is faster, the kernel 13 % slower
                // (its roles' code no longer fits the instruction caches).
                float s[16], top = -INFINITY;
#pragma unroll 1
                for (uint32_t j0 = 0; j0 < 64; j0 += 16)
                {
                    rt_ld<16>(ts + j0, s);
                    if (!all)
                        rt_mask16(s, (uint32_t)(seen >> j0));
                    top = fmaxf(top, rt_max16(s) * (j0 < 32 ? fa : fb));
                }
                const float noff = fminf(off, 14.0f - top);
                float use = noff < INFINITY ? noff : 0.0f, corr = use - off;
                if (__any_sync(0xffffffffu, fabsf(use) > RT_FAR || rt_far(off)))
                {
                    const bool far = fabsf(use) > RT_FAR;
                    const float2 r = rt_far_unit(ts, seen, far ? fa : 1.0f, far ? fb : 1.0f, far ? use : 0.0f, off,
                                                 &sm.lo[item & 3u][i]);
                    corr += r.x;
                    if (far)
                    {
                        use = r.y;
                        fa = fb = 1.0f;
                    }
                    __syncwarp(); // together into the loads
                }
                corr = rt_exp2(corr); // 0 before the first key
                off = noff;
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll 1
                for (uint32_t j0 = 0; j0 < 64; j0 += 16)
                {
                    rt_ld<16>(ts + j0, s);
                    if (!all)
                        rt_mask16(s, (uint32_t)(seen >> j0));
                    sum = rt_add2(sum, rt_weights(s, j0 < 32 ? fa : fb, use, ts + j0));
                }
                l = fmaf(l, corr, sum.x + sum.y);
                sm.alpha[g & 3u][i] = corr;
                if (u + 1 == c.u1)
                    sm.stats[item & 3u][i] = make_float2(bad ? __uint_as_float(0x7FC00000u) : l, off);
                rt_wait_st();
                rt_fence_before();
                __syncwarp();
                if (lane == 0)
                    rp_arrive(lead(&sm.p_full[b]));
            }
        }
        failed = !ok;
    }
    else if (warp < RT_W_CV)
    {
        // ---- output sums: thread = row, a warpgroup for each half of the dims
        rt_regs_inc<RT_REGS_O>();
        constexpr int W = HDP / 2;
        const int i = (warp & 3) * 32 + lane, half = (warp - RT_W_O) >> 2, d_first = half * W;
        const uint32_t t_o = tmem + ((uint32_t)((warp & 3) * 32) << 16) + RT_T_O + d_first;
        uint32_t g = 0, item = 0;
        bool ok = true;
        RtCursor<TREE> c;
        for (bool more = c.start(a, st0, share, R2); more && ok; more = c.next(a, R2), ++item)
        {
            float acc[W]; // in units of `unit`, the largest scale of V that counts so far
#pragma unroll
            for (int d = 0; d < W; ++d)
                acc[d] = 0.0f;
            const bool any = __any_sync(0xffffffffu, rt_row_at(c.q, c.h, 2 * c.t + (int)rank, i, G, R, 0, 0) >= 0);
            float2 stat = make_float2(0.0f, INFINITY);
            float unit = 0.0f;
            bool bad = false;
            for (int u = c.u0; u < c.u1; ++u, ++g)
            {
                if (!wait_all(smem_addr(&sm.o_full), g & 1u) ||
                    !wait_all(smem_addr(&sm.info[1][g % RP_INFO]), (g / RP_INFO) & 1u))
                {
                    ok = false;
                    break;
                }
                if (!any)
                {
                    if (lane == 0)
                        rp_arrive(lead(&sm.o_empty));
                    continue;
                }
                rt_fence_after();
                float corr = sm.alpha[g & 3u][i];
                const RpVInfo* in = sm.vinfo[g % RP_INFO];
                const uint32_t bad0 = in[0].bad[0] | in[1].bad[0], bad1 = in[0].bad[1] | in[1].bad[1];
                if ((bad0 | bad1) != 0u)
                    bad |= (sm.seen[g & 3u][i] & ((uint64_t)bad0 | (uint64_t)bad1 << 32)) != 0ull;
                if (u + 1 == c.u1)
                    stat = sm.stats[item & 3u][i];
                const float f = in[half].down; // a power of two
                // exact, or an underflow of sums that no longer count; where the sums so far
                // count nothing, neither does their scale. By selects, and a vote: the loads
                // from tensor memory below are the whole warp's together.
                const bool over = f > unit, none = corr == 0.0f;
                corr = over ? corr * rt_ratio(unit, f) : corr;
                unit = over || none ? f : unit;
                const float2 c2 = make_float2(corr, corr);
                const float down = rt_ratio(f, unit);
                const bool scaled = __any_sync(0xffffffffu, down != 1.0f);
#pragma unroll
                for (int d0 = 0; d0 < W; d0 += 16)
                {
                    float t[16];
                    rt_ld<16>(t_o + d0, t);
                    if (scaled)
#pragma unroll
                        for (int d = 0; d < 16; ++d)
                            t[d] *= down;
#pragma unroll
                    for (int d = 0; d < 16; d += 2)
                    {
                        const float2 y = fma2_rn(make_float2(acc[d0 + d], acc[d0 + d + 1]), c2, make_float2(t[d], t[d + 1]));
                        acc[d0 + d] = y.x;
                        acc[d0 + d + 1] = y.y;
                    }
                }
                rt_fence_before();
                __syncwarp();
                if (lane == 0)
                    rp_arrive(lead(&sm.o_empty));
            }
            if (!ok)
                break;
            if (!any)
                continue;
            const float l = bad ? __uint_as_float(0x7FC00000u) : stat.x;
            // the row's mean, of a cut tile too: the sums of values near the largest fp32
            // pass it. In this order: 1 / l of the sums is at most 2^15, unit / l of small
            // values would be denormal.
            const float by = l == 0.0f ? 0.0f : 1.0f / l;
            float* to;
            int n = W; // dims to store
            if (c.whole)
            {
                const long long at = rt_row_at(c.q, c.h, 2 * c.t + (int)rank, i, G, R, a.ldo, hd);
                to = a.out + at + d_first;
                n = at < 0 ? 0 : hd - d_first;
            }
            else
            {
                float* slot = rt_slot<HDP>(a, blockIdx.x, item == 0 ? 0 : 1);
                to = slot + (size_t)i * HDP + d_first;
                if (d_first == 0)
                {
                    reinterpret_cast<float2*>(slot + 128 * HDP)[i] = make_float2(l, stat.y);
                    if (rt_far(stat.y))
                        slot[128 * HDP + 256 + i] = sm.lo[item & 3u][i];
                }
            }
            // a row a thread: whole 32-byte sectors where the addresses allow it
            if (((uint32_t)reinterpret_cast<uintptr_t>(to) & 31u) == 0u && (n & 7) == 0)
            {
#pragma unroll
                for (int d = 0; d < W; d += 8)
                    if (d < n)
                        rt_store8(to + d, acc + d, by, unit);
            }
            else
            {
#pragma unroll
                for (int d = 0; d < W; d += 4)
                    if (d < n)
                        *reinterpret_cast<float4*>(to + d) =
                            make_float4(acc[d] * by * unit, acc[d + 1] * by * unit, acc[d + 2] * by * unit, acc[d + 3] * by * unit);
            }
        }
        failed = !ok;
    }
    else if (warp < RT_W_Q)
    {
        // ---- a stage from fp32 to its fp16 parts, in place: warps 0-3 the K
        // stages (32 keys x 128 dims), warps 4-7 the V stages (64 keys x 64 dims)
        rt_regs_dec<RT_REGS_CV>();
        const int kind = (warp - RT_W_CV) >> 2, ct = tid - (RT_W_CV + 4 * kind) * 32, cw = ct >> 5;
        constexpr int NCH = RP_STAGE / 16 / 128; // 16-byte pieces a thread: piece n is number 128 n + ct of the stage
        const int per_row = kind ? 16 : 32, row0 = ct / per_row, col = ct % per_row, rows = 128 / per_row;
        const int key0 = kind ? 0 : (int)rank * 32; // key of the stage's first row
        // its place in the swizzled rows: 64-dim blocks of K are 4 KB apart; the
        // rows of odd pieces are 4 (K) or 8 (V) further in the swizzle
        const int e = (col & 15) * 4, sw = (e >> 3) ^ (row0 & 7);
        const uint32_t off = (uint32_t)(col >> 4) * 4096u + (uint32_t)row0 * 128u + (uint32_t)((e & 7) * 2);
        const uint32_t off0 = off + (uint32_t)sw * 16u, off1 = off + (uint32_t)(kind ? sw : sw ^ 4) * 16u;
        const uint32_t step = (uint32_t)rows * 128u;
        uint32_t slot = 0, ph = 0, par = 0;
        bool ok = true;
        for (uint32_t g = 0; g < (uint32_t)share; ++g)
        {
            const bool got = wait(smem_addr(&sm.raw[kind][slot]), ph);
            const uint32_t stage = stage_at(kind, slot);
            const int valid = got ? sm.stage_valid[kind][slot] : 0;
            float4 x[NCH];
            float mx = 0.0f, my = 0.0f; // NaN is kept
#pragma unroll
            for (int n = 0; n < NCH; ++n)
            {
                const uint4 w = lds128(stage + (uint32_t)(n * 128 + ct) * 16u);
                x[n] = make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
            }
            if (valid < 64)
            {
#pragma unroll
                for (int n = 0; n < NCH; ++n)
                    if (key0 + row0 + n * rows >= valid) // behind the last key
                        x[n] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int n = 0; n < NCH; ++n)
            {
                mx = rt_max_abs(mx, x[n].x, x[n].y);
                my = rt_max_abs(my, x[n].z, x[n].w);
            }
            mx = rt_max_abs(mx, my, 0.0f);
            if (!(mx < INFINITY))
            {
                // NaN or infinity: the key is noted and its values are zeros
                mx = 0.0f;
#pragma unroll
                for (int n = 0; n < NCH; ++n)
                {
                    if (!(rt_max_abs(0.0f, x[n]) < INFINITY))
                    {
                        const int row = row0 + n * rows;
                        atomicOr(&sm.bad[kind][par][row >> 5], 1u << (row & 31));
                        x[n] = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    mx = rt_max_abs(mx, x[n]);
                }
            }
            const uint32_t wm = __reduce_max_sync(0xffffffffu, __float_as_uint(mx)); // not negative: ordered as integers
            if (lane == 0)
                sm.wmax[kind][par][cw] = wm;
            // every read of the stage is done; a failed wait ends the four warps together
            if (named_bar_or(1 + kind, 128, !got))
            {
                ok = false;
                break;
            }
            const uint4 m = *reinterpret_cast<const uint4*>(&sm.wmax[kind][par][0]);
            float up, down;
            rt_scale_of(max(max(m.x, m.y), max(m.z, m.w)), up, down);
            if (ct == 0)
            {
                // both CTAs' softmax and output warps read them
                const uint32_t b0 = sm.bad[kind][par][0], b1 = sm.bad[kind][par][1];
                sm.bad[kind][par][0] = sm.bad[kind][par][1] = 0u; // next used two stages on
                const uint32_t bar = smem_addr(&sm.info[kind][g % RP_INFO]), there = rank ^ 1u;
                if (kind == 0)
                {
                    RpKInfo& in = sm.kinfo[g % RP_INFO][rank];
                    in.down = down;
                    in.bad = b0;
                    sm.valid[g % RP_INFO] = valid;
                    mbar_arrive_expect_tx(bar, 8u); // of the other CTA's entry
                    rp_st_async(rp_peer(smem_addr(&in), there), __float_as_uint(down), b0, rp_peer(bar, there));
                }
                else
                {
                    RpVInfo& in = sm.vinfo[g % RP_INFO][rank];
                    in.down = down;
                    in.bad[0] = b0;
                    in.bad[1] = b1;
                    mbar_arrive_expect_tx(bar, 16u);
                    rp_st_async(rp_peer(smem_addr(&in), there), __float_as_uint(down), 0u, rp_peer(bar, there));
                    rp_st_async(rp_peer(smem_addr(&in.bad[0]), there), b0, b1, rp_peer(bar, there));
                }
            }
            const float2 up2 = make_float2(up, up);
#pragma unroll
            for (int n = 0; n < NCH; ++n)
            {
                uint32_t h0, l0, h1, l1;
                const float2 a2 = mul2_rn(make_float2(x[n].x, x[n].y), up2), b2 = mul2_rn(make_float2(x[n].z, x[n].w), up2);
                rt_split2(a2.x, a2.y, h0, l0);
                rt_split2(b2.x, b2.y, h1, l1);
                const uint32_t at = stage + ((n & 1) ? off1 : off0) + (uint32_t)n * step;
                asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(h0), "r"(h1) : "memory");
                asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + 8192u), "r"(l0), "r"(l1) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the MMA reads through the async proxy
            __syncwarp();
            if (lane == 0)
                rp_arrive(lead(&sm.conv[kind][slot]));
            par ^= 1u;
            if (++slot == RP_NS)
            {
                slot = 0;
                ph ^= 1u;
            }
        }
        failed = !ok;
    }
    else
    {
        // ---- queries: bulk copies bring the next tile's rows to shared memory
        // while this one's go to tensor memory; thread = row
        rt_regs_dec<RT_REGS_Q>();
        const int w = warp & 3, i = w * 32 + lane;
        const uint32_t lanes = (uint32_t)(w * 32) << 16;
        const uint32_t row = ring + 2 * RP_NS * RP_STAGE + (uint32_t)i * RP_Q_ROW, raw = smem_addr(&sm.q_raw[w]);
        const float sign = a.scale < 0.0f ? -1.0f : 1.0f; // the softmax takes |scale|
        uint32_t item = 0;
        bool ok = true;
        RtCursor<TREE> c;
        auto copy = [&]() -> bool { // true: the row has a token
            const long long at = rt_row_at(c.q, c.h, 2 * c.t + (int)rank, i, G, R, a.ldq, hd);
            const uint32_t n = __popc(__ballot_sync(0xffffffffu, at >= 0));
            if (lane == 0)
                mbar_arrive_expect_tx(raw, n * (uint32_t)hd * 4u);
            __syncwarp();
            if (at >= 0)
                bulk_g2s(row, a.q + at, (uint32_t)hd * 4u, raw);
            return at >= 0;
        };
        bool more = c.start(a, st0, share, R2), live = more && copy();
        for (; more; ++item)
        {
            const uint32_t qb = item & 1u;
            if (!wait_all(raw, item & 1u) ||
                (item >= 2 && !wait_all(smem_addr(&sm.q_empty[qb]), ((item >> 1) & 1u) ^ 1u)))
            {
                ok = false;
                break;
            }
            rt_fence_after();
            float mx = 0.0f; // NaN is kept
            if (live)
#pragma unroll 4
                for (int d = 0; d < hd; d += 4)
                {
                    const uint4 x = lds128(row + (uint32_t)d * 4u);
                    mx = rt_max_abs(mx, make_float4(__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z),
                                                    __uint_as_float(x.w)));
                }
            float q_up, q_down;
            rt_scale_of(__float_as_uint(mx) & 0x7FFFFFFFu, q_up, q_down);
            q_up *= sign;
            sm.q_down[item & 3u][i] = q_down;
#pragma unroll 1
            for (int d0 = 0; d0 < HDP; d0 += 16)
            {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int d = 0; d < 4; ++d)
                {
                    uint4 x = make_uint4(0u, 0u, 0u, 0u);
                    if (live && d0 + d * 4 < hd)
                        x = lds128(row + (uint32_t)(d0 + d * 4) * 4u);
                    rt_split2(__uint_as_float(x.x) * q_up, __uint_as_float(x.y) * q_up, hi[2 * d], lo[2 * d]);
                    rt_split2(__uint_as_float(x.z) * q_up, __uint_as_float(x.w) * q_up, hi[2 * d + 1], lo[2 * d + 1]);
                }
                rt_st8(tmem + lanes + RT_T_Q + qb * 128u + d0 / 2, hi);
                rt_st8(tmem + lanes + RT_T_Q + qb * 128u + RP_T_QLO + d0 / 2, lo);
            }
            rt_wait_st();
            rt_fence_before();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the next copy overwrites what was read
            __syncwarp();
            if (lane == 0)
                rp_arrive(lead(&sm.q_full[qb]));
            more = c.next(a, R2);
            live = more && copy();
        }
        if (!ok) // a copy may be in flight: it has landed before the CTA exits
            mbar_wait_bounded(raw, item & 1u, RT_WAIT_LIMIT_NS);
        failed = !ok;
    }
    if (failed && lane == 0)
        fail();
    if (warp == 1 && lane == 0) // every MMA is done before the CTAs may leave
        mbar_wait_bounded(smem_addr(&sm.done), 0, RT_WAIT_LIMIT_NS);
    rt_fence_before();
    __syncthreads();
    cluster_sync_all(); // neither CTA reads, writes or signals the other's memory any more
    if (warp == 1)
    {
        rt_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(RT_T_COLS) : "memory");
    }
}

} // namespace aaedn_dev

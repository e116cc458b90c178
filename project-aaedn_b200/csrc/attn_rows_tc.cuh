// attn_rows_tc.cuh — attention of packed query rows over the paged fp32 K/V
// cache on the 5th-generation tensor cores: what the kernels for head_dim up to
// 64 (here) and 65..128 (attn_rows_pair.cuh) share, the first of them, and the
// joining kernel.
//
// Tile: 128 query rows that share a K/V head (128 / G tokens x the G query
// heads of the K/V head) against the keys in units of one page (64 tokens):
// S = Q K^T (M 128, N 64), online softmax, O += P V (M 128, N 64). The Q and P
// operands and the accumulators are in tensor memory, K and V in shared
// memory.
//
// Precision: the cache is fp32, the MMA takes 16-bit factors. A factor x is
// carried as x_hi + x_lo, both fp16, of x scaled by a power of two (q: per
// row, K and V: per unit, P: by 2^14) that puts the largest magnitude at
// 2^14..2^15: 22 significant bits for magnitudes down to 2^-17 of the
// largest, an absolute 2^-39 of it below (the low part is then subnormal). Each product is three MMAs (hi lo,
// lo hi, hi hi; lo lo is below 2^-22 of it), the small ones first, so that
// the tensor core's rounding of its accumulator (up to one unit per MMA)
// only counts for the hi hi ones. bf16 would need six products for this, and
// TF32 three at half the rate. P V accumulates one unit in tensor memory and
// is added to fp32 registers (one rounding a unit, with the softmax
// correction), because a long chain of tensor-core additions is biased
// towards zero: 2^-24 each.
//
// Work split: the units of all (sequence, K/V head, tile) in a row are cut
// into equal shares, one persistent CTA (or pair) each, so long prompts, many
// short ones and a small tree over a long cache all fill the GPU. A tile that
// a cut goes through is written as partial means (at most two a CTA) that a
// second kernel joins, in a fixed order: no atomics, the same bits every time.
//
// Roles (28 warps, 1 CTA an SM): warp 0 copies pages (bulk copies into a ring
// of stages), warp 1 issues the MMAs; warps 4-7 softmax (one row a thread:
// S from tensor memory, P back over it); warps 8-15 the output sums (a row and
// half of its dims a thread, in registers); warps 16-23 turn a stage from fp32
// into the two fp16 parts in place, in the 128-byte-swizzled layout the MMA
// reads (rows = keys: K-major for K, the same bytes are MN-major for V); warps
// 24-27 the queries, a tile ahead. Ring order is the MMA's: K0, K1, V0, K2,
// V1, ..., so S of the next unit is computed while the softmax of this one
// runs. The roles' loops are rolled where they can be: 28 warps run them side
// by side, and they are faster small enough for the instruction caches than
// they are unrolled.
//
// Keys that do not exist (behind the cached tokens, in a page outside the
// pool) are zeros that every row masks; a non-finite K or V row is replaced
// by zeros and noted, and the rows that attend it become NaN, so it cannot
// reach the other rows of the tile through 0 * NaN.
//
// Bound by the conversion of K and V and by the ways between the roles, not by
// the MMAs. On a B200 at head_dim 64 (32 query heads over 8), calls in a burst: a
// prompt of 2048 tokens 119 us, eight prompts of 4120 tokens together 174 us, a
// tree of 16 over 4001 cached tokens 27 us; four short sequences at head_dim 48
// 23 us, of which 16 us are the call's two launches.
#pragma once

#include "attn_rows.h"
#include "common.cuh"

namespace aaedn_dev
{

constexpr int RT_WARPS = 28, RT_THREADS = RT_WARPS * 32;
constexpr int RT_W_SM = 4, RT_W_O = 8, RT_W_CV = 16, RT_W_Q = 24; // first warps of the roles
constexpr int RT_CONV_THREADS = 256;
constexpr int RT_REGS = 72; // registers a thread at launch: 65536 / 896, whole eights
// the warpgroups' shares after setmaxnreg: together the launch's
constexpr int RT_REGS_IO = 40, RT_REGS_SM = 80, RT_REGS_O = 104, RT_REGS_CV = 64, RT_REGS_Q = 48;
static_assert(RT_REGS_IO + RT_REGS_SM + 2 * RT_REGS_O + 2 * RT_REGS_CV + RT_REGS_Q == 7 * RT_REGS, "register shares");
constexpr uint64_t RT_WAIT_LIMIT_NS = 2000000000ull;
constexpr int RT_INFO = 16; // units whose scales are kept

// tensor memory columns (the CTA allocates all of it, so its base is 0): S and
// P of two units, O of one, Q of two tiles (high parts, then low parts)
constexpr uint32_t RT_T_S = 0, RT_T_O = 128, RT_T_Q = 256, RT_T_QLO = 32, RT_T_COLS = 512;

// The kernel here: head_dim padded to 64.
constexpr int RT_HDP = 64, RT_NS = 8; // stages of one page of K or V
constexpr uint32_t RT_STAGE = 64u * RT_HDP * 4u;
constexpr uint32_t RT_Q_ROW = RT_HDP * 4u + 16u; // a query row in shared memory: no bank conflicts across rows
constexpr size_t RT_SMEM = (size_t)RT_NS * RT_STAGE + 128 * RT_Q_ROW + 1024; // + alignment slack

// ---- the split of the work ----------------------------------------------------
// sum over i < n of floor((a i + b) / 64), 0 < a: the numerators' sum less that of
// their remainders. Those repeat with the period 64 / g, g = gcd(a, 64), and are
// over one period b mod g plus each multiple of g below 64; what n leaves of a
// period is summed term by term.
__host__ __device__ inline unsigned long long rt_floor_sum(unsigned long long n, unsigned a, unsigned long long b)
{
    const unsigned low = a & (0u - a), g = low < 64u ? low : 64u, period = 64u / g;
    unsigned long long rest = n / period * (unsigned long long)(period * ((unsigned)b & (g - 1u)) + g * (period * (period - 1u) / 2u));
    unsigned r = (unsigned)b & 63u;
    for (unsigned i = (unsigned)n & (period - 1u); i > 0; --i)
    {
        rest += r;
        r = (r + a) & 63u;
    }
    return (a * (n * (n - 1) / 2) + b * n - rest) / 64;
}

struct RtSeq
{
    int begin, n, past; // first packed row, rows, cached tokens
    int tiles;          // tiles of R tokens
    int cap, nodes;     // slots the table has; tree: mask bits that count
};

__host__ __device__ inline int rt_keys(const RtSeq& q, bool tree, int R, int tile)
{
    const int last = tree ? q.nodes : (tile + 1 < q.tiles ? (tile + 1) * R : q.n);
    const long long k = (long long)q.past + last;
    return k < q.cap ? (int)k : q.cap;
}

// units of the first `tiles` tiles of one K/V head (a call: its code is used
// once per CTA and would crowd the loops out of the instruction cache)
__host__ __device__ __noinline__ unsigned long long rt_units_before(const RtSeq q, bool tree, int R, int tiles)
{
    if (tiles <= 0)
        return 0;
    if (tree)
        return (unsigned long long)tiles * ((rt_keys(q, true, R, 0) + 63) / 64);
    unsigned long long full = (unsigned long long)(tiles < q.tiles ? tiles : q.tiles - 1), sum = 0;
    // tile i < full sees past + (i + 1) R keys, at most cap
    unsigned long long below = 0; // tiles under the cap
    if (q.cap > q.past)
        below = (unsigned long long)(q.cap - q.past) / (unsigned)R;
    if (below > full)
        below = full;
    if (below)
        sum += rt_floor_sum(below, (unsigned)R, (unsigned long long)q.past + (unsigned)R + 63);
    sum += (full - below) * (((unsigned long long)q.cap + 63) / 64);
    if (tiles >= q.tiles)
        sum += (rt_keys(q, false, R, q.tiles - 1) + 63) / 64;
    return sum;
}

__device__ __forceinline__ RtSeq rt_seq(const AttnRowsArgs& a, int s, int R)
{
    RtSeq q;
    q.begin = min(max(a.row_start[s], 0), a.rows);
    const int end = min(max(a.row_start[s + 1], q.begin), a.rows);
    q.n = end - q.begin;
    q.past = max(a.past[s], 0);
    q.tiles = (q.n + R - 1) / R;
    q.cap = (int)(a.pt_stride * ROWS_PAGE); // pt_stride <= 2^24
    q.nodes = min(q.n, a.mask_words * 64);
    return q;
}

// A tile costs its units and RT_TILE_COST more (its queries, the first and
// last unit's latencies, its output): shares are equal in this measure, so a
// share of many short tiles has fewer units. Measured per unit 1.5 us and per
// tile 3 to 4 us: with no tile cost, the shares over short caches took 1.7
// times as long as the average one.
constexpr int RT_TILE_COST = 2;

// Where a share starts (also what the joining kernel reads; the entry behind
// the last share holds the end).
struct RtStart
{
    int s, h, t, u;            // sequence, K/V head, tile, unit in the tile
    unsigned long long begin;  // the units before it
    unsigned long long total;  // units of the call
};

constexpr size_t RT_HEADER_BYTES = 64 * 1024;
// partial means: [CTA][2] of [128 rows][HDP], [128 rows] (sum, offset) and [128 rows]
// of the second part of a far offset
template <int HDP>
__host__ __device__ inline size_t rt_slot_bytes()
{
    return (size_t)128 * HDP * 4 + 128 * 12;
}
template <int HDP>
__device__ __forceinline__ float* rt_slot(const AttnRowsArgs& a, int cta, int which)
{
    return reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + RT_HEADER_BYTES +
                                    (size_t)(cta * 2 + which) * rt_slot_bytes<HDP>());
}

// The start of share `share` of `shares` (one warp; the result in every lane).
template <bool TREE>
__device__ __noinline__ RtStart rt_locate(const AttnRowsArgs a, int R, int share, int shares)
{
    const int lane = threadIdx.x & 31;
    // units and tiles of a sequence
    auto size_of = [&](int s, unsigned long long& units, unsigned long long& tiles) {
        units = tiles = 0;
        if (s >= a.n_seqs)
            return;
        const RtSeq q = rt_seq(a, s, R);
        if (!q.n)
            return;
        units = (unsigned long long)a.n_kv * rt_units_before(q, TREE, R, q.tiles);
        tiles = (unsigned long long)a.n_kv * (unsigned)q.tiles;
    };
    unsigned long long cost = 0, total = 0, un, ti;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32)
    {
        size_of(s0 + lane, un, ti);
        total += un;
        cost += un + RT_TILE_COST * ti;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
    {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        cost += __shfl_xor_sync(0xffffffffu, cost, o);
    }
    RtStart r{};
    r.total = total;
    r.begin = total; // the end, unless found below
    const unsigned long long at = cost * (unsigned)share / (unsigned)shares;
    unsigned long long cost0 = 0, units0 = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32)
    {
        size_of(s0 + lane, un, ti);
        unsigned long long ui = un, ci = un + RT_TILE_COST * ti;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const unsigned long long v = __shfl_up_sync(0xffffffffu, ui, o), w = __shfl_up_sync(0xffffffffu, ci, o);
            if (lane >= o)
            {
                ui += v;
                ci += w;
            }
        }
        const unsigned hit = __ballot_sync(0xffffffffu, cost0 + ci > at);
        if (hit)
        {
            const int l = __ffs(hit) - 1;
            r.s = s0 + l;
            const unsigned long long su = __shfl_sync(0xffffffffu, un, l), st = __shfl_sync(0xffffffffu, ti, l);
            unsigned long long off = at - (cost0 + __shfl_sync(0xffffffffu, ci, l) - su - RT_TILE_COST * st);
            r.begin = units0 + __shfl_sync(0xffffffffu, ui, l) - su;
            const RtSeq q = rt_seq(a, r.s, R);
            const unsigned long long per = su / (unsigned)a.n_kv, pc = per + RT_TILE_COST * (unsigned)q.tiles;
            r.h = (int)(off / pc);
            off -= pc * (unsigned)r.h;
            int lo = 0, hi = q.tiles - 1; // the last tile whose cost starts at or before off
            while (lo < hi)
            {
                const int mid = (lo + hi + 1) >> 1;
                if (rt_units_before(q, TREE, R, mid) + (unsigned long long)RT_TILE_COST * mid <= off)
                    lo = mid;
                else
                    hi = mid - 1;
            }
            const unsigned long long before = rt_units_before(q, TREE, R, lo), in = off - before - (unsigned long long)RT_TILE_COST * lo;
            r.t = lo;
            r.u = in > RT_TILE_COST ? (int)(in - RT_TILE_COST) : 0; // the tile's own cost comes first
            r.begin += per * (unsigned)r.h + before + (unsigned)r.u;
            break;
        }
        units0 += __shfl_sync(0xffffffffu, ui, 31);
        cost0 += __shfl_sync(0xffffffffu, ci, 31);
    }
    return r;
}

// A CTA's items in order: (sequence, K/V head, tile) with units [u0, u1).
template <bool TREE>
struct RtCursor
{
    RtSeq q;
    int s, h, t, u0, u1, keys;
    bool whole; // the item has every unit of its tile
    unsigned long long left;

    __device__ __forceinline__ void set(int R)
    {
        keys = rt_keys(q, TREE, R, t);
        const int units = (keys + 63) / 64;
        u1 = (unsigned long long)(units - u0) <= left ? units : u0 + (int)left;
        whole = u0 == 0 && u1 == units;
    }
    // the first item; false: the CTA has none
    __device__ __forceinline__ bool start(const AttnRowsArgs& a, const RtStart& st, unsigned long long share, int R)
    {
        left = share;
        if (!left)
            return false;
        s = st.s;
        h = st.h;
        t = st.t;
        u0 = st.u;
        q = rt_seq(a, s, R);
        set(R);
        return true;
    }
    __device__ __forceinline__ bool next(const AttnRowsArgs& a, int R)
    {
        left -= (unsigned)(u1 - u0);
        if (!left)
            return false;
        u0 = 0;
        if (++t >= q.tiles)
        {
            t = 0;
            if (++h >= a.n_kv)
            {
                h = 0;
                do
                {
                    if (++s >= a.n_seqs)
                        return false; // the arrays changed under the kernel
                    q = rt_seq(a, s, R);
                } while (q.n == 0);
            }
        }
        set(R);
        return true;
    }
};

// ---- tensor memory ------------------------------------------------------------
__device__ __forceinline__ void rt_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void rt_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void rt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// N columns of the warp's 32 lanes; one statement, so that the registers are
// read only after the wait.
template <int N>
__device__ __forceinline__ void rt_ld(uint32_t taddr, float* v);

template <>
__device__ __forceinline__ void rt_ld<16>(uint32_t taddr, float* v)
{
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
                 "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15 "
                 "}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                   "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i)
        v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void rt_ld8(uint32_t taddr, uint32_t (&r)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}

__device__ __forceinline__ void rt_st8(uint32_t taddr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// D[tensor memory] (+)= A[tensor memory] B[shared memory], fp16 in, fp32 out.
// The descriptor comes as its two words: steps along the operand only add to
// the low one.
__device__ __forceinline__ void rt_mma(uint32_t d, uint32_t a, uint32_t desc_lo, uint32_t desc_hi, uint32_t idesc,
                                       uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 desc;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 desc, {%2, %3};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], desc, %4, p;\n\t}" ::"r"(d),
                 "r"(a), "r"(desc_lo), "r"(desc_hi), "r"(idesc), "r"(acc)
                 : "memory");
}

// True in one lane of the (converged) warp.
__device__ __forceinline__ bool rt_elect()
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

__device__ __forceinline__ void rt_commit(uint32_t mbar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(mbar) : "memory");
}

// Shared-memory descriptors of the 128-byte-swizzled operand. K: rows = keys,
// K-major, 8-key groups 1024 bytes apart. V: the same bytes as an MN-major
// operand: 64-dim blocks 8192 bytes apart (leading offset), 8-key groups
// 1024 bytes apart (stride offset).
constexpr uint32_t RT_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29); // stride 1024, version 1, 128-byte swizzle
__device__ __forceinline__ uint32_t rt_desc_lo(uint32_t saddr, uint32_t lead)
{
    return ((saddr >> 4) & 0x3FFFu) | ((lead >> 4) << 16);
}
// kind::f16 with fp16 A and B, fp32 D, M = 128; b_mn: B is MN-major
__host__ __device__ constexpr uint32_t rt_idesc(int n, bool b_mn)
{
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ float rt_exp2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float2 rt_add2(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 pa, pb, pd;\n\tmov.b64 pa, {%2, %3};\n\tmov.b64 pb, {%4, %5};\n\t"
        "add.rn.f32x2 pd, pa, pb;\n\tmov.b64 {%0, %1}, pd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// x and y as their fp16 high and low parts (pairs, x in the low half); the low
// part x - hi is exact in fp32 before its own rounding
__device__ __forceinline__ void rt_split2(float x, float y, uint32_t& hi, uint32_t& lo)
{
    float rx, ry;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
    asm("{\n\t.reg .b16 a, b, m;\n\tmov.b32 {a, b}, %2;\n\tmov.b16 m, 0xBC00;\n\t" // m = -1
        "fma.rn.f32.f16 %0, a, m, %3;\n\tfma.rn.f32.f16 %1, b, m, %4;\n\t}"
        : "=f"(rx), "=f"(ry)
        : "r"(hi), "f"(x), "f"(y));
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(ry), "f"(rx));
}

// p[0..7] = v[0..7] * by * unit, p 32-byte aligned
__device__ __forceinline__ void rt_store8(float* p, const float* v, float by, float unit)
{
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0] * by * unit),
                 "f"(v[1] * by * unit), "f"(v[2] * by * unit), "f"(v[3] * by * unit), "f"(v[4] * by * unit),
                 "f"(v[5] * by * unit), "f"(v[6] * by * unit), "f"(v[7] * by * unit)
                 : "memory");
}

// max(m, |x|, |y|); a NaN stays
__device__ __forceinline__ float rt_max_abs(float m, float x, float y)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(x)), "f"(fabsf(y)));
    return r;
}
__device__ __forceinline__ float rt_max_abs(float m, const float4& v)
{
    return rt_max_abs(rt_max_abs(m, v.x, v.y), v.z, v.w);
}

// The power of two that puts a magnitude with these bits at 2^14..2^15, and
// its inverse (both normal numbers).
__device__ __forceinline__ void rt_scale_of(uint32_t max_bits, float& up, float& down)
{
    const int e = min(141 - (int)(max_bits >> 23), 126);
    const int k = max_bits ? max(e, -113) : 0;
    up = __uint_as_float((uint32_t)(k + 127) << 23);
    down = __uint_as_float((uint32_t)(127 - k) << 23);
}

// a / b of two powers of two, a <= b (a 0: some power of two)
__device__ __forceinline__ float rt_ratio(float a, float b)
{
    const int d = (int)(__float_as_uint(b) >> 23) - (int)(__float_as_uint(a) >> 23);
    return d > 126 ? 0.0f : __uint_as_float((uint32_t)(127 - d) << 23);
}

template <int REGS>
__device__ __forceinline__ void rt_regs_inc()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void rt_regs_dec()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

// Waits for the phase with the given parity; false: another role gave up, or
// about two seconds passed. The clock is read once in 256 tries. (A suspend
// hint on the tries cost up to a microsecond of each wake-up.)
__device__ __forceinline__ bool rt_wait(uint32_t bar, uint32_t parity, const volatile uint32_t* abort)
{
    uint64_t t0 = 0;
    for (uint32_t n = 0; !mbar_try_wait(bar, parity); ++n)
    {
        if (*abort)
            return false;
        if ((n & 255u) == 255u)
        {
            const uint64_t t = globaltimer_ns();
            if (t0 == 0)
                t0 = t;
            else if (t - t0 > RT_WAIT_LIMIT_NS)
                return false;
        }
    }
    return true;
}

struct RtUnitInfo
{
    float k_down, v_down;      // what undoes the unit's scaling of K and V
    int valid;                 // keys of the unit that exist
    uint32_t kbad[2], vbad[2]; // keys with a non-finite K / V value
};

struct RtShared
{
    uint64_t raw[8], conv[8], free_[8]; // per stage: copied, converted, read by the MMAs
    uint64_t s_full[2], p_full[2], o_full, o_empty, q_raw[4], q_full[2], q_empty[2], done;
    uint32_t tmem, abort;
    RtStart start, end;
    int stage_valid[8];
    alignas(16) uint32_t wmax[2][8];
    RtUnitInfo info[RT_INFO];
    float alpha[4][128];
    float q_down[4][128]; // what undoes an item's rows' scaling of Q
    uint64_t seen[4][128]; // which of a unit's keys a row attends
    float2 stats[4][128]; // (sum, offset) of an item's rows
    float lo[4][128]; // and the second part of a far offset
};

// i / G for i < 128 and G <= 64, by the reciprocal in 2^-16 (kernel-wide
// constant; the product's excess is below 1 / G)
__device__ __forceinline__ int rt_div(int i, int G)
{
    return (int)(((uint32_t)i * ((65535u + (uint32_t)G) / (uint32_t)G)) >> 16);
}

// Where row i of a tile is in q or out (floats from the base; ld floats a
// packed row), or -1 for a row without a token.
__device__ __forceinline__ long long rt_row_at(const RtSeq& q, int h, int t, int i, int G, int R, size_t ld, int hd)
{
    const int tok = rt_div(i, G), r = t * R + tok;
    if (tok >= R || r >= q.n)
        return -1;
    return (long long)((size_t)(q.begin + r) * ld + (size_t)(h * G + i - tok * G) * hd);
}

// What a score of the scaled factors is times scale log2(e): a normal number (a
// key of zeros has the score 0, not NaN, next to the largest ones).
__device__ __forceinline__ float rt_score_scale(float f) { return fminf(fmaxf(f, 1.17549435e-38f), 3.40282347e+38f); }

// scores of keys that a row does not attend
__device__ __forceinline__ void rt_mask16(float (&s)[16], uint32_t seen)
{
#pragma unroll
    for (int j = 0; j < 16; ++j)
        s[j] = (seen >> j) & 1u ? s[j] : -INFINITY;
}

__device__ __forceinline__ float rt_max16(const float (&s)[16])
{
    float m0 = s[0], m1 = s[1];
#pragma unroll
    for (int j = 2; j < 16; j += 2)
    {
        m0 = fmaxf(m0, s[j]);
        m1 = fmaxf(m1, s[j + 1]);
    }
    return fmaxf(m0, m1);
}

// Weights exp2(s f + use) of 16 scores into tensor memory at `t` (8 columns of
// high and 8 of low parts); returns their sum (fp32, two halves).
__device__ __forceinline__ float2 rt_weights(const float (&s)[16], float f, float use, uint32_t t)
{
    const float2 f2 = make_float2(f, f), use2 = make_float2(use, use);
    float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    uint32_t hi[8], lo[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        float2 x = fma2_rn(make_float2(s[2 * j], s[2 * j + 1]), f2, use2);
        x.x = rt_exp2(x.x);
        x.y = rt_exp2(x.y);
        part[j & 1] = rt_add2(part[j & 1], x);
        rt_split2(x.x, x.y, hi[j], lo[j]);
    }
    rt_st8(t, hi);
    rt_st8(t + 8, lo);
    return rt_add2(part[0], part[1]);
}

// Offsets above this are far: 14 - top and s f + off are then no longer both near
// the exact value (spacings of 1/8 and more in exp2's argument; at 2^25 the weights
// would leave the range of fp16), so a far offset is the sum of two floats. That
// costs 1.5 % of long prompts, the vote on it; trees are equal.
constexpr float RT_FAR = 1048576.0f;
__device__ __forceinline__ bool rt_far(float off) { return fabsf(off) > RT_FAR && off < INFINITY; }

// Before the weights of a unit with far rows: their scores in tensor memory become
// fma(s, f, use), one rounding of the exact value, whose largest gives the second
// part of the offset, in *lo from here on (off: the first part before this unit).
// Other rows come with f = 1 and use = 0. Returns the second parts' difference
// and the new one. A call: hardly ever run, its code would crowd the loops.
__device__ __noinline__ float2 rt_far_unit(uint32_t ts, uint64_t seen, float fa, float fb, float use, float off, float* lo)
{
    float top = -INFINITY;
#pragma unroll 1
    for (uint32_t j0 = 0; j0 < 64; j0 += 8)
    {
        uint32_t w[8];
        rt_ld8(ts + j0, w);
#pragma unroll
        for (int j = 0; j < 8; ++j)
        {
            const float x = fmaf(__uint_as_float(w[j]), j0 < 32 ? fa : fb, use);
            w[j] = __float_as_uint(x);
            top = (uint32_t)(seen >> j0) >> j & 1u ? fmaxf(top, x) : top;
        }
        rt_st8(ts + j0, w);
    }
    rt_wait_st();
    const float old = rt_far(off) ? *lo : 0.0f;
    float now = 0.0f;
    if (use != 0.0f)
        *lo = now = fminf(use == off ? old : INFINITY, 14.0f - top);
    __syncwarp();
    return make_float2(now - old, now);
}

// Which of the 64 keys of a unit a row attends. limit: causal: the row's last
// slot; tree: past. nodes: tree: the sequence's nodes (mask bits that count).
template <bool TREE>
__device__ __forceinline__ uint64_t rt_seen(int u, int valid, int limit, const uint64_t* mask, int words)
{
    uint64_t m;
    const int base = u * 64;
    if (!TREE)
    {
        const int lim = limit - base; // keys 0..lim
        m = lim >= 63 ? ~0ull : lim < 0 ? 0ull : (2ull << lim) - 1;
    }
    else
    {
        const int d = base - limit; // node of the unit's first key
        if (d <= -64)
            m = ~0ull;
        else if (d < 0)
            m = ((1ull << -d) - 1) | (mask[0] << -d);
        else
        {
            const int w = d >> 6, sh = d & 63;
            m = w < words ? mask[w] >> sh : 0ull;
            if (sh && w + 1 < words)
                m |= mask[w + 1] << (64 - sh);
        }
    }
    return valid >= 64 ? m : valid <= 0 ? 0ull : m & ((1ull << valid) - 1);
}

// ---------------------------------------------------------------------------
template <bool TREE>
__global__ void __launch_bounds__(RT_THREADS, 1) attn_rows_tc_kernel(const AttnRowsArgs a, unsigned* err)
{
    constexpr int HDP = RT_HDP, NS = RT_NS;
    extern __shared__ __align__(16) uint8_t rt_raw[];
    __shared__ RtShared sm;
    const uint32_t ring = (smem_addr(rt_raw) + 1023u) & ~1023u; // the swizzle works on address bits
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.n_heads / a.n_kv, R = 128 / G, hd = a.head_dim;
    volatile uint32_t* abort = &sm.abort;

    auto stage_at = [&](uint32_t pos) { return ring + (pos % NS) * RT_STAGE; };
    auto bar_raw = [&](uint32_t pos) { return smem_addr(&sm.raw[pos % NS]); };
    auto bar_conv = [&](uint32_t pos) { return smem_addr(&sm.conv[pos % NS]); };
    auto bar_free = [&](uint32_t pos) { return smem_addr(&sm.free_[pos % NS]); };
    auto phase = [&](uint32_t pos) { return (pos / NS) & 1u; };
    auto fail = [&]() {
        *abort = 1u;
        atomicExch(err, 1u);
    };
    // false: the role ends (and says so in `failed`), and with it all others
    auto wait = [&](uint32_t bar, uint32_t parity) -> bool { return rt_wait(bar, parity, abort); };
    bool failed = false;

    if (warp == 0)
    {
        const RtStart st = rt_locate<TREE>(a, R, blockIdx.x, gridDim.x);
        if (lane == 0)
        {
            sm.start = st;
            reinterpret_cast<RtStart*>(a.workspace)[blockIdx.x] = st;
        }
    }
    else if (warp == 3)
    {
        const RtStart en = rt_locate<TREE>(a, R, blockIdx.x + 1, gridDim.x);
        if (lane == 0)
        {
            sm.end = en;
            if (blockIdx.x + 1 == gridDim.x)
                reinterpret_cast<RtStart*>(a.workspace)[gridDim.x] = en;
        }
    }
    else if (warp == 1)
    {
        if (lane == 0)
        {
            for (int i = 0; i < 8; ++i)
            {
                mbar_init(smem_addr(&sm.raw[i]), 1);
                mbar_init(smem_addr(&sm.conv[i]), RT_CONV_THREADS / 32);
                mbar_init(smem_addr(&sm.free_[i]), 1);
            }
            for (int i = 0; i < 2; ++i)
            {
                mbar_init(smem_addr(&sm.s_full[i]), 1);
                mbar_init(smem_addr(&sm.p_full[i]), 4);
                mbar_init(smem_addr(&sm.q_full[i]), 4);
                mbar_init(smem_addr(&sm.q_empty[i]), 1);
            }
            for (int i = 0; i < 4; ++i)
                mbar_init(smem_addr(&sm.q_raw[i]), 1);
            mbar_init(smem_addr(&sm.o_full), 1);
            mbar_init(smem_addr(&sm.o_empty), 8);
            mbar_init(smem_addr(&sm.done), 1);
            mbar_init_fence();
            sm.abort = 0u;
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sm.tmem)),
                     "r"(RT_T_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    else if (warp == 2 && lane < RT_INFO)
    {
        sm.info[lane].kbad[0] = sm.info[lane].kbad[1] = 0u;
        sm.info[lane].vbad[0] = sm.info[lane].vbad[1] = 0u;
    }
    rt_fence_before();
    __syncthreads();
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
        if (warp == 0)
        {
            // ---- producer: K0, K1, V0, K2, V1, ... of every item
            uint32_t pos = 0;
            bool ok = true;
            auto emit = [&](const float* pool, int page, int h, int valid) {
                // lane 0; a page outside the pool is a unit without keys
                if (pos >= NS && !wait(bar_free(pos), phase(pos) ^ 1u))
                    return false;
                const bool there = page >= 0 && page < a.n_pages;
                sm.stage_valid[pos % NS] = there ? valid : 0;
                if (there)
                {
                    const uint32_t bytes = (uint32_t)valid * hd * 4u;
                    mbar_arrive_expect_tx(bar_raw(pos), bytes);
                    bulk_g2s(stage_at(pos), pool + ((size_t)page * a.n_kv + h) * (size_t)(ROWS_PAGE * hd), bytes,
                             bar_raw(pos));
                }
                else
                    mbar_arrive(bar_raw(pos));
                ++pos;
                return true;
            };
            RtCursor<TREE> c;
            int vpage = 0, vh = 0, vvalid = 0; // the V that is due
            bool due = false;
            for (bool more = c.start(a, st0, share, R); more && ok; more = c.next(a, R))
            {
                const int* pt = rows_page_table(a, c.s);
                int mine = 0;
                for (int u = c.u0; u < c.u1 && ok; ++u)
                {
                    const int k = (u - c.u0) & 31;
                    if (k == 0) // the next 32 page numbers, one a lane
                        mine = u + lane < c.u1 ? __ldg(pt + u + lane) : 0;
                    const int page = __shfl_sync(0xffffffffu, mine, k), valid = min(64, c.keys - u * 64);
                    if (lane == 0)
                        for (int v = 0; v < 2 && ok; ++v) // K of this unit, V of the one before
                            if (v == 0 || due)
                                ok = emit(v ? a.v : a.k, v ? vpage : page, v ? vh : c.h, v ? vvalid : valid);
                    ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
                    vpage = page;
                    vh = c.h;
                    vvalid = valid;
                    due = true;
                }
            }
            if (lane == 0)
            {
                if (ok && due)
                    ok = emit(a.v, vpage, vh, vvalid);
                failed = !ok;
                // the copies it issued have landed before the CTA may exit
                for (uint32_t p = pos > NS ? pos - NS : 0; p < pos; ++p)
                    mbar_wait_bounded(bar_raw(p), phase(p), RT_WAIT_LIMIT_NS);
            }
            __syncwarp();
        }
        else if (warp == 1)
        {
            // ---- MMA issuer: the warp walks the units, one lane issues
            constexpr uint32_t id_qk = rt_idesc(64, false), id_pv = rt_idesc(HDP, true);
            uint32_t pos = 0, g = 0, item = 0;
            RtCursor<TREE> c;
            bool more = c.start(a, st0, share, R), ok = true;
            int u = more ? c.u0 : 0;
            while (ok)
            {
                if (more)
                {
                    const uint32_t qb = item & 1u;
                    if ((u == c.u0 && !wait_all(smem_addr(&sm.q_full[qb]), (item >> 1) & 1u)) || !wait_all(bar_conv(pos), phase(pos)))
                    {
                        ok = false;
                        break;
                    }
                    rt_fence_after();
                    const uint32_t k_hi = rt_desc_lo(stage_at(pos), 16u), d = RT_T_S + (g & 1u) * 64u;
                    const bool last = u + 1 == c.u1;
                    if (rt_elect())
                    {
#pragma unroll 1
                        for (uint32_t p = 0; p < 3; ++p) // q_hi k_lo, q_lo k_hi, q_hi k_hi
                        {
                            const uint32_t q = RT_T_Q + qb * 128u + (p == 1 ? RT_T_QLO : 0u), k = k_hi + (p == 0 ? 512u : 0u);
#pragma unroll
                            for (uint32_t n = 0; n < HDP / 16; ++n)
                                rt_mma(d, q + n * 8u, k + n * 2u, RT_DESC_HI, id_qk, p | n);
                        }
                        rt_commit(smem_addr(&sm.s_full[g & 1u]));
                        rt_commit(bar_free(pos));
                        if (last)
                            rt_commit(smem_addr(&sm.q_empty[qb]));
                    }
                    __syncwarp();
                    ++pos;
                }
                if (g > 0) // P V of the unit before
                {
                    const uint32_t j = g - 1u;
                    if (!wait_all(bar_conv(pos), phase(pos)) || !wait_all(smem_addr(&sm.p_full[j & 1u]), (j >> 1) & 1u) ||
                        (j >= 1u && !wait_all(smem_addr(&sm.o_empty), (j - 1u) & 1u)))
                    {
                        ok = false;
                        break;
                    }
                    rt_fence_after();
                    const uint32_t v_hi = rt_desc_lo(stage_at(pos), 8192u), ph = RT_T_S + (j & 1u) * 64u;
                    if (rt_elect())
                    {
#pragma unroll 1
                        for (uint32_t p = 0; p < 3; ++p) // p_hi v_lo, p_lo v_hi, p_hi v_hi
                        {
                            const uint32_t w = ph + (p == 1 ? 8u : 0u), v = v_hi + (p == 0 ? 512u : 0u);
#pragma unroll
                            for (uint32_t n = 0; n < 4; ++n)
                                rt_mma(RT_T_O, w + n * 16u, v + n * 128u, RT_DESC_HI, id_pv, p | n);
                        }
                        rt_commit(smem_addr(&sm.o_full));
                        rt_commit(bar_free(pos));
                    }
                    __syncwarp();
                    ++pos;
                }
                if (!more)
                    break;
                ++g;
                if (++u >= c.u1)
                {
                    more = c.next(a, R);
                    u = c.u0;
                    ++item;
                }
            }
            failed = !ok;
            if (rt_elect())
                rt_commit(smem_addr(&sm.done)); // every MMA issued, whatever happened
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
        for (bool more = c.start(a, st0, share, R); more && ok; more = c.next(a, R), ++item)
        {
            const int r = c.t * R + ti;
            const bool live = ti < R && r < c.q.n;
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
                if (!wait_all(smem_addr(&sm.s_full[b]), (g >> 1) & 1u))
                {
                    ok = false;
                    break;
                }
                rt_fence_after();
                const uint32_t ts = tmem + lanes + RT_T_S + b * 64u;
                if (u == c.u0)
                    qf = qs * sm.q_down[item & 3u][i];
                const RtUnitInfo& in = sm.info[g % RT_INFO];
                float f = rt_score_scale(qf * in.k_down);
                const uint64_t seen = live ? rt_seen<TREE>(u, in.valid, limit, mask, a.mask_words) : 0ull;
                sm.seen[g & 3u][i] = seen;
                if ((in.kbad[0] | in.kbad[1]) != 0u &&
                    (seen & ((uint64_t)in.kbad[0] | (uint64_t)in.kbad[1] << 32)) != 0ull)
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
                    top = fmaxf(top, rt_max16(s) * f);
                }
                const float noff = fminf(off, 14.0f - top);
                float use = noff < INFINITY ? noff : 0.0f, corr = use - off;
                if (__any_sync(0xffffffffu, fabsf(use) > RT_FAR || rt_far(off)))
                {
                    const bool far = fabsf(use) > RT_FAR;
                    const float2 r = rt_far_unit(ts, seen, far ? f : 1.0f, far ? f : 1.0f, far ? use : 0.0f, off,
                                                 &sm.lo[item & 3u][i]);
                    corr += r.x;
                    if (far)
                    {
                        use = r.y;
                        f = 1.0f;
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
                    sum = rt_add2(sum, rt_weights(s, f, use, ts + j0));
                }
                l = fmaf(l, corr, sum.x + sum.y);
                sm.alpha[g & 3u][i] = corr;
                if (u + 1 == c.u1)
                    sm.stats[item & 3u][i] = make_float2(bad ? __uint_as_float(0x7FC00000u) : l, off);
                rt_wait_st();
                rt_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(smem_addr(&sm.p_full[b]));
            }
        }
        failed = !ok;
    }
    else if (warp < RT_W_CV)
    {
        // ---- output sums: thread = row, a warpgroup for each half of the dims
        rt_regs_inc<RT_REGS_O>();
        constexpr int W = HDP / 2;
        const int i = (warp & 3) * 32 + lane, d_first = warp < RT_W_O + 4 ? 0 : W;
        const uint32_t t_o = tmem + ((uint32_t)((warp & 3) * 32) << 16) + RT_T_O + d_first;
        uint32_t g = 0, item = 0;
        bool ok = true;
        RtCursor<TREE> c;
        for (bool more = c.start(a, st0, share, R); more && ok; more = c.next(a, R), ++item)
        {
            float acc[W]; // in units of `unit`, the largest scale of V that counts so far
#pragma unroll
            for (int d = 0; d < W; ++d)
                acc[d] = 0.0f;
            float2 stat = make_float2(0.0f, INFINITY);
            float unit = 0.0f;
            bool bad = false;
            for (int u = c.u0; u < c.u1; ++u, ++g)
            {
                if (!wait_all(smem_addr(&sm.o_full), g & 1u))
                {
                    ok = false;
                    break;
                }
                rt_fence_after();
                float corr = sm.alpha[g & 3u][i];
                const RtUnitInfo& in = sm.info[g % RT_INFO];
                if ((in.vbad[0] | in.vbad[1]) != 0u)
                    bad |= (sm.seen[g & 3u][i] & ((uint64_t)in.vbad[0] | (uint64_t)in.vbad[1] << 32)) != 0ull;
                if (u + 1 == c.u1)
                    stat = sm.stats[item & 3u][i];
                const float f = in.v_down; // a power of two
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
                    mbar_arrive(smem_addr(&sm.o_empty));
            }
            if (!ok)
                break;
            const float l = bad ? __uint_as_float(0x7FC00000u) : stat.x;
            // the row's mean, of a cut tile too: the sums of values near the largest fp32
            // pass it. In this order: 1 / l of the sums is at most 2^15, unit / l of small
            // values would be denormal.
            const float by = l == 0.0f ? 0.0f : 1.0f / l;
            float* to;
            int n = W; // dims to store
            if (c.whole)
            {
                const long long at = rt_row_at(c.q, c.h, c.t, i, G, R, a.ldo, hd);
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
        // ---- a stage from fp32 to its fp16 parts, in place
        rt_regs_dec<RT_REGS_CV>();
        const int ct = tid - RT_W_CV * 32, cw = ct >> 5;
        constexpr int NCH = 64 * HDP / 4 / RT_CONV_THREADS; // 16-byte pieces a thread
        constexpr int PR = HDP / 4, RS = RT_CONV_THREADS / PR; // pieces a row, rows from one piece of a thread to its next
        const int row0 = ct / PR, col = ct % PR;
        const bool in_row = col * 4 < hd;
        const uint32_t in_off = (uint32_t)(row0 * hd + col * 4) * 4u, in_step = (uint32_t)(RS * hd) * 4u;
        // its place in the swizzled rows (RS is a multiple of 8: the same swizzle for every piece)
        const int e = col * 4;
        const uint32_t out_off = (uint32_t)row0 * 128u + (uint32_t)(((e >> 3) ^ (row0 & 7)) * 16 + (e & 7) * 2);
        uint32_t slot = 0, ph = 0, par = 0;
        auto convert = [&](uint32_t unit, bool is_k) -> bool {
            const bool got = wait(smem_addr(&sm.raw[slot]), ph);
            const uint32_t stage = ring + slot * RT_STAGE;
            RtUnitInfo& in = sm.info[unit % RT_INFO];
            const int valid = got ? sm.stage_valid[slot] : 0;
            float4 x[NCH];
            float mx = 0.0f, my = 0.0f; // NaN is kept
            if (valid == 64 && hd == HDP)
            {
#pragma unroll
                for (int n = 0; n < NCH; ++n)
                {
                    const uint4 w = lds128(stage + in_off + n * in_step);
                    x[n] = make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
                }
            }
            else
            {
#pragma unroll
                for (int n = 0; n < NCH; ++n)
                {
                    uint4 w = make_uint4(0u, 0u, 0u, 0u); // behind the last key, behind head_dim
                    if (in_row && row0 + n * RS < valid)
                        w = lds128(stage + in_off + n * in_step);
                    x[n] = make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
                }
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
                        const int row = row0 + n * RS;
                        atomicOr(is_k ? &in.kbad[row >> 5] : &in.vbad[row >> 5], 1u << (row & 31));
                        x[n] = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    mx = rt_max_abs(mx, x[n]);
                }
            }
            const uint32_t wm = __reduce_max_sync(0xffffffffu, __float_as_uint(mx)); // not negative: ordered as integers
            if (lane == 0)
                sm.wmax[par][cw] = wm;
            // every read of the stage is done; a failed wait ends all eight warps together
            if (named_bar_or(1, RT_CONV_THREADS, !got))
                return false;
            const uint4 m0 = *reinterpret_cast<const uint4*>(&sm.wmax[par][0]);
            const uint4 m1 = *reinterpret_cast<const uint4*>(&sm.wmax[par][4]);
            float up, down;
            rt_scale_of(max(max(max(m0.x, m0.y), max(m0.z, m0.w)), max(max(m1.x, m1.y), max(m1.z, m1.w))), up, down);
            if (ct == 0)
            {
                if (is_k)
                {
                    in.k_down = down;
                    in.valid = valid;
                    // the unit after the next one's notes (its slot's last readers are long done)
                    RtUnitInfo& later = sm.info[(unit + 2) % RT_INFO];
                    later.kbad[0] = later.kbad[1] = later.vbad[0] = later.vbad[1] = 0u;
                }
                else
                    in.v_down = down;
            }
            const float2 up2 = make_float2(up, up);
#pragma unroll
            for (int n = 0; n < NCH; ++n)
            {
                uint32_t h0, l0, h1, l1;
                const float2 a2 = mul2_rn(make_float2(x[n].x, x[n].y), up2), b2 = mul2_rn(make_float2(x[n].z, x[n].w), up2);
                rt_split2(a2.x, a2.y, h0, l0);
                rt_split2(b2.x, b2.y, h1, l1);
                const uint32_t at = stage + out_off + n * (RS * 128u);
                asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(h0), "r"(h1) : "memory");
                asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + 8192u), "r"(l0), "r"(l1) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the MMA reads through the async proxy
            __syncwarp();
            if (lane == 0)
                mbar_arrive(smem_addr(&sm.conv[slot]));
            par ^= 1u;
            if (++slot == NS)
            {
                slot = 0;
                ph ^= 1u;
            }
            return true;
        };
        // K of every unit, each followed by V of the unit before; the last V
        const uint32_t left = (uint32_t)share;
        bool ok = true;
        for (uint32_t e = 1; e <= 2u * left && ok; ++e)
        {
            // e: 1 K0, 2 K1, 3 V0, 4 K2, 5 V1, ... 2 left: the last V
            const bool is_k = e == 1u || (!(e & 1u) && e < 2u * left);
            ok = convert(is_k ? e >> 1 : (e == 2u * left ? left - 1u : (e - 3u) >> 1), is_k);
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
        const uint32_t row = ring + NS * RT_STAGE + (uint32_t)i * RT_Q_ROW, raw = smem_addr(&sm.q_raw[w]);
        const float sign = a.scale < 0.0f ? -1.0f : 1.0f; // the softmax takes |scale|
        uint32_t item = 0;
        bool ok = true;
        RtCursor<TREE> c;
        auto copy = [&]() -> bool { // true: the row has a token
            const long long at = rt_row_at(c.q, c.h, c.t, i, G, R, a.ldq, hd);
            const uint32_t n = __popc(__ballot_sync(0xffffffffu, at >= 0));
            if (lane == 0)
                mbar_arrive_expect_tx(raw, n * (uint32_t)hd * 4u);
            __syncwarp();
            if (at >= 0)
                bulk_g2s(row, a.q + at, (uint32_t)hd * 4u, raw);
            return at >= 0;
        };
        bool more = c.start(a, st0, share, R), live = more && copy();
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
                rt_st8(tmem + lanes + RT_T_Q + qb * 128u + RT_T_QLO + d0 / 2, lo);
            }
            rt_wait_st();
            rt_fence_before();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the next copy overwrites what was read
            __syncwarp();
            if (lane == 0)
                mbar_arrive(smem_addr(&sm.q_full[qb]));
            more = c.next(a, R);
            live = more && copy();
        }
        if (!ok) // a copy may be in flight: it has landed before the CTA exits
            mbar_wait_bounded(raw, item & 1u, RT_WAIT_LIMIT_NS);
        failed = !ok;
    }
    if (failed && lane == 0)
        fail();
    rt_fence_before();
    __syncthreads();
    if (warp == 1)
    {
        // every MMA issued is done before its tensor memory is given back
        if (lane == 0)
            mbar_wait_bounded(smem_addr(&sm.done), 0, RT_WAIT_LIMIT_NS);
        __syncwarp();
        rt_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(RT_T_COLS) : "memory");
    }
}

// ---------------------------------------------------------------------------
// Joins the partial means of the tiles that a share's end went through: CTA
// (boundary c, 8 rows), one row a warp. The tile's shares are taken in order.
// At most two slots a CTA, 20 MB in all, from L2 behind two dependent loads:
// 13 us after eight sequences of 4120 tokens, by itself and from cold caches.
// ---------------------------------------------------------------------------
constexpr int RJ_WARPS = 8;

// A row with a far least offset, to `o` (one warp): the shares from `first` on that
// have units of the tile [t0, t1), one after the other, with the second parts of
// their offsets.
template <int HDP, int NC>
__device__ __noinline__ void rt_join_far(const AttnRowsArgs& a, int grid, int first, int part, int i, unsigned long long t0,
                                         unsigned long long t1, float off, float* o)
{
    const int lane = threadIdx.x & 31;
    const RtStart* starts = reinterpret_cast<const RtStart*>(a.workspace);
    float lo = INFINITY, l = 0.0f, inv = 0.0f, acc[HDP / 32];
    for (int turn = 0; turn < 3; ++turn) // the least second part that goes with off; the sum; the mean
    {
        for (int c = first; c < grid && starts[c].begin < t1; ++c)
        {
            if (starts[c].begin >= starts[c + 1].begin)
                continue;
            const float* slot = rt_slot<HDP>(a, c * NC + part, starts[c].begin >= t0 ? 0 : 1);
            const float2 s = __ldcg(reinterpret_cast<const float2*>(slot + 128 * HDP) + i);
            const float second = rt_far(s.y) ? __ldcg(slot + 128 * HDP + 256 + i) : 0.0f;
            if (turn == 0)
            {
                lo = s.y == off ? fminf(lo, second) : lo;
                continue;
            }
            const float w = s.y < INFINITY ? s.x * rt_exp2((off - s.y) + (lo - second)) : 0.0f;
            l += turn == 1 ? w : 0.0f;
            if (turn == 2)
#pragma unroll
                for (int d = 0; d < HDP / 32; ++d)
                    acc[d] = fmaf(__ldcg(slot + (size_t)i * HDP + d * 32 + lane), w * inv, acc[d]);
        }
        inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int d = 0; d < HDP / 32; ++d)
            acc[d] = turn < 2 ? 0.0f * inv : acc[d];
    }
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
        if (d * 32 + lane < a.head_dim)
            o[d * 32 + lane] = acc[d];
}

// NC CTAs work on a share together (128 rows each). At most 40 registers: with the
// 55 it takes by itself a prompt of 2048 tokens is 1 us slower.
template <int HDP, bool TREE, int NC>
__global__ void __launch_bounds__(RJ_WARPS * 32, 6) attn_rows_join_kernel(const AttnRowsArgs a, int grid)
{
    pdl_wait();
    const int c0 = blockIdx.x + 1, lane = threadIdx.x & 31;
    const RtStart* starts = reinterpret_cast<const RtStart*>(a.workspace);
    const RtStart st = starts[c0];
    // share c0 starts inside a tile, and no earlier one does
    if (st.u == 0 || st.begin >= st.total)
        return;
    const unsigned long long t0 = st.begin - (unsigned)st.u;
    const int first = c0 - 1; // starts at or before the tile and ends inside it
    const unsigned long long begin0 = starts[first].begin;
    if (begin0 > t0)
        return;
    const int G = a.n_heads / a.n_kv, R = 128 / G, i2 = blockIdx.y * RJ_WARPS + (threadIdx.x >> 5);
    const int part = i2 >> 7, i = i2 & 127, ti = i / G; // CTA of the share, row of the CTA
    const RtSeq q = rt_seq(a, st.s, NC * R);
    const int r = (st.t * NC + part) * R + ti;
    if (ti >= R || r >= q.n)
        return;
    const unsigned long long t1 = t0 + (unsigned)((rt_keys(q, TREE, NC * R, st.t) + 63) / 64);
    // lane j takes the sum and offset of share c + j, 32 shares at a time; a
    // share without units of the tile has none
    auto stat_of = [&](int c, bool& more) -> float2 {
        float2 v = make_float2(0.0f, INFINITY);
        const int k = c + lane;
        const unsigned long long b = k < grid ? starts[k].begin : t1, e = k < grid ? starts[k + 1].begin : t1;
        if (b < t1 && b < e)
            v = __ldcg(reinterpret_cast<const float2*>(rt_slot<HDP>(a, k * NC + part, b >= t0 ? 0 : 1) + 128 * HDP) + i);
        more = __all_sync(0xffffffffu, b < t1);
        return v;
    };
    bool more, more0;
    const float2 s0 = stat_of(first, more0); // mostly all of them
    float off = -warp_max(-s0.y);
    more = more0;
    for (int c = first + 32; more; c += 32)
        off = fminf(off, -warp_max(-stat_of(c, more).y));
    float* o = a.out + (size_t)(q.begin + r) * a.ldo + (size_t)(st.h * G + (i - ti * G)) * a.head_dim;
    if (rt_far(off))
    {
        rt_join_far<HDP, NC>(a, grid, first, part, i, t0, t1, off, o);
        return;
    }
    // what a share's mean counts: its sum at the least offset, over all of them
    float2 s = s0;
    auto weight = [&]() -> float { return s.y < INFINITY ? s.x * rt_exp2(off - s.y) : s.x; };
    float l = warp_sum(weight());
    more = more0;
    for (int c = first + 32; more; c += 32)
    {
        s = stat_of(c, more);
        l += warp_sum(weight());
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float acc[HDP / 32];
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
        acc[d] = 0.0f * inv; // NaN where no key counts but a query is NaN
    s = s0;
    more = more0;
    for (int c = first;; c += 32)
    {
        if (c > first)
            s = stat_of(c, more);
        const float w = weight() * inv;
        unsigned has = __ballot_sync(0xffffffffu, s.y < INFINITY);
        // in order, four shares' means loaded before the first is used
        while (has)
        {
            float v[4][HDP / 32], wj[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
            {
                const int j = has ? __ffs(has) - 1 : -1;
                has &= has - 1;
                wj[k] = __shfl_sync(0xffffffffu, w, j < 0 ? 0 : j);
                // the first share has the tile as its last item unless it starts with it
                const float* slot = rt_slot<HDP>(a, (c + j) * NC + part, c + j > first || begin0 >= t0 ? 0 : 1);
#pragma unroll
                for (int d = 0; d < HDP / 32; ++d)
                    v[k][d] = j < 0 ? 0.0f : __ldcg(slot + (size_t)i * HDP + d * 32 + lane);
                if (j < 0)
                    wj[k] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int d = 0; d < HDP / 32; ++d)
                    acc[d] = fmaf(v[k][d], wj[k], acc[d]);
        }
        if (!more)
            break;
    }
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
        if (d * 32 + lane < a.head_dim)
            o[d * 32 + lane] = acc[d];
}

} // namespace aaedn_dev

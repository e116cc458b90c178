// sample_rows.cu — next tokens of many rows of logits in one launch:
// temperature, top-k, min-p, top-p and a multinomial draw per row from the
// caller's uniforms, the many-row form of sample.cu with its order of the
// vocabulary (logit descending, ties by the lower id).
//
// With M the row's largest logit and p_i = exp((l_i - M) / T), the kept
// tokens are a prefix of that order: the first top_k of them; of those the
// ones with p_i >= min_p; of those, up to and including the first whose
// cumulative mass reaches top_p times their mass. The token is the first
// kept one whose cumulative mass reaches u times the kept mass. So every
// step is one search: the first token in the order whose cumulative count
// (top_k) or cumulative mass (top_p, the draw) reaches a target; min_p only
// takes masses out of the sums.
//
// p is computed in fp64 (within 2^-47) and held as an integer number of units
// of 2^-44: sums of integers are exact in any order, so the result does not
// depend on the order of the atomics. A million tokens as likely as the largest
// are below 2^64 units. The units' rounding moves a cumulative sum by at most
// 2^-45 a token, below 2^-25 of the mass for a million tokens, and a uniform
// has 24 bits. A step's sum in a CTA is in three 32-bit parts of 15, 15 and 14
// bits a token, so a CTA's slice is at most 131071 tokens.
//
// A row is a thread-block cluster of C CTAs, each with a slice of the
// vocabulary in shared memory (one read of the logits). One pass makes a
// histogram of the masses over 1024 equal steps of M - l; a search picks the
// step that crosses its target, gathers that step's few tokens in the first
// CTA, sorts them and scans their masses. A step with more tokens than the
// list holds (ties, far outliers) is narrowed by a radix descent over (logit
// bits, id), 10 bits a pass. With top_k the row is counted by fixed steps of
// 1/16 of a logit while it is read, and where the tokens down to the k-th's
// step fit the list (2048), one sort answers all; else the step of the k-th
// token, of the steps of M - l, bounds the masses.
#include "common.cuh"

#include "device_check.hpp"
#include "sample_rows.h"

namespace aaedn_dev
{

namespace
{

constexpr int SR_THREADS = 1024, SR_WARPS = SR_THREADS / 32;
constexpr int SR_BINS = 1024; // one per thread
constexpr int SR_LIST = 2048; // two a thread
constexpr int SR_LOADS = 8; // a thread's loads in flight
constexpr uint32_t SR_SLICE = 40000; // logits of a CTA in shared memory
constexpr int SR_MASS_BITS = 44;
constexpr uint32_t SR_MAX_SLICE = 131071; // tokens of a CTA
static_assert(((uint64_t)SR_MAX_VOCAB << SR_MASS_BITS) >> SR_MASS_BITS == SR_MAX_VOCAB, "a row's mass");
static_assert((uint64_t)SR_MAX_SLICE * 0x7FFF <= 0xFFFFFFFFull &&
                  ((uint64_t)SR_MAX_SLICE << (SR_MASS_BITS - 30)) <= 0xFFFFFFFFull,
              "a step's mass parts");
static_assert((SR_MAX_VOCAB + 7) / 8 <= SR_MAX_SLICE, "8 CTAs a row at most");

struct SrShared
{
    uint32_t cnt[SR_BINS], m0[SR_BINS], m1[SR_BINS], m2[SR_BINS]; // this CTA's histogram
    uint64_t pm[SR_BINS];                                         // cumulative mass of the row's steps
    uint32_t pc[SR_BINS];                                         // cumulative count
    uint64_t lkey[SR_LIST]; // first CTA: the row's listed tokens, by order key
    uint64_t lbuf[SR_LIST]; // this CTA's part of them; first CTA then: cumulative masses
    double tbl[128]; // 2^(j / 128)
    uint64_t wsum_m[SR_WARPS];
    uint32_t wsum_c[SR_WARPS];
    float red_max[SR_WARPS], red_min[SR_WARPS];
    uint32_t red_idx[SR_WARPS];
    float cta_max, cta_min;
    uint32_t cta_idx;
    uint32_t n_list, n_mine, at_list;
    int pick;
    uint64_t above_m, tot_m;
    uint32_t above_c, n_in;
    uint64_t found_key, found_mass;
};

// ---- shared memory of the cluster's CTAs ------------------------------------
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank)
{
    uint32_t ra;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_addr(p)), "r"(rank));
    return ra;
}
__device__ __forceinline__ uint32_t peer_ld32(uint32_t a)
{
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void peer_st64(uint32_t a, uint64_t v)
{
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t peer_add32(uint32_t a, uint32_t v)
{
    uint32_t r;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(r) : "r"(a), "r"(v) : "memory");
    return r;
}

template <int C>
__device__ __forceinline__ void row_sync()
{
    if constexpr (C > 1)
        cluster_sync_all();
    else
        __syncthreads();
}

// Larger = earlier in the order: the logit's bits as an ordered integer, then
// the lower id.
__device__ __forceinline__ uint64_t order_key(float l, uint32_t id)
{
    const uint32_t b = __float_as_uint(l == 0.0f ? 0.0f : l); // -0 ties with 0
    const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((uint64_t)o << 32) | (0xFFFFFFFFu - id);
}

__device__ __forceinline__ float order_logit(uint64_t key)
{
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}

struct SrRow
{
    float M, invw;
    double dM, per_t, min_p; // per_t: 128 / (T ln 2)
    float far;               // M - l beyond which the mass rounds to zero units
};

__device__ __forceinline__ int sr_bin(float l, const SrRow& r)
{
    return min((int)((r.M - l) * r.invw), SR_BINS - 1); // monotone in l; NaN (0 * inf) counts as 0
}

// The step of 1/16 that a logit lies in, from +32 down to -32 (beyond: the end
// ones): monotone like sr_bin, but needs no largest logit.
__device__ __forceinline__ int sr_fixed_bin(float l)
{
    return min(max((int)((32.0f - l) * 16.0f), 0), SR_BINS - 1);
}

// exp((l - M) / T) in units of 2^-44; 0 for tokens below min_p. Table lookup
// (P. T. P. Tang, "Table-driven implementation of the exponential function in
// IEEE floating-point arithmetic", 1989): (l - M) / T = (k + r) ln2 / 128 with
// |r| <= 1/2, exp = 2^(k / 128) exp(r ln2 / 128), the polynomial to r^4 (its
// next term is 1.2e-15, the rounding of per_t 33 * 2^-53: within 2^-47). l - M
// is exact, so the largest logit has exactly 2^44 units. Ten fp64
// instructions a token (256 rows 142 us, with a shorter table and two more 149).
__device__ __forceinline__ uint64_t sr_mass(float l, const SrRow& r, const double* tbl)
{
    if (!(r.M - l <= r.far))
        return 0;
    constexpr double MAGIC = 6755399441055744.0, TWO52 = 4503599627370496.0; // 1.5 * 2^52, 2^52
    constexpr double A = 0.69314718055994530942 / 128.0;
    const double d = (double)l - r.dM, t = fma(d, r.per_t, MAGIC);
    const int k = __double2loint(t);
    const double f = fma(d, r.per_t, MAGIC - t);
    double p = fma(f, A * A * A * A / 24.0, A * A * A / 6.0);
    p = fma(p, f, A * A / 2.0);
    p = fma(p, f, A);
    p = fma(p, f, 1.0);
    const double base = tbl[k & 127];
    const double scaled = __hiloint2double(__double2hiint(base) + ((k >> 7) + SR_MASS_BITS) * (1 << 20), __double2loint(base));
    if (r.min_p > 0.0 && scaled * p < r.min_p)
        return 0;
    return (uint64_t)__double_as_longlong(fma(scaled, p, TWO52)) & ((1ull << 52) - 1);
}

// Inclusive scan over the CTA's threads of a count and a mass.
__device__ __forceinline__ void sr_scan(uint32_t& c, uint64_t& m, SrShared& s)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const uint32_t oc = __shfl_up_sync(0xffffffffu, c, o);
        const uint64_t om = __shfl_up_sync(0xffffffffu, m, o);
        if (lane >= o)
        {
            c += oc;
            m += om;
        }
    }
    __syncthreads(); // the sums of the scan before are read
    if (lane == 31)
    {
        s.wsum_c[warp] = c;
        s.wsum_m[warp] = m;
    }
    __syncthreads();
    uint32_t bc = lane < warp ? s.wsum_c[lane] : 0;
    uint64_t bm = lane < warp ? s.wsum_m[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
    {
        bc += __shfl_xor_sync(0xffffffffu, bc, o);
        bm += __shfl_xor_sync(0xffffffffu, bm, o);
    }
    c += bc;
    m += bm;
}

__device__ __forceinline__ void sr_clear(SrShared& s)
{
    const int t = threadIdx.x;
    s.cnt[t] = s.m0[t] = s.m1[t] = s.m2[t] = 0;
}

__device__ __forceinline__ void sr_add(SrShared& s, int bin, uint64_t mass)
{
    const uint32_t p0 = (uint32_t)mass & 0x7FFF, p1 = (uint32_t)(mass >> 15) & 0x7FFF, p2 = (uint32_t)(mass >> 30);
    if (p0)
        atomicAdd(&s.m0[bin], p0);
    if (p1)
        atomicAdd(&s.m1[bin], p1);
    if (p2) // masses of 2^-15 of the largest and more
        atomicAdd(&s.m2[bin], p2);
}

// The row's totals of bin threadIdx.x over the cluster's histograms.
template <int C>
__device__ __forceinline__ void sr_collect(SrShared& s, uint32_t& c, uint64_t& m)
{
    const int t = threadIdx.x;
    c = 0;
    m = 0;
    if constexpr (C == 1)
    {
        c = s.cnt[t];
        m = (uint64_t)s.m0[t] + ((uint64_t)s.m1[t] << 15) + ((uint64_t)s.m2[t] << 30);
    }
    else
    {
        uint32_t v[C][4];
#pragma unroll
        for (int r = 0; r < C; ++r)
        {
            v[r][0] = peer_ld32(peer_addr(&s.cnt[t], r));
            v[r][1] = peer_ld32(peer_addr(&s.m0[t], r));
            v[r][2] = peer_ld32(peer_addr(&s.m1[t], r));
            v[r][3] = peer_ld32(peer_addr(&s.m2[t], r));
        }
#pragma unroll
        for (int r = 0; r < C; ++r)
        {
            c += v[r][0];
            m += (uint64_t)v[r][1] + ((uint64_t)v[r][2] << 15) + ((uint64_t)v[r][3] << 30);
        }
    }
}

// The counts alone of the row's bin threadIdx.x.
template <int C>
__device__ __forceinline__ uint32_t sr_collect_counts(SrShared& s)
{
    if constexpr (C == 1)
        return s.cnt[threadIdx.x];
    uint32_t v[C], c = 0;
#pragma unroll
    for (int r = 0; r < C; ++r)
        v[r] = peer_ld32(peer_addr(&s.cnt[threadIdx.x], r));
#pragma unroll
    for (int r = 0; r < C; ++r)
        c += v[r];
    return c;
}

// One token into this CTA's part of the list (what does not fit is counted only).
__device__ __forceinline__ void sr_append(SrShared& s, uint64_t key)
{
    const uint32_t at = atomicAdd(&s.n_mine, 1u);
    if (at < (uint32_t)SR_LIST)
        s.lbuf[at] = key;
}

// The CTAs' parts into the first CTA's list, in any order (it is sorted); n_list
// counts what did not fit too.
template <int C>
__device__ __forceinline__ void sr_push(SrShared& s)
{
    __syncthreads();
    const uint32_t n = s.n_mine;
    if (threadIdx.x == 0)
        s.at_list = C == 1 ? (s.n_list = n, 0u) : peer_add32(peer_addr(&s.n_list, 0), n);
    __syncthreads();
    const uint32_t at = s.at_list;
    for (uint32_t i = threadIdx.x; i < min(n, (uint32_t)SR_LIST); i += SR_THREADS)
        if (at + i < (uint32_t)SR_LIST)
        {
            if constexpr (C == 1)
                s.lkey[at + i] = s.lbuf[i];
            else
                peer_st64(peer_addr(&s.lkey[at + i], 0), s.lbuf[i]);
        }
}

// The list's first n tokens in order (keys are distinct). Up to 512 a token's
// place is how many keys are larger, two threads counting for a token; more
// take a bitonic network (2048: 66 steps, 15 of them over the whole CTA).
__device__ __forceinline__ void sr_sort(SrShared& s, uint32_t n)
{
    const uint32_t t = threadIdx.x;
    if (n <= SR_THREADS / 2)
    {
        const uint32_t i = t >> 1, part = t & 1;
        uint32_t place = 0;
        uint64_t key = 0;
        if (i < n)
        {
            key = s.lkey[i];
#pragma unroll 4
            for (uint32_t j = part; j < n; j += 2)
                place += s.lkey[j] > key;
        }
        place += __shfl_xor_sync(0xffffffffu, place, 1);
        __syncthreads();
        if (i < n && part == 0)
            s.lkey[place] = key;
        __syncthreads();
        return;
    }
    const uint32_t size = n <= SR_THREADS ? SR_THREADS : SR_LIST;
    for (uint32_t i = n + t; i < size; i += SR_THREADS)
        s.lkey[i] = 0; // behind every token
    __syncthreads();
    for (uint32_t block = 2; block <= size; block *= 2)
        for (uint32_t step = block / 2; step > 0; step /= 2)
        {
            const uint32_t i = 2 * step * (t / step) + (t & (step - 1)), j = i + step;
            if (j < size)
            {
                const uint64_t x = s.lkey[i], y = s.lkey[j];
                if ((x < y) == ((i & block) == 0))
                {
                    s.lkey[i] = y;
                    s.lkey[j] = x;
                }
            }
            // up to 32 apart, the pairs of a warp are 64 tokens of its own, in this step and the next
            if (step > 32 || (step == 1 && block >= 64))
                __syncthreads();
            else
                __syncwarp();
        }
    __syncthreads();
}

// Bound by the passes over the slice (a row without top-k reads it four times)
// and the cluster's barriers between them, not by the masses: 256 rows keep the
// issue slots 68 % and the fp64 pipe 7 % active. In a burst one row of 32000
// takes 12 us, 32 rows of 128256 39 us, 256 rows 140 us (20 would be one read of
// the logits). A row with top_k 50 takes 17 us of its cluster, one without top-k
// 25 to 35.
// C CTAs a row; RES: the slice's logits stay in shared memory, else every pass
// reads them again (from L2 after the first).
template <int C, bool RES>
__global__ void __launch_bounds__(SR_THREADS, RES ? 1 : 2) sample_rows_kernel(const SampleRowsArgs a)
{
    extern __shared__ __align__(16) uint8_t sr_raw[];
    SrShared& s = *reinterpret_cast<SrShared*>(sr_raw);
    float* slice = reinterpret_cast<float*>(sr_raw + sizeof(SrShared));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t row = blockIdx.x / C, rank = blockIdx.x % C;
    const uint32_t per = (a.vocab + C - 1) / C;
    const uint32_t v0 = rank * per, n_mine = v0 < a.vocab ? min(per, a.vocab - v0) : 0u;
    const float* src = a.logits + (size_t)row * a.ld + v0;

    // fn(logit, id) for each of this thread's tokens that is not NaN. Rolled:
    // unrolled over registers, the passes' code outgrew the instruction caches.
    constexpr int UNROLL = RES ? 4 : 8;
    auto each = [&](auto&& fn) {
#pragma unroll UNROLL
        for (uint32_t j = tid; j < n_mine; j += SR_THREADS)
        {
            const float l = RES ? slice[j] : src[j];
            if (l == l)
                fn(l, v0 + j);
        }
    };

    const float T = a.temperature ? a.temperature[row] : 1.0f;
    const int k = a.top_k ? a.top_k[row] : 0;
    const bool cut_k = k > 0 && (uint32_t)k < a.vocab && T > 0.0f;
    if (tid < 128)
        s.tbl[tid] = exp2((double)tid / 128.0);
    sr_clear(s);
    if (tid == 0)
        s.n_list = s.n_mine = 0;
    __syncthreads();
    // ---- the row from memory: its largest logit (the lowest id of it) and the
    // smallest finite one; with top_k the tokens of each 1/16 of a logit
    float mx = -INFINITY, mn = INFINITY;
    uint32_t mi = 0xFFFFFFFFu;
    for (uint32_t j0 = tid; j0 < n_mine; j0 += SR_THREADS * SR_LOADS)
    {
        float l[SR_LOADS];
#pragma unroll
        for (int u = 0; u < SR_LOADS; ++u)
            l[u] = j0 + u * SR_THREADS < n_mine ? (RES ? __ldcs(src + j0 + u * SR_THREADS) : src[j0 + u * SR_THREADS])
                                                : __uint_as_float(0x7FC00000u);
#pragma unroll
        for (int u = 0; u < SR_LOADS; ++u)
        {
            const uint32_t j = j0 + u * SR_THREADS;
            if (RES && j < n_mine)
                slice[j] = l[u]; // read back by this thread only
            if (l[u] == l[u])
            {
                if (l[u] > mx || mi == 0xFFFFFFFFu)
                {
                    mx = l[u];
                    mi = v0 + j;
                }
                if (l[u] > -INFINITY)
                    mn = fminf(mn, l[u]);
                if (cut_k)
                    atomicAdd(&s.cnt[sr_fixed_bin(l[u])], 1u);
            }
        }
    }
    auto better = [](float& v, uint32_t& i, float ov, uint32_t oi) {
        if (ov > v || (ov == v && oi < i))
        {
            v = ov;
            i = oi;
        }
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
    {
        better(mx, mi, __shfl_xor_sync(0xffffffffu, mx, o), __shfl_xor_sync(0xffffffffu, mi, o));
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
    if (lane == 0)
    {
        s.red_max[warp] = mx;
        s.red_idx[warp] = mi;
        s.red_min[warp] = mn;
    }
    __syncthreads();
    mx = s.red_max[lane];
    mi = s.red_idx[lane];
    mn = s.red_min[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
    {
        better(mx, mi, __shfl_xor_sync(0xffffffffu, mx, o), __shfl_xor_sync(0xffffffffu, mi, o));
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
    if constexpr (C > 1)
    {
        if (tid == 0)
        {
            s.cta_max = mx;
            s.cta_idx = mi;
            s.cta_min = mn;
        }
        row_sync<C>();
        mx = -INFINITY;
        mi = 0xFFFFFFFFu;
        mn = INFINITY;
#pragma unroll
        for (int r = 0; r < C; ++r)
        {
            better(mx, mi, __uint_as_float(peer_ld32(peer_addr(&s.cta_max, r))), peer_ld32(peer_addr(&s.cta_idx, r)));
            mn = fminf(mn, __uint_as_float(peer_ld32(peer_addr(&s.cta_min, r))));
        }
    }
    if (!(T > 0.0f) || !isfinite(mx))
    {
        // greedy (T <= 0), or no finite logit to normalise by
        if (rank == 0 && tid == 0)
            a.tokens[row] = mi == 0xFFFFFFFFu ? 0u : mi;
        row_sync<C>(); // no CTA leaves while another reads its shared memory
        return;
    }
    SrRow R;
    R.M = mx;
    R.dM = (double)mx;
    R.per_t = 128.0 / 0.69314718055994530942 / (double)T;
    const float mp = a.min_p ? a.min_p[row] : 0.0f;
    R.min_p = mp > 0.0f ? fmin((double)mp, 1.0) * (double)(1ull << SR_MASS_BITS) : 0.0;
    R.far = fminf(33.0f * T, 3.0e38f); // exp(-33) is below half a unit; an infinite distance is always far
    const float span = fminf(mx - mn, 40.0f * T);
    R.invw = span > 0.0f ? (float)SR_BINS / span : 0.0f;

    const float tp = a.top_p ? a.top_p[row] : 1.0f;
    const float uu = a.u[row];
    // the mass of the list's token i, i < n
    auto mass_at = [&](uint32_t i, uint32_t n) -> uint64_t {
        return i < n ? sr_mass(order_logit(s.lkey[i]), R, s.tbl) : 0ull;
    };
    uint32_t c;
    uint64_t m;
    uint64_t key, W;
    // the step that holds the k-th token, by the counts of a histogram
    auto pick_count = [&]() {
        c = sr_collect_counts<C>(s);
        const uint32_t own = c;
        uint64_t unused = 0;
        sr_scan(c, unused, s);
        if (tid == SR_THREADS - 1 && c < (uint32_t)k) // fewer tokens than k (NaN logits): all of them
        {
            s.pick = SR_BINS - 1;
            s.n_in = c;
        }
        if (c >= (uint32_t)k && c - own < (uint32_t)k)
        {
            s.pick = tid;
            s.n_in = c;
        }
        __syncthreads();
    };
    if (cut_k)
    {
        pick_count();
        int last = s.pick;
        if (s.n_in <= (uint32_t)SR_LIST)
        {
            // everything that top_k can keep fits the list: one sort answers all
            each([&](float l, uint32_t id) {
                if (sr_fixed_bin(l) <= last)
                    sr_append(s, order_key(l, id));
            });
            sr_push<C>(s);
            row_sync<C>();
            if (rank == 0)
            {
                const uint32_t n = min(s.n_list, (uint32_t)SR_LIST), kept = min(n, (uint32_t)k), i = 2 * tid;
                sr_sort(s, n);
                const uint64_t m0 = mass_at(i, kept), m1 = mass_at(i + 1, kept);
                uint32_t lc = 0;
                uint64_t lm = m0 + m1;
                sr_scan(lc, lm, s);
                s.lbuf[i] = lm - m1; // cumulative
                s.lbuf[i + 1] = lm;
                __syncthreads();
                // first i with cum[i] >= target
                auto cross = [&](double target) {
#pragma unroll
                    for (uint32_t e = i; e < i + 2; ++e)
                        if (e < kept && (double)s.lbuf[e] >= target && !(e > 0 && (double)s.lbuf[e - 1] >= target))
                            s.pick = e;
                    __syncthreads();
                    const int at = s.pick;
                    __syncthreads();
                    return at;
                };
                W = kept ? s.lbuf[kept - 1] : 0ull;
                if (tp < 1.0f)
                    W = s.lbuf[cross((double)tp * (double)W)];
                const int at = cross(uu > 0.0f ? fmin((double)uu, 1.0) * (double)W : 0.0);
                if (tid == 0)
                    a.tokens[row] = 0xFFFFFFFFu - (uint32_t)(s.lkey[at] & 0xFFFFFFFFu);
            }
            return; // no CTA reads another's shared memory after the last barrier
        }
        // more tokens than that: the steps of M - l, first the one of the k-th
        // token, then the masses up to it
        row_sync<C>(); // the counts are read
        sr_clear(s);
        __syncthreads();
        each([&](float l, uint32_t) { atomicAdd(&s.cnt[sr_bin(l, R)], 1u); });
        row_sync<C>();
        pick_count();
        last = s.pick;
        s.pc[tid] = c;
        row_sync<C>();
        sr_clear(s);
        __syncthreads();
        each([&](float l, uint32_t) {
            const int b = sr_bin(l, R);
            if (b <= last)
                sr_add(s, b, sr_mass(l, R, s.tbl));
        });
    }
    else
        // ---- the masses of the 1024 steps of M - l
        each([&](float l, uint32_t) { sr_add(s, sr_bin(l, R), sr_mass(l, R, s.tbl)); });
    row_sync<C>();
    {
        uint32_t unused;
        sr_collect<C>(s, unused, m);
        unused = 0;
        sr_scan(unused, m, s);
    }
    s.pm[tid] = m; // cumulative
    row_sync<C>(); // the histograms are free again

    // The first token whose cumulative count (by_count) or mass reaches the
    // target: its order key and the mass up to and including it.
    auto search = [&](bool by_count, uint32_t k, double target, uint64_t& key_out, uint64_t& mass_out) {
        // one thread a step (or digit); hit: it crosses the target
        auto pick_step = [&](uint32_t c_incl, uint64_t m_incl, uint32_t c_excl, uint64_t m_excl, bool first) {
            const bool in = by_count ? c_incl >= k : (double)m_incl >= target;
            const bool before = !first && (by_count ? c_excl >= k : (double)m_excl >= target);
            if (in && !before)
            {
                s.pick = tid;
                s.above_c = c_excl;
                s.above_m = m_excl;
                s.n_in = c_incl - c_excl;
            }
        };
        // the step of the largest logit is the first and never empty, so a target of 0 ends there
        pick_step(by_count ? s.pc[tid] : 0u, s.pm[tid], by_count && tid ? s.pc[tid - 1] : 0u, tid ? s.pm[tid - 1] : 0ull,
                  tid == 0);
        if (tid == 0)
            s.n_list = s.n_mine = 0;
        __syncthreads();
        const int step = s.pick;
        uint32_t above_c = s.above_c;
        uint64_t above_m = s.above_m;
        uint64_t prefix = 0;
        int shift = 64; // the key bits from here up are fixed to prefix
        auto mine = [&](uint64_t key) { return shift == 64 || (key >> shift) == (prefix >> shift); };
        row_sync<C>(); // n_list is zero in every CTA
        while (true)
        {
            // gather the step's tokens in the first CTA
            each([&](float l, uint32_t id) {
                if (sr_bin(l, R) == step)
                {
                    const uint64_t key = order_key(l, id);
                    if (mine(key))
                        sr_append(s, key);
                }
            });
            sr_push<C>(s);
            row_sync<C>();
            const uint32_t n = C == 1 ? s.n_list : peer_ld32(peer_addr(&s.n_list, 0));
            if (n <= (uint32_t)SR_LIST || shift == 0)
                break;
            // too many: narrow the step by the next 10 bits of the order key
            const int nshift = shift > 10 ? shift - 10 : 0;
            sr_clear(s);
            __syncthreads();
            each([&](float l, uint32_t id) {
                const uint64_t key = order_key(l, id);
                if (sr_bin(l, R) == step && mine(key))
                {
                    const int d = SR_BINS - 1 - (int)((key >> nshift) & ((1u << (shift - nshift)) - 1u));
                    atomicAdd(&s.cnt[d], 1u);
                    sr_add(s, d, sr_mass(l, R, s.tbl));
                }
            });
            row_sync<C>();
            uint32_t dc;
            uint64_t dm;
            sr_collect<C>(s, dc, dm);
            const uint32_t own_c = dc;
            const uint64_t own_m = dm;
            sr_scan(dc, dm, s);
            // an empty digit cannot be the one (a target of 0 ends at the first token)
            if (own_c)
                pick_step(above_c + dc, above_m + dm, above_c + dc - own_c, above_m + dm - own_m, dc == own_c);
            if (tid == 0)
                s.n_list = s.n_mine = 0;
            __syncthreads();
            prefix |= (uint64_t)(SR_BINS - 1 - s.pick) << nshift;
            shift = nshift;
            above_c = s.above_c;
            above_m = s.above_m;
            row_sync<C>();
        }
        if (rank == 0)
        {
            const uint32_t n = min(s.n_list, (uint32_t)SR_LIST), i = 2 * tid;
            sr_sort(s, n);
            const uint64_t m0 = mass_at(i, n), m1 = mass_at(i + 1, n);
            uint32_t unused = 0;
            uint64_t lm = m0 + m1;
            sr_scan(unused, lm, s);
#pragma unroll
            for (uint32_t e = i; e < i + 2; ++e)
            {
                // mass up to and including token e, and before it
                const uint64_t upto = above_m + (e == i ? lm - m1 : lm), under = upto - (e == i ? m0 : m1);
                const bool in = by_count ? above_c + e + 1 >= k : (double)upto >= target;
                const bool before = e > 0 && (by_count ? above_c + e >= k : (double)under >= target);
                if (e < n && ((in && !before) || (!in && e == n - 1)))
                {
#pragma unroll
                    for (int r = 0; r < C; ++r)
                    {
                        if constexpr (C == 1)
                        {
                            s.found_key = s.lkey[e];
                            s.found_mass = upto;
                        }
                        else
                        {
                            peer_st64(peer_addr(&s.found_key, r), s.lkey[e]);
                            peer_st64(peer_addr(&s.found_mass, r), upto);
                        }
                    }
                }
            }
        }
        row_sync<C>();
        key_out = s.found_key;
        mass_out = s.found_mass;
    };

    W = s.pm[SR_BINS - 1];
    if (cut_k && (uint32_t)k < s.pc[SR_BINS - 1])
        search(true, (uint32_t)k, 0.0, key, W);
    if (tp < 1.0f)
        search(false, 0, (double)tp * (double)W, key, W);
    search(false, 0, uu > 0.0f ? fmin((double)uu, 1.0) * (double)W : 0.0, key, W);
    if (rank == 0 && tid == 0)
        a.tokens[row] = 0xFFFFFFFFu - (uint32_t)(key & 0xFFFFFFFFu);
    row_sync<C>();
}

template <int C, bool RES>
int sr_launch(const SampleRowsArgs& a, cudaStream_t st)
{
    static PerDeviceOnce attrs;
    const int arc = attrs.run([]() -> int {
        AAEDN_CUDA_TRY(cudaFuncSetAttribute(sample_rows_kernel<C, RES>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            (int)(sizeof(SrShared) + (RES ? SR_SLICE * 4 : 0))));
        return AAEDN_OK;
    });
    if (arc)
        return arc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.rows * C);
    cfg.blockDim = dim3(SR_THREADS);
    cfg.dynamicSmemBytes = sizeof(SrShared) + (RES ? (size_t)(a.vocab + C - 1) / C * 4 : 0);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_rows_kernel<C, RES>, a);
    if (e != cudaSuccess)
        return set_error(AAEDN_ECUDA, "launch of sample_rows_kernel failed: %s", cudaGetErrorString(e));
    count_launch();
    return AAEDN_OK;
}

} // namespace

int sample_rows(const SampleRowsArgs& a, cudaStream_t st)
{
    // The fewest CTAs a row whose shared memory holds it, then more while the
    // rows leave SMs idle and a CTA has over 2048 tokens. Measured at a
    // vocabulary of 128256 (an earlier step, 32 rows now 39): 8 rows by 4 CTAs
    // each 39 us, by 8 33; 32 rows by 4 41, by 8 63; 256 rows by 4 198, by 8
    // 386 (each CTA's passes cost their barriers and histogram whatever its
    // slice).
    int C = 1;
    while (C < 8 && (a.vocab + C - 1) / C > SR_SLICE)
        C *= 2;
    while (C < 8 && (size_t)a.rows * C * 2 <= (size_t)sm_count() && (a.vocab + C - 1) / C > 2048)
        C *= 2;
    // More than four rounds of CTAs: two share an SM and hide each other's
    // barriers, half as many a row, and read their slices again from L2 in every
    // pass. By slices in shared memory and this way: 256 rows of 128256 172 us
    // and 147, 512 337 and 234, 512 of 50257 150 and 116; 160 of 128256 (4.3
    // rounds) 125 and 121, 96 73 and 101.
    const bool many = (size_t)a.rows * C > 4 * (size_t)sm_count();
    if (many && C > 1 && (a.vocab + C / 2 - 1) / (C / 2) <= SR_MAX_SLICE)
        C /= 2;
    if (many || (a.vocab + C - 1) / C > SR_SLICE)
        switch (C)
        {
        case 1: return sr_launch<1, false>(a, st);
        case 2: return sr_launch<2, false>(a, st);
        case 4: return sr_launch<4, false>(a, st);
        default: return sr_launch<8, false>(a, st);
        }
    switch (C)
    {
    case 1: return sr_launch<1, true>(a, st);
    case 2: return sr_launch<2, true>(a, st);
    case 4: return sr_launch<4, true>(a, st);
    default: return sr_launch<8, true>(a, st);
    }
}

} // namespace aaedn_dev

using namespace aaedn_dev;

extern "C" int aaedn_cu_sample_rows(const float* d_logits, size_t ld, size_t rows, uint32_t vocab,
                                    const float* d_temperature, const int32_t* d_top_k, const float* d_top_p,
                                    const float* d_min_p, const float* d_u, uint32_t* d_tokens, void* stream)
{
    const char* fn = "aaedn_cu_sample_rows";
    if (rows == 0)
        return AAEDN_OK;
    if (vocab == 0 || vocab > SR_MAX_VOCAB)
        return set_error(AAEDN_EINVAL, "%s: vocab %u outside 1..%u", fn, vocab, SR_MAX_VOCAB);
    if (rows > ((size_t)1 << 24) || ld < vocab)
        return set_error(AAEDN_EINVAL, "%s: at most 2^24 rows (%zu), ld %zu at least vocab", fn, rows, ld);
    if (!d_logits || !d_u || !d_tokens)
        return set_error(AAEDN_EINVAL, "%s: %s is null", fn, !d_logits ? "d_logits" : !d_u ? "d_u" : "d_tokens");
    int rc;
    if ((rc = check_device_ptr(fn, d_logits, "d_logits", 4)) || (rc = check_device_ptr(fn, d_u, "d_u", 4)) ||
        (rc = check_device_ptr(fn, d_tokens, "d_tokens", 4)) ||
        (d_temperature && (rc = check_device_ptr(fn, d_temperature, "d_temperature", 4))) ||
        (d_top_k && (rc = check_device_ptr(fn, d_top_k, "d_top_k", 4))) ||
        (d_top_p && (rc = check_device_ptr(fn, d_top_p, "d_top_p", 4))) ||
        (d_min_p && (rc = check_device_ptr(fn, d_min_p, "d_min_p", 4))))
        return rc;
    SampleRowsArgs a{};
    a.logits = d_logits;
    a.ld = ld;
    a.rows = (uint32_t)rows;
    a.vocab = vocab;
    a.temperature = d_temperature;
    a.top_k = d_top_k;
    a.top_p = d_top_p;
    a.min_p = d_min_p;
    a.u = d_u;
    a.tokens = d_tokens;
    return sample_rows(a, as_stream(stream));
}

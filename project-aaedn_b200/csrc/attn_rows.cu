// attn_rows.cu — attention of packed query rows over the paged fp32 K/V cache
// (the sequences of a batch in one call), causal or under a tree mask, and
// its C ABI.
#include <algorithm>
#include <atomic>
#include <climits>

#include "common.cuh"

#include "attn_rows.h"
#include "gemm_tc.h" // tc_encode_fn
#include "device_check.hpp"

namespace aaedn_dev
{

// Set when a bounded wait of a call without its own error word ran out (an
// array of the module: no allocation, so a first call can be captured).
__device__ unsigned g_attn_rows_err;
static std::atomic<uint64_t> g_attn_rows_used{0}; // devices (bits) with such a call

int attn_rows_err_check()
{
    int dev = 0;
    if (!g_attn_rows_used.load(std::memory_order_acquire))
        return AAEDN_OK; // no call yet: nothing to read back
    AAEDN_CUDA_TRY(cudaGetDevice(&dev));
    if (!(g_attn_rows_used.load(std::memory_order_acquire) >> (dev & 63) & 1u))
        return AAEDN_OK;
    unsigned e = 0;
    AAEDN_CUDA_TRY(cudaMemcpyFromSymbol(&e, g_attn_rows_err, sizeof e));
    if (!e)
        return AAEDN_OK;
    const unsigned zero = 0;
    AAEDN_CUDA_TRY(cudaMemcpyToSymbol(g_attn_rows_err, &zero, sizeof zero));
    return set_error(AAEDN_ETIMEOUT, "a bounded wait of a packed or tree attention ran out");
}

// The sequence of packed row r: the s with row_start[s] <= r <
// row_start[s + 1], or -1 (a row that belongs to no sequence).
__device__ __forceinline__ int rows_seq_of(const AttnRowsArgs& a, int r)
{
    int lo = 0, hi = a.n_seqs; // first s with row_start[s + 1] > r
    while (lo < hi)
    {
        const int mid = (lo + hi) >> 1;
        if (a.row_start[mid + 1] > r)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo < a.n_seqs && a.row_start[lo] <= r ? lo : -1;
}

__device__ __forceinline__ const int* rows_page_table(const AttnRowsArgs& a, int s)
{
    return a.page_table + (size_t)(a.seq_of ? a.seq_of[s] : s) * a.pt_stride;
}

} // namespace aaedn_dev

#include "attn_rows_pair.cuh"
#include "attn_rows_tc.cuh"

namespace aaedn_dev
{

// ---------------------------------------------------------------------------
// head_dim 129..256: CTA = (up to 32 packed rows of one sequence, query head)
// against tiles of 32 keys in shared memory, online softmax, fp32 throughout.
// Warp w has rows w, w + 8, ...; lanes take the keys for the scores and the
// dims for P V. Masked keys get no weight; a V row with a non-finite value is
// zeros in shared memory and noted: a row that attends it becomes NaN, the
// others never multiply it. A row with no key gives zeros. Bound by the tiles'
// loads and barriers (8 us a tile where an SM has one CTA): 1077 rows, 16
// heads of 256 dims 0.79 ms, eight trees of 16 over 900, 32 heads 0.46 ms; by a
// warp a row that reads its keys for itself 2.9 and 1.3 ms (only single rows
// over short caches, 64 over 200 keys, were faster that way: 0.29 against 0.57).
// ---------------------------------------------------------------------------
constexpr int RL_ROWS = 32, RL_KEYS = 32, RL_WARPS = 8, RL_RW = RL_ROWS / RL_WARPS, RL_LD = 256 + 4;
constexpr size_t RL_SMEM = (size_t)(RL_ROWS + 2 * RL_KEYS) * RL_LD * 4;

template <bool TREE>
__global__ void __launch_bounds__(RL_WARPS * 32, 2) attn_rows_tile_kernel(const AttnRowsArgs a)
{
    extern __shared__ __align__(16) float rl_smem[];
    __shared__ unsigned bad[2]; // keys of a tile whose V is not finite, two tiles in turn
    float* Qs = rl_smem;
    float* Ks = Qs + RL_ROWS * RL_LD;
    float* Vs = Ks + RL_KEYS * RL_LD;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y;
    const int hd = a.head_dim, hd4 = hd >> 2, kvh = h / (a.n_heads / a.n_kv);
    // the piece from packed row 32 x, or from the start of sequence x - blocks
    // where that is inside a block of 32 rows: to the end of its block or sequence
    const int blocks = (a.rows + RL_ROWS - 1) / RL_ROWS;
    const bool starts = (int)blockIdx.x >= blocks;
    const int r0 = starts ? a.row_start[blockIdx.x - blocks] : (int)blockIdx.x * RL_ROWS;
    if (starts && (r0 < 0 || r0 >= a.rows || r0 % RL_ROWS == 0))
        return;
    const int s = starts ? (int)blockIdx.x - blocks : rows_seq_of(a, r0);
    if (s < 0)
        return;
    const int first = a.row_start[s], r1 = min(min(a.rows, a.row_start[s + 1]), r0 / RL_ROWS * RL_ROWS + RL_ROWS);
    if (r1 <= r0)
        return;
    const int np = r1 - r0;
    const long long cap = (long long)a.pt_stride * ROWS_PAGE;
    if (tid < 2)
        bad[tid] = 0u;
    unsigned turn = 0;
    const long long past = max(a.past[s], 0);
    // keys 0..nk-1 are looked at
    const long long nk = min(cap, TREE ? past + min((long long)a.mask_words * 64, (long long)min(a.row_start[s + 1], a.rows) - first)
                                       : past + ((long long)r1 - first));
    const int* pt = rows_page_table(a, s);
    for (int i = tid; i < np * hd4; i += RL_WARPS * 32)
    {
        const int r = i / hd4, c = i - r * hd4;
        *reinterpret_cast<float4*>(Qs + r * RL_LD + 4 * c) =
            *reinterpret_cast<const float4*>(a.q + (size_t)(r0 + r) * a.ldq + (size_t)h * hd + 4 * c);
    }
    const int mine = (np - warp + RL_WARPS - 1) / RL_WARPS; // rows of this warp
    // the weights are held in units that keep their sum at 1 or less, and so every
    // sum of the values within their range
    float m[RL_RW], l[RL_RW], unit[RL_RW];
    float4 acc[RL_RW][2];
#pragma unroll
    for (int k = 0; k < RL_RW; ++k)
    {
        m[k] = -INFINITY;
        l[k] = 0.0f;
        unit[k] = 1.0f;
        acc[k][0] = acc[k][1] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (long long t0 = 0; t0 < nk; t0 += RL_KEYS)
    {
        const int page = pt[t0 / ROWS_PAGE];
        if (page < 0 || page >= a.n_pages)
            continue; // not a page: as masked keys
        const size_t base = (((size_t)page * a.n_kv + kvh) * ROWS_PAGE + (size_t)(t0 % ROWS_PAGE)) * hd;
        const int valid = (int)min((long long)RL_KEYS, nk - t0);
        __syncthreads(); // the tile before is read
#pragma unroll 4
        for (int i = tid; i < RL_KEYS * hd4; i += RL_WARPS * 32)
        {
            const int r = i / hd4, c = i - r * hd4;
            float4 kv = make_float4(0.f, 0.f, 0.f, 0.f), vv = kv;
            if (r < valid)
            {
                kv = *reinterpret_cast<const float4*>(a.k + base + (size_t)r * hd + 4 * c);
                vv = *reinterpret_cast<const float4*>(a.v + base + (size_t)r * hd + 4 * c);
                if (!(fabsf(vv.x) + fabsf(vv.y) + fabsf(vv.z) + fabsf(vv.w) < INFINITY) &&
                    !(isfinite(vv.x) && isfinite(vv.y) && isfinite(vv.z) && isfinite(vv.w)))
                {
                    atomicOr(&bad[turn & 1u], 1u << r);
                    vv = make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
            *reinterpret_cast<float4*>(Ks + r * RL_LD + 4 * c) = kv;
            *reinterpret_cast<float4*>(Vs + r * RL_LD + 4 * c) = vv;
        }
        if (tid == 0)
            bad[(turn + 1u) & 1u] = 0u;
        __syncthreads();
        const unsigned nan_v = bad[turn & 1u];
        ++turn;
        const long long key = t0 + lane;
        float w[RL_RW];
#pragma unroll
        for (int k = 0; k < RL_RW; ++k)
            w[k] = 0.0f;
        for (int c = 0; c < hd4; ++c)
        {
            const float4 kf = *reinterpret_cast<const float4*>(Ks + lane * RL_LD + 4 * c);
#pragma unroll
            for (int k = 0; k < RL_RW; ++k)
                if (k < mine)
                {
                    const float4 qf = *reinterpret_cast<const float4*>(Qs + (k * RL_WARPS + warp) * RL_LD + 4 * c);
                    w[k] = fmaf(qf.x, kf.x, w[k]);
                    w[k] = fmaf(qf.y, kf.y, w[k]);
                    w[k] = fmaf(qf.z, kf.z, w[k]);
                    w[k] = fmaf(qf.w, kf.w, w[k]);
                }
        }
#pragma unroll
        for (int k = 0; k < RL_RW; ++k)
        {
            if (k >= mine)
                continue;
            const int row = r0 + k * RL_WARPS + warp;
            bool see = lane < valid;
            if (!TREE)
                see = see && key <= past + ((long long)row - first);
            else if (see && key >= past)
            {
                const int j = (int)(key - past);
                see = ((a.mask[(size_t)row * a.mask_words + (j >> 6)] >> (j & 63)) & 1) != 0;
            }
            const float sc = see ? w[k] * a.scale : -INFINITY;
            const float mnew = fmaxf(m[k], warp_max(sc)), ref = mnew == -INFINITY ? 0.0f : mnew;
            float corr = expf(m[k] - ref);
            m[k] = mnew;
            w[k] = see ? expf(sc - ref) * unit[k] : 0.0f;
            l[k] = l[k] * corr + warp_sum(w[k]);
            if (l[k] > 1.0f)
            {
                // by a power of two, which is exact, to at most 1
                const float down = __uint_as_float((253u - (__float_as_uint(l[k]) >> 23)) << 23);
                unit[k] *= down;
                corr *= down;
                w[k] *= down;
                l[k] *= down;
            }
            if ((__ballot_sync(0xffffffffu, see) & nan_v) != 0u)
                l[k] = __uint_as_float(0x7FC00000u);
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                acc[k][e].x *= corr;
                acc[k][e].y *= corr;
                acc[k][e].z *= corr;
                acc[k][e].w *= corr;
            }
        }
        for (int j = 0; j < valid; ++j)
        {
            const float4 v0 = *reinterpret_cast<const float4*>(Vs + j * RL_LD + 4 * lane);
            const float4 v1 = *reinterpret_cast<const float4*>(Vs + j * RL_LD + 128 + 4 * lane);
#pragma unroll
            for (int k = 0; k < RL_RW; ++k)
                if (k < mine)
                {
                    const float wj = __shfl_sync(0xffffffffu, w[k], j);
                    acc[k][0].x = fmaf(wj, v0.x, acc[k][0].x);
                    acc[k][0].y = fmaf(wj, v0.y, acc[k][0].y);
                    acc[k][0].z = fmaf(wj, v0.z, acc[k][0].z);
                    acc[k][0].w = fmaf(wj, v0.w, acc[k][0].w);
                    acc[k][1].x = fmaf(wj, v1.x, acc[k][1].x);
                    acc[k][1].y = fmaf(wj, v1.y, acc[k][1].y);
                    acc[k][1].z = fmaf(wj, v1.z, acc[k][1].z);
                    acc[k][1].w = fmaf(wj, v1.w, acc[k][1].w);
                }
        }
    }
#pragma unroll
    for (int k = 0; k < RL_RW; ++k)
        if (k < mine)
        {
            const float inv = l[k] == 0.0f ? 0.0f : 1.0f / l[k];
            float* o = a.out + (size_t)(r0 + k * RL_WARPS + warp) * a.ldo + (size_t)h * hd;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (e * 32 + lane < hd4)
                    *reinterpret_cast<float4*>(o + e * 128 + 4 * lane) =
                        make_float4(acc[k][e].x * inv, acc[k][e].y * inv, acc[k][e].z * inv, acc[k][e].w * inv);
        }
}

template <typename Kern>
static int rows_tc_attrs(Kern kern, size_t smem)
{
    AAEDN_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaFuncAttributes at;
    AAEDN_CUDA_TRY(cudaFuncGetAttributes(&at, kern));
    if (at.numRegs != RT_REGS) // the roles' register shares are drawn from the launch's
        return set_error(AAEDN_EUNSUPPORTED, "an attn_rows kernel was built with %d registers, not %d", at.numRegs, RT_REGS);
    return AAEDN_OK;
}

int attn_rows_init()
{
    static PerDeviceOnce once;
    return once.run([]() -> int {
        int rc;
        AAEDN_CUDA_TRY(cudaFuncSetAttribute(attn_rows_tile_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            (int)RL_SMEM));
        AAEDN_CUDA_TRY(cudaFuncSetAttribute(attn_rows_tile_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            (int)RL_SMEM));
        if ((rc = rows_tc_attrs(attn_rows_tc_kernel<false>, RT_SMEM)) ||
            (rc = rows_tc_attrs(attn_rows_tc_kernel<true>, RT_SMEM)) ||
            (rc = rows_tc_attrs(attn_rows_pair_kernel<false>, RP_SMEM)))
            return rc;
        return rows_tc_attrs(attn_rows_pair_kernel<true>, RP_SMEM);
    });
}

// the word that a bounded wait's failure sets
static int rows_err_word(const AttnRowsArgs& a, unsigned** err)
{
    *err = a.err;
    if (!a.err)
    {
        void* p = nullptr;
        AAEDN_CUDA_TRY(cudaGetSymbolAddress(&p, g_attn_rows_err));
        *err = static_cast<unsigned*>(p);
        int dev = 0;
        AAEDN_CUDA_TRY(cudaGetDevice(&dev));
        g_attn_rows_used.fetch_or(1ull << (dev & 63), std::memory_order_release);
    }
    return AAEDN_OK;
}

// CTAs of a launch: one an SM, as far as the workspace's partial sums go
template <int HDP>
static int rows_grid()
{
    return std::min<int>(sm_count(), (int)((AAEDN_ATTN_ROWS_WORKSPACE_BYTES - RT_HEADER_BYTES) / (2 * rt_slot_bytes<HDP>())));
}

// The tensor map of a page pool as rows of head_dim floats, `dims` x `keys` a copy.
static int rows_map(CUtensorMap& map, const AttnRowsArgs& a, const float* pool, int dims, int keys)
{
    const PFN_cuTensorMapEncodeTiled_v12000 enc = tc_encode_fn();
    if (!enc)
        return set_error(AAEDN_ECUDA, "packed attention: cuTensorMapEncodeTiled is not available");
    const cuuint64_t size[2] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.n_pages * (cuuint64_t)a.n_kv * ROWS_PAGE};
    const cuuint64_t stride[1] = {(cuuint64_t)a.head_dim * 4};
    const cuuint32_t box[2] = {(cuuint32_t)dims, (cuuint32_t)keys};
    const cuuint32_t one[2] = {1, 1};
    const CUresult r = enc(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<float*>(pool), size, stride, box, one,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(AAEDN_ECUDA, "packed attention: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return AAEDN_OK;
}

template <int HDP, bool TREE, int NC>
static int rows_join(const AttnRowsArgs& a, int shares, cudaStream_t st)
{
    if (shares < 2)
        return AAEDN_OK;
    const cudaError_t e = launch_kernel(attn_rows_join_kernel<HDP, TREE, NC>, dim3((unsigned)shares - 1, NC * 128 / RJ_WARPS),
                                        dim3(RJ_WARPS * 32), 0, st, true, a, shares);
    if (e != cudaSuccess)
        return set_error(AAEDN_ECUDA, "launch of attn_rows_join_kernel failed: %s", cudaGetErrorString(e));
    count_launch();
    return AAEDN_OK;
}

template <bool TREE>
static int rows_pair_launch(const AttnRowsArgs& a, cudaStream_t st)
{
    unsigned* err;
    CUtensorMap kmap, vmap;
    int rc;
    if ((rc = rows_err_word(a, &err)) || (rc = rows_map(kmap, a, a.k, 128, 32)) || (rc = rows_map(vmap, a, a.v, 64, 64)))
        return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (unsigned)(rows_grid<RP_HDP>() / 2));
    cfg.blockDim = dim3(RT_THREADS);
    cfg.dynamicSmemBytes = RP_SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    // as many pairs as run at once: the shares are equal, so one pair that
    // waits for another's SMs would double the time (a GPU whose SMs do not
    // all pair up inside their cluster groups holds fewer than SMs / 2)
    static std::atomic<int> fit[64];
    int dev = 0;
    AAEDN_CUDA_TRY(cudaGetDevice(&dev));
    std::atomic<int>& slot = fit[dev & 63];
    int pairs = slot.load(std::memory_order_relaxed);
    if (pairs <= 0)
    {
        AAEDN_CUDA_TRY(cudaOccupancyMaxActiveClusters(&pairs, attn_rows_pair_kernel<TREE>, &cfg));
        pairs = std::max(1, std::min(pairs, rows_grid<RP_HDP>() / 2));
        slot.store(pairs, std::memory_order_relaxed);
    }
    cfg.gridDim = dim3(2 * (unsigned)pairs);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_rows_pair_kernel<TREE>, a, err, kmap, vmap);
    if (e != cudaSuccess)
        return set_error(AAEDN_ECUDA, "launch of attn_rows_pair_kernel failed: %s", cudaGetErrorString(e));
    count_launch();
    return rows_join<RP_HDP, TREE, 2>(a, pairs, st);
}

template <bool TREE>
static int rows_tc_launch(const AttnRowsArgs& a, cudaStream_t st)
{
    unsigned* err;
    if (int rc = rows_err_word(a, &err))
        return rc;
    const int grid = rows_grid<RT_HDP>();
    attn_rows_tc_kernel<TREE><<<grid, RT_THREADS, RT_SMEM, st>>>(a, err);
    AAEDN_LAUNCH_CHECK("attn_rows_tc_kernel");
    return rows_join<RT_HDP, TREE, 1>(a, grid, st);
}

// The kernel by head_dim. Up to 64 one SM a tile: the pair's stages are 128
// dims wide, and half of each MMA would be padding (prompt of 2048 tokens 123
// us, by the pairs 131; a tree of 16 over 4001 tokens 26, by the pairs 34).
// 65..128 the pairs (a prompt of 4096 tokens, 64 heads over 8: 924 us when they
// came, by single SMs 1053; eight sequences of 4120 tokens 259 and 274). Both as
// measured when the choice was made.
// Above, a tile's operands and sums do not fit one SM's tensor memory: fp32 on
// the FMA units. (Where both run, one warp a row, the simplest kernel, was 70 to
// 90 times slower than the tensor cores on prompts: 13.6 against 0.15 ms.)
int attn_rows(const AttnRowsArgs& a, cudaStream_t st)
{
    if (int rc = attn_rows_init())
        return rc;
    if (a.head_dim <= 128)
    {
        if (a.head_dim <= 64)
            return a.mask ? rows_tc_launch<true>(a, st) : rows_tc_launch<false>(a, st);
        return a.mask ? rows_pair_launch<true>(a, st) : rows_pair_launch<false>(a, st);
    }
    const dim3 tiles((unsigned)((a.rows + RL_ROWS - 1) / RL_ROWS + a.n_seqs), (unsigned)a.n_heads);
    if (a.mask)
        attn_rows_tile_kernel<true><<<tiles, RL_WARPS * 32, RL_SMEM, st>>>(a);
    else
        attn_rows_tile_kernel<false><<<tiles, RL_WARPS * 32, RL_SMEM, st>>>(a);
    AAEDN_LAUNCH_CHECK("attn_rows_tile_kernel");
    return AAEDN_OK;
}

} // namespace aaedn_dev

using namespace aaedn_dev;

namespace
{

int rows_call(const char* fn, bool tree, const float* d_q, size_t ldq, const aaedn_kv_cache* cache,
              const int32_t* d_row_start, const int32_t* d_past, const uint64_t* d_mask, size_t mask_words,
              size_t n_seqs, size_t rows, size_t n_heads, float scale, float* d_out, size_t ldo, void* d_workspace,
              size_t workspace_bytes, void* stream)
{
    if (n_seqs == 0 || rows == 0)
        return AAEDN_OK;
    if (!cache)
        return set_error(AAEDN_EINVAL, "%s: cache is null", fn);
    const aaedn_kv_cache& c = *cache;
    const size_t hd = c.head_dim;
    if (hd == 0 || hd % 4 || hd > 256)
        return set_error(AAEDN_EINVAL, "%s: head_dim %zu is not a multiple of 4 in 4..256", fn, hd);
    if (c.n_kv_heads == 0 || n_heads == 0 || n_heads % c.n_kv_heads || n_heads / c.n_kv_heads > 64 || n_heads > 65535)
        return set_error(AAEDN_EINVAL, "%s: n_heads %zu must be n_kv_heads (%u) times 1..64, at most 65535", fn, n_heads,
                         c.n_kv_heads);
    if (n_seqs > 65536 || rows > (size_t)(1 << 24))
        return set_error(AAEDN_EINVAL, "%s: at most 65536 sequences and 2^24 rows (%zu, %zu)", fn, n_seqs, rows);
    if (c.n_pages == 0 || c.n_pages > (uint32_t)INT_MAX || c.pt_stride == 0 || c.pt_stride > (size_t)(1 << 24))
        return set_error(AAEDN_EINVAL, "%s: n_pages %u and pt_stride %zu must be at least 1 (pt_stride at most 2^24)", fn,
                         c.n_pages, c.pt_stride);
    if (ldq < n_heads * hd || ldo < n_heads * hd || ldq % 4 || ldo % 4)
        return set_error(AAEDN_EINVAL, "%s: ldq %zu and ldo %zu must be multiples of 4 of at least n_heads * head_dim", fn,
                         ldq, ldo);
    if (tree && (mask_words == 0 || mask_words > 1024))
        return set_error(AAEDN_EINVAL, "%s: mask_words %zu outside 1..1024", fn, mask_words);
    if (!isfinite(scale))
        return set_error(AAEDN_EINVAL, "%s: scale is not finite", fn);
    int rc;
    if ((rc = check_device_ptr(fn, d_q, "d_q", 16)) || (rc = check_device_ptr(fn, c.d_k, "d_k", 16)) ||
        (rc = check_device_ptr(fn, c.d_v, "d_v", 16)) || (rc = check_device_ptr(fn, c.d_page_table, "d_page_table", 4)) ||
        (rc = check_device_ptr(fn, d_row_start, "d_row_start", 4)) || (rc = check_device_ptr(fn, d_past, "the cached lengths", 4)) ||
        (rc = check_device_ptr(fn, d_out, "d_out", 16)) || (rc = check_device_ptr(fn, d_workspace, "d_workspace", 16)))
        return rc;
    if (tree && (rc = check_device_ptr(fn, d_mask, "d_mask", 8)))
        return rc;
    if (workspace_bytes < AAEDN_ATTN_ROWS_WORKSPACE_BYTES)
        return set_error(AAEDN_EINVAL, "%s: workspace of %zu bytes, %u needed", fn, workspace_bytes,
                         AAEDN_ATTN_ROWS_WORKSPACE_BYTES);
    AttnRowsArgs a{};
    a.q = d_q;
    a.ldq = ldq;
    a.k = c.d_k;
    a.v = c.d_v;
    a.page_table = c.d_page_table;
    a.pt_stride = c.pt_stride;
    a.n_pages = (int)c.n_pages;
    a.row_start = d_row_start;
    a.past = d_past;
    a.n_seqs = (int)n_seqs;
    a.rows = (int)rows;
    a.mask = tree ? d_mask : nullptr;
    a.mask_words = (int)mask_words;
    a.n_heads = (int)n_heads;
    a.n_kv = (int)c.n_kv_heads;
    a.head_dim = (int)hd;
    a.scale = scale;
    a.out = d_out;
    a.ldo = ldo;
    a.workspace = d_workspace;
    a.err = nullptr; // the library's own word, reported by aaedn_device_sync
    return attn_rows(a, as_stream(stream));
}

} // namespace

extern "C" int aaedn_cu_attention_packed(const float* d_q, size_t ldq, const aaedn_kv_cache* cache,
                                         const int32_t* d_row_start, const int32_t* d_past, size_t n_seqs, size_t rows,
                                         size_t n_heads, float scale, float* d_out, size_t ldo, void* d_workspace,
                                         size_t workspace_bytes, void* stream)
{
    return rows_call("aaedn_cu_attention_packed", false, d_q, ldq, cache, d_row_start, d_past, nullptr, 0, n_seqs, rows,
                     n_heads, scale, d_out, ldo, d_workspace, workspace_bytes, stream);
}

extern "C" int aaedn_cu_attention_tree(const float* d_q, size_t ldq, const aaedn_kv_cache* cache,
                                       const int32_t* d_row_start, const int32_t* d_past, const uint64_t* d_mask,
                                       size_t mask_words, size_t n_seqs, size_t rows, size_t n_heads, float scale,
                                       float* d_out, size_t ldo, void* d_workspace, size_t workspace_bytes, void* stream)
{
    return rows_call("aaedn_cu_attention_tree", true, d_q, ldq, cache, d_row_start, d_past, d_mask, mask_words, n_seqs,
                     rows, n_heads, scale, d_out, ldo, d_workspace, workspace_bytes, stream);
}

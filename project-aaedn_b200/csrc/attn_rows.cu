// attn_rows.cu — attention of packed query rows over the paged fp32 K/V cache
// (the sequences of a batch in one call), causal or under a tree mask, and
// its C ABI.
#include <algorithm>
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

int attn_rows_err_check()
{
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
// One warp per (packed row, query head), for head_dim 129..256. Keys come 32
// at a time: lane j scores key s0 + j against q (in shared memory), the softmax
// is carried online (running max and sum), then the lanes take the head dims
// and add the keys' weighted V rows. fp32 throughout; a key that the row may
// not attend is never read, so what such a slot holds (NaN, an unused page) has
// no effect. A row with no key gives zeros. Bound by its own loads: every row
// reads its keys for itself, from L2 (1077 tokens, 16 heads of 256 dims: 2.9
// ms).
// ---------------------------------------------------------------------------
constexpr int RW_WARPS = 4;

template <bool TREE>
__global__ void __launch_bounds__(RW_WARPS * 32) attn_rows_warp_kernel(const AttnRowsArgs a)
{
    __shared__ __align__(16) float qs[RW_WARPS][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.x * RW_WARPS + warp, h = blockIdx.y;
    if (row >= a.rows)
        return;
    const int s = rows_seq_of(a, row);
    if (s < 0)
        return;
    const int hd = a.head_dim, kvh = h / (a.n_heads / a.n_kv);
    const float* qr = a.q + (size_t)row * a.ldq + (size_t)h * hd;
    for (int d = lane; d < hd; d += 32)
        qs[warp][d] = qr[d];
    __syncwarp();
    const long long past = max(a.past[s], 0), cap = (long long)a.pt_stride * ROWS_PAGE;
    const long long local = (long long)row - a.row_start[s];
    // keys 0..nk-1 are looked at
    const long long nk = min(cap, TREE ? past + min((long long)a.mask_words * 64,
                                                    (long long)min(a.row_start[s + 1], a.rows) - a.row_start[s])
                                       : past + local + 1);
    const int* pt = rows_page_table(a, s);
    const uint64_t* mask = TREE ? a.mask + (size_t)row * a.mask_words : nullptr;
    auto kv_at = [&](const float* base, long long key) -> const float* {
        const int page = pt[key / ROWS_PAGE];
        if (page < 0 || page >= a.n_pages)
            return nullptr; // not a page: as a masked key
        return base + (((size_t)page * a.n_kv + kvh) * ROWS_PAGE + (size_t)(key % ROWS_PAGE)) * hd;
    };
    auto seen = [&](long long key) {
        if (!TREE || key < past)
            return true;
        const int j = (int)(key - past);
        return ((mask[j >> 6] >> (j & 63)) & 1) != 0;
    };
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float mrun = -INFINITY, lrun = 0.0f;
    for (long long s0 = 0; s0 < nk; s0 += 32)
    {
        const long long key = s0 + lane;
        const float* kr = key < nk && seen(key) ? kv_at(a.k, key) : nullptr;
        float sc = -INFINITY;
        if (kr)
        {
            float dot = 0.0f;
            for (int c = 0; c < (hd >> 2); ++c)
            {
                const float4 kv = reinterpret_cast<const float4*>(kr)[c];
                const float4 qv = reinterpret_cast<const float4*>(qs[warp])[c];
                dot = fmaf(qv.x, kv.x, dot);
                dot = fmaf(qv.y, kv.y, dot);
                dot = fmaf(qv.z, kv.z, dot);
                dot = fmaf(qv.w, kv.w, dot);
            }
            sc = dot * a.scale;
        }
        const float mnew = fmaxf(mrun, warp_max(sc));
        const float ref = mnew == -INFINITY ? 0.0f : mnew; // nothing attended so far
        const float w = kr ? expf(sc - ref) : 0.0f;
        const float corr = expf(mrun - ref);
        lrun = lrun * corr + warp_sum(w);
        mrun = mnew;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            acc[i] *= corr;
        const unsigned live = __ballot_sync(0xffffffffu, kr != nullptr);
        for (int j = 0; j < 32; ++j)
        {
            const float wj = __shfl_sync(0xffffffffu, w, j);
            if (!((live >> j) & 1))
                continue;
            const float* vr = kv_at(a.v, s0 + j);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (lane + 32 * i < hd)
                    acc[i] = fmaf(wj, vr[lane + 32 * i], acc[i]);
        }
    }
    const float inv = lrun == 0.0f ? 0.0f : 1.0f / lrun;
    float* o = a.out + (size_t)row * a.ldo + (size_t)h * hd;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < hd)
            o[lane + 32 * i] = acc[i] * inv;
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
// came, by single SMs 1053; eight sequences of 4120 tokens 259 and 274).
// Above, a tile's operands do not fit one SM's tensor memory beside its sums:
// one warp a row (on prompts 70 to 90 times slower where both can run: 13.6
// against 0.15 ms; only calls of a few rows over short caches lose nothing by
// it: 5 rows without a cache 16 us, by the pairs 20).
int attn_rows(const AttnRowsArgs& a, cudaStream_t st)
{
    if (a.head_dim <= 128)
    {
        if (int rc = attn_rows_init())
            return rc;
        if (a.head_dim <= 64)
            return a.mask ? rows_tc_launch<true>(a, st) : rows_tc_launch<false>(a, st);
        return a.mask ? rows_pair_launch<true>(a, st) : rows_pair_launch<false>(a, st);
    }
    const dim3 grid((unsigned)((a.rows + RW_WARPS - 1) / RW_WARPS), (unsigned)a.n_heads);
    if (a.mask)
        attn_rows_warp_kernel<true><<<grid, RW_WARPS * 32, 0, st>>>(a);
    else
        attn_rows_warp_kernel<false><<<grid, RW_WARPS * 32, 0, st>>>(a);
    AAEDN_LAUNCH_CHECK("attn_rows_warp_kernel");
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

// kv_pages.cu — copies of whole cache pages and the compaction of a
// sequence's last slots, in every layer's K and V with one launch.
#include <cuda.h>
#include <cudaTypedefs.h> // PFN_cuMemGetAddressRange

#include <climits>
#include <mutex>

#include "common.cuh"

#include "attn_rows.h" // ROWS_PAGE
#include "device_check.hpp"
#include "kv_pages.h"

namespace aaedn_dev
{

// ---------------------------------------------------------------------------
// Page copies. Pure traffic: 2 * page bytes a pair and array, bound by HBM.
// A CTA moves 16 KB of one page, each thread four 16-byte loads before its
// first store: four pages of 8 heads x 128 dims in 64 arrays (134 MB of
// traffic) 23 us, 5.9 TB/s.
// ---------------------------------------------------------------------------
constexpr int KC_THREADS = 256, KC_UNROLL = 4;

__device__ __forceinline__ void kv_copy_chunk(float* base, size_t page_floats, int n_pages, int src, int dst)
{
    if (src < 0 || src >= n_pages || dst < 0 || dst >= n_pages || src == dst)
        return;
    const float4* s = reinterpret_cast<const float4*>(base + (size_t)src * page_floats);
    float4* d = reinterpret_cast<float4*>(base + (size_t)dst * page_floats);
    const size_t n4 = page_floats / 4, i0 = (size_t)blockIdx.x * KC_THREADS * KC_UNROLL + threadIdx.x;
    float4 v[KC_UNROLL];
#pragma unroll
    for (int u = 0; u < KC_UNROLL; ++u)
        if (i0 + u * KC_THREADS < n4)
            v[u] = s[i0 + u * KC_THREADS];
#pragma unroll
    for (int u = 0; u < KC_UNROLL; ++u)
        if (i0 + u * KC_THREADS < n4)
            d[i0 + u * KC_THREADS] = v[u];
}

__global__ void __launch_bounds__(KC_THREADS) kv_copy_kernel(const KvArrays arrays, size_t page_floats, int n_pages,
                                                             const int* __restrict__ src, const int* __restrict__ dst)
{
    kv_copy_chunk(arrays.base[blockIdx.y], page_floats, n_pages, src[blockIdx.z], dst[blockIdx.z]);
}

__global__ void __launch_bounds__(KC_THREADS) kv_copy_host_kernel(const KvArrays arrays, size_t page_floats,
                                                                  int n_pages, const KvPairs pairs)
{
    kv_copy_chunk(arrays.base[blockIdx.y], page_floats, n_pages, pairs.src[blockIdx.z], pairs.dst[blockIdx.z]);
}

template <typename Fn>
static int for_arrays(float* const* arrays, size_t n_arrays, Fn&& fn)
{
    for (size_t a0 = 0; a0 < n_arrays; a0 += KV_MAX_ARRAYS)
    {
        KvArrays part;
        const size_t n = n_arrays - a0 < (size_t)KV_MAX_ARRAYS ? n_arrays - a0 : (size_t)KV_MAX_ARRAYS;
        for (size_t i = 0; i < (size_t)KV_MAX_ARRAYS; ++i)
            part.base[i] = i < n ? arrays[a0 + i] : nullptr;
        if (int rc = fn(part, (unsigned)n))
            return rc;
    }
    return AAEDN_OK;
}

static unsigned kv_copy_chunks(size_t page_floats)
{
    return (unsigned)((page_floats / 4 + KC_THREADS * KC_UNROLL - 1) / (KC_THREADS * KC_UNROLL));
}

int kv_copy_pages(float* const* arrays, size_t n_arrays, size_t page_floats, int n_pages, const int* d_src,
                  const int* d_dst, size_t n, cudaStream_t st)
{
    return for_arrays(arrays, n_arrays, [&](const KvArrays& part, unsigned na) -> int {
        for (size_t p0 = 0; p0 < n; p0 += 65535)
        {
            const unsigned np = (unsigned)(n - p0 < 65535 ? n - p0 : 65535);
            kv_copy_kernel<<<dim3(kv_copy_chunks(page_floats), na, np), KC_THREADS, 0, st>>>(part, page_floats, n_pages,
                                                                                           d_src + p0, d_dst + p0);
            AAEDN_LAUNCH_CHECK("kv_copy_kernel");
        }
        return AAEDN_OK;
    });
}

int kv_copy_pages_host(float* const* arrays, size_t n_arrays, size_t page_floats, int n_pages, const KvPairs& pairs,
                       int n, cudaStream_t st)
{
    return for_arrays(arrays, n_arrays, [&](const KvArrays& part, unsigned na) -> int {
        kv_copy_host_kernel<<<dim3(kv_copy_chunks(page_floats), na, (unsigned)n), KC_THREADS, 0, st>>>(
            part, page_floats, n_pages, pairs);
        AAEDN_LAUNCH_CHECK("kv_copy_host_kernel");
        return AAEDN_OK;
    });
}

// ---------------------------------------------------------------------------
// Compaction: slot base[s] + i takes the row of slot base[s] + keep[i], for
// the strictly ascending keep list of sequence s. keep[i] >= i, so a row is
// overwritten only by entries at or after the one that reads it: a thread
// owns one 16-byte column of every slot and walks the list in order, eight
// rows loaded before the eight stores, and no other thread touches its
// column. CTA (array, sequence). One layer's few rows are little work, so the
// launch is what costs: 16 sequences, 24 slots each, 8 heads x 128 dims in 64
// arrays 19 us, most of them the call on the host; a launch an array would be
// 64 of those.
// ---------------------------------------------------------------------------
constexpr int KP_THREADS = 256, KP_BATCH = 8;

__global__ void __launch_bounds__(KP_THREADS) kv_compact_kernel(const KvArrays arrays, const KvCompactArgs a)
{
    const int s = blockIdx.y;
    float* pool = arrays.base[blockIdx.x];
    const int k0 = max(a.keep_start[s], 0), n = min(max(a.keep_start[s + 1], 0), a.n_keep) - k0;
    const long long base = a.base[s], cap = (long long)a.pt_stride * ROWS_PAGE;
    const int* pt = a.page_table + (size_t)(a.seq_of ? a.seq_of[s] : s) * a.pt_stride;
    const int hd4 = a.head_dim >> 2;
    auto at = [&](long long slot, int h, int c) -> float4* {
        if (slot < 0 || slot >= cap)
            return nullptr;
        const int page = pt[slot / ROWS_PAGE];
        if (page < 0 || page >= a.n_pages)
            return nullptr;
        return reinterpret_cast<float4*>(
                   pool + (((size_t)page * a.n_kv + h) * ROWS_PAGE + (size_t)(slot % ROWS_PAGE)) * a.head_dim) + c;
    };
    for (int col = threadIdx.x; col < a.n_kv * hd4; col += KP_THREADS)
    {
        const int h = col / hd4, c = col - h * hd4;
        for (int i0 = 0; i0 < n; i0 += KP_BATCH)
        {
            float4 v[KP_BATCH];
            bool ok[KP_BATCH];
#pragma unroll
            for (int u = 0; u < KP_BATCH; ++u)
            {
                ok[u] = false;
                if (i0 + u < n)
                {
                    const int keep = a.keep[k0 + i0 + u];
                    const float4* p = keep == i0 + u ? nullptr : at(base + keep, h, c); // already in place
                    ok[u] = p != nullptr;
                    if (p)
                        v[u] = *p;
                }
            }
#pragma unroll
            for (int u = 0; u < KP_BATCH; ++u)
                if (ok[u])
                    if (float4* p = at(base + i0 + u, h, c))
                        *p = v[u];
        }
    }
}

int kv_compact(float* const* arrays, size_t n_arrays, const KvCompactArgs& a, cudaStream_t st)
{
    return for_arrays(arrays, n_arrays, [&](const KvArrays& part, unsigned na) -> int {
        kv_compact_kernel<<<dim3(na, (unsigned)a.n_seqs), KP_THREADS, 0, st>>>(part, a);
        AAEDN_LAUNCH_CHECK("kv_compact_kernel");
        return AAEDN_OK;
    });
}

} // namespace aaedn_dev

using namespace aaedn_dev;

// cuMemGetAddressRange of the driver, or null.
static PFN_cuMemGetAddressRange_v3020 range_fn()
{
    static PFN_cuMemGetAddressRange_v3020 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, []() {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuMemGetAddressRange", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuMemGetAddressRange_v3020>(p);
    });
    return fn;
}

static int check_arrays(const char* fn, float* const* h_arrays, size_t n_arrays, uint32_t n_pages)
{
    if (!h_arrays)
        return set_error(AAEDN_EINVAL, "%s: h_arrays is null", fn);
    if (n_arrays > 4096)
        return set_error(AAEDN_EINVAL, "%s: at most 4096 arrays (%zu)", fn, n_arrays);
    if (n_pages == 0 || n_pages > (uint32_t)INT_MAX)
        return set_error(AAEDN_EINVAL, "%s: n_pages %u", fn, n_pages);
    // pools are mostly parts of one allocation: its extent, asked for once,
    // vouches for the others in it (a query each took longer than the copies)
    uintptr_t lo = 0, hi = 0;
    const PFN_cuMemGetAddressRange_v3020 range = range_fn();
    for (size_t i = 0; i < n_arrays; ++i)
    {
        const uintptr_t p = reinterpret_cast<uintptr_t>(h_arrays[i]);
        if (p >= lo && p < hi && (p & 15) == 0)
            continue;
        if (int rc = check_device_ptr(fn, h_arrays[i], "an array", 16))
            return rc;
        CUdeviceptr base = 0;
        size_t size = 0;
        if (range && range(&base, &size, (CUdeviceptr)p) == CUDA_SUCCESS)
        {
            lo = (uintptr_t)base;
            hi = lo + size;
        }
    }
    return AAEDN_OK;
}

extern "C" int aaedn_cu_kv_copy_pages(float* const* h_arrays, size_t n_arrays, size_t page_floats, uint32_t n_pages,
                                      const int32_t* d_src, const int32_t* d_dst, size_t n, void* stream)
{
    const char* fn = "aaedn_cu_kv_copy_pages";
    if (n_arrays == 0 || n == 0 || page_floats == 0)
        return AAEDN_OK;
    if (page_floats % 4 || page_floats > ((size_t)1 << 31))
        return set_error(AAEDN_EINVAL, "%s: page_floats %zu is not a multiple of 4 up to 2^31", fn, page_floats);
    if (n > (size_t)INT_MAX)
        return set_error(AAEDN_EINVAL, "%s: %zu pairs", fn, n);
    int rc;
    if ((rc = check_arrays(fn, h_arrays, n_arrays, n_pages)) || (rc = check_device_ptr(fn, d_src, "d_src", 4)) ||
        (rc = check_device_ptr(fn, d_dst, "d_dst", 4)))
        return rc;
    return kv_copy_pages(h_arrays, n_arrays, page_floats, (int)n_pages, d_src, d_dst, n, as_stream(stream));
}

extern "C" int aaedn_cu_kv_compact(float* const* h_arrays, size_t n_arrays, uint32_t n_pages, uint32_t n_kv_heads,
                                   uint32_t head_dim, const int32_t* d_page_table, size_t pt_stride,
                                   const int32_t* d_base, const int32_t* d_keep, const int32_t* d_keep_start,
                                   size_t n_seqs, size_t n_keep, void* stream)
{
    const char* fn = "aaedn_cu_kv_compact";
    if (n_arrays == 0 || n_seqs == 0 || n_keep == 0)
        return AAEDN_OK;
    if (n_keep > (size_t)INT_MAX)
        return set_error(AAEDN_EINVAL, "%s: n_keep %zu", fn, n_keep);
    if (n_kv_heads == 0 || n_kv_heads > 65535 || head_dim == 0 || head_dim % 4 || head_dim > 1024)
        return set_error(AAEDN_EINVAL, "%s: n_kv_heads %u in 1..65535, head_dim %u a multiple of 4 in 4..1024", fn,
                         n_kv_heads, head_dim);
    if (n_seqs > 65535 || pt_stride == 0 || pt_stride > (size_t)(1 << 24))
        return set_error(AAEDN_EINVAL, "%s: at most 65535 sequences (%zu), pt_stride 1..2^24 (%zu)", fn, n_seqs,
                         pt_stride);
    int rc;
    if ((rc = check_arrays(fn, h_arrays, n_arrays, n_pages)) ||
        (rc = check_device_ptr(fn, d_page_table, "d_page_table", 4)) ||
        (rc = check_device_ptr(fn, d_base, "d_base", 4)) || (rc = check_device_ptr(fn, d_keep, "d_keep", 4)) ||
        (rc = check_device_ptr(fn, d_keep_start, "d_keep_start", 4)))
        return rc;
    KvCompactArgs a{};
    a.n_pages = (int)n_pages;
    a.n_kv = (int)n_kv_heads;
    a.head_dim = (int)head_dim;
    a.page_table = d_page_table;
    a.pt_stride = pt_stride;
    a.base = d_base;
    a.keep = d_keep;
    a.keep_start = d_keep_start;
    a.n_seqs = (int)n_seqs;
    a.n_keep = (int)n_keep;
    return kv_compact(h_arrays, n_arrays, a, as_stream(stream));
}

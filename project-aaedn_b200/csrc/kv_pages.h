// kv_pages.h — host interface of the cache page operators (kv_pages.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace aaedn_dev
{

constexpr int KV_MAX_ARRAYS = 256; // page pools (K and V of every layer) of one launch

struct KvArrays
{
    float* base[KV_MAX_ARRAYS];
};

// One page copy, by value for callers whose page numbers are on the host.
constexpr int KV_MAX_PAIRS = 64;
struct KvPairs
{
    int src[KV_MAX_PAIRS], dst[KV_MAX_PAIRS];
};

// page dst[i] = page src[i] in each of n_arrays pools, for i < n.
int kv_copy_pages(float* const* arrays, size_t n_arrays, size_t page_floats, int n_pages, const int* d_src,
                  const int* d_dst, size_t n, cudaStream_t st);
// The same for n <= KV_MAX_PAIRS pairs on the host.
int kv_copy_pages_host(float* const* arrays, size_t n_arrays, size_t page_floats, int n_pages, const KvPairs& pairs,
                       int n, cudaStream_t st);

struct KvCompactArgs
{
    int n_pages, n_kv, head_dim;
    const int* page_table;
    size_t pt_stride;
    const int* seq_of; // row of page_table of sequence s; null: s
    const int *base, *keep, *keep_start;
    int n_seqs;
    int n_keep; // entries of keep
};
int kv_compact(float* const* arrays, size_t n_arrays, const KvCompactArgs& a, cudaStream_t st);

} // namespace aaedn_dev

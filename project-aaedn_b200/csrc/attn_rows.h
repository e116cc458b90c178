// attn_rows.h — host interface of the attention of packed query rows over a
// paged K/V cache (attn_rows.cu): the rows of several sequences in one call,
// causal (prompts and continued chats) or under a tree mask (drafted tokens).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace aaedn_dev
{

constexpr int ROWS_PAGE = 64; // tokens of a cache page

// Sequence s owns the query rows [row_start[s], row_start[s + 1]); its row r
// is the token in cache slot past[s] + r and attends
//   causal (mask null): the slots 0 .. past[s] + r;
//   tree:   the slots below past[s], and slot past[s] + j for every bit j of
//           its mask words (bit j % 64 of word j / 64).
// The slots' K and V rows are in the pages that page_table[s] lists. All
// arrays are in device memory; the kernels bound what they read by rows,
// pt_stride and n_pages whatever the arrays hold.
struct AttnRowsArgs
{
    const float* q; // [rows][ldq]: n_heads * head_dim floats of every row
    size_t ldq;
    const float *k, *v; // [n_pages][n_kv][ROWS_PAGE][head_dim]
    const int* page_table; // [n_seqs][pt_stride]
    size_t pt_stride;
    const int* seq_of; // row of page_table of sequence s; null: s
    int n_pages;
    const int *row_start, *past; // [n_seqs + 1], [n_seqs]
    int n_seqs, rows;
    const uint64_t* mask; // [rows][mask_words], or null: causal
    int mask_words;
    int n_heads, n_kv, head_dim;
    float scale;
    float* out; // [rows][ldo]
    size_t ldo;
    void* workspace; // AAEDN_ATTN_ROWS_WORKSPACE_BYTES
    unsigned* err;   // device word set to 1 when a bounded wait ran out; null: the library's own word
};

int attn_rows(const AttnRowsArgs& a, cudaStream_t st);
// Sets the kernels' attributes on the current device (before a capture).
int attn_rows_init();
// Reads and clears the library's own word on the current device:
// AAEDN_ETIMEOUT when a bounded wait ran out since the last check.
int attn_rows_err_check();

} // namespace aaedn_dev

// sample_rows.h — host interface of the many-row sampler (sample_rows.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace aaedn_dev
{

struct SampleRowsArgs
{
    const float* logits; // [rows][ld]
    size_t ld;
    uint32_t rows, vocab;
    const float* temperature; // [rows] or null: 1
    const int* top_k;         // [rows] or null: off; <= 0 or >= vocab: off
    const float* top_p;       // [rows] or null: off; >= 1: off
    const float* min_p;       // [rows] or null: off; <= 0: off
    const float* u;           // [rows]
    uint32_t* tokens;         // [rows]
};

constexpr uint32_t SR_MAX_VOCAB = 1000000; // a row's mass stays below 2^64 units (sample_rows.cu)

int sample_rows(const SampleRowsArgs& a, cudaStream_t st);

} // namespace aaedn_dev

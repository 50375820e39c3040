// Launch interface of the scores of logits (logprobs.cu) for the C ABI.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace dsv41 {

constexpr int kMaxTop = 32;       // alternatives of a row
constexpr int kMaxGiven = 1024;   // given tokens of a row

struct LogprobParams {
    const void* logits;       // [rows][row_stride], vocab columns
    int64_t row_stride;       // elements
    const int64_t* tokens;    // [rows][given]
    int rows, vocab, given, top;
    float *logprobs, *entropy, *lse;   // [rows][given], [rows], [rows]
    int64_t* top_ids;         // [rows][top]
    float* top_logprobs;      // [rows][top]
};

// dtype 0 fp16, 1 bf16, 2 fp32
cudaError_t launch_logprobs(const LogprobParams& p, int dtype, cudaStream_t st);

}  // namespace dsv41

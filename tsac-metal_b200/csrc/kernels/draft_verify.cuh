// Verification of drafted tokens (draft_verify.cu); the rule is stated in
// include/tsac_cuda.h.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace tsacb::dev
{
constexpr int DRAFT_MAX_NODES = 64;

enum class ValueType : int
{
    bf16 = 0,
    fp16 = 1,
    fp32 = 2
};

struct VerifyArgs
{
    const void* target;                     // [batch][nodes][vocab], unit stride over the vocabulary
    const void* draft;                      // the same, or null
    long long target_batch, target_node;    // strides in elements
    long long draft_batch, draft_node;
    const int* tokens;                      // [batch][max_nodes]
    const int* parents;                     // [batch][max_nodes]
    const float* coins;                     // [batch][max_nodes]
    const float* draws;                     // [batch]
    const int* nodes;                       // [batch] or null: max_nodes each
    int* accepted;                          // [batch]
    int* path;                              // [batch][max_nodes]
    int* token;                             // [batch]
    int vocab, max_nodes;
    unsigned* error_word;
};

cudaError_t draft_verify(const VerifyArgs& a, ValueType type, int batch, cudaStream_t stream);
} // namespace tsacb::dev

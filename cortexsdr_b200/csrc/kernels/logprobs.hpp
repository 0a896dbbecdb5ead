// Launcher of the log probabilities of given tokens (logprobs.cu). Asynchronous on the context's stream.
#pragma once

#include <cstddef>
#include <cstdint>

#include "../internal.hpp"

namespace csdr {

constexpr uint32_t kMaxTop = 32;

struct LogprobArgs {
    const void* logits;
    size_t stride;              // elements between rows
    uint32_t rows, vocab;
    const int32_t* targets;     // may be null
    float *logprob, *entropy;   // rows; may be null
    uint32_t top;
    int32_t* top_ids;           // rows x top
    float* top_logprobs;
};
void launch_logprobs(csdr_context* ctx, int dtype, const LogprobArgs& a);

}  // namespace csdr

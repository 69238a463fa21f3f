// The rules on logits as the entry point (logits.cu) and the runtime's greedy loop call them.
#pragma once
#include <cuda_runtime.h>
#include "b200p.h"

namespace b200p {

constexpr int kMostBias = 1024;                  // entries of a row's bias list

// b200p_logits_adjust after its checks of arguments.  length_stride: distance between the rows' entries of prompt_lengths and
// token_lengths, 1 or (one length for all rows) 0.
int logits_adjust(const void* in, void* out, const b200p_logits_args* a, int prompt_length_stride, int token_length_stride, cudaStream_t st);

} // namespace b200p

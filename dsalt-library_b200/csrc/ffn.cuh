// Stages of the gated feed-forward block, in the order a training step runs them.
#pragma once

#include "common.cuh"

namespace dsalt {
enum FfnStage { FFN_HIDDEN = 0, FFN_OUT = 1, FFN_BWD_HIDDEN = 2, FFN_BWD_INPUT = 3, FFN_BWD_WEIGHTS = 4 };
// any number of tokens, tensor cores (ffn_tc.cu); early: the launch before it in the
// stream is another of these stages, beside whose end it may start
cudaError_t launch_ffn_tc(int stage, const DsaltGatedFfnParams& p, bool early, cudaStream_t st);
// the forward for few tokens (ffn_few.cu): both stages, the second launched early
bool ffn_few_tokens(const DsaltGatedFfnParams& p);
cudaError_t launch_ffn_few(const DsaltGatedFfnParams& p, cudaStream_t st);
}  // namespace dsalt

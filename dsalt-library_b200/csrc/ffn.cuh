// Stages of the gated feed-forward block (ffn_tc.cu), in the order a training step runs them.
#pragma once

#include "common.cuh"

namespace dsalt {
enum FfnStage { FFN_HIDDEN = 0, FFN_OUT = 1, FFN_BWD_HIDDEN = 2, FFN_BWD_INPUT = 3, FFN_BWD_WEIGHTS = 4 };
cudaError_t launch_ffn(int stage, const DsaltGatedFfnParams& p, cudaStream_t st);
}  // namespace dsalt

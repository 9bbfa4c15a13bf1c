// Stages of the gated feed-forward block, in the order a training step runs them.
#pragma once

#include "common.cuh"

namespace dsalt {
enum FfnStage { FFN_HIDDEN = 0, FFN_OUT = 1, FFN_BWD_HIDDEN = 2, FFN_BWD_INPUT = 3, FFN_BWD_WEIGHTS = 4 };
// any number of tokens, tensor cores (ffn_tc.cu); early: the launch before it in the
// stream is another of these stages, beside whose end it may start
cudaError_t launch_ffn_tc(int stage, const DsaltGatedFfnParams& p, bool early, cudaStream_t st);
// the forward for a handful of tokens (ffn_few.cu) and for up to kMidTokens (ffn_mid.cu):
// both stages, the second launched early.  Measured, at this width alone (us, the forward in
// a replayed graph, bf16, d = 1024, F = 2816): one token 7.3 few; 16: 9.6 few; 24: 13.7 mid, 14.4 few;
// 64: 16.3 mid, 28 few; 256: 20.3 mid, 24 tc; 384: 23.1 mid, 26.8 tc; 512: 30.8 mid, 26.8 tc.
constexpr int kFewTokens = 16, kMidTokens = 384;
cudaError_t launch_ffn_few(const DsaltGatedFfnParams& p, cudaStream_t st);
cudaError_t launch_ffn_mid(const DsaltGatedFfnParams& p, cudaStream_t st);
// h_lo is used: up to DSALT_FFN_FEW_TOKENS tokens
inline bool ffn_two_words(const DsaltGatedFfnParams& p) { return p.T <= DSALT_FFN_FEW_TOKENS; }
}  // namespace dsalt

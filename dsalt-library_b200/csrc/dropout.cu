// Dropout whose mask is computed from (seed, site, element index) and never stored
// (dropout.cuh): y = keep ? x·65536 / (65536 − threshold) : 0.  The backward is the
// same pass over the gradient.  A dropped element is 0 whatever x holds there.  y may be x:
// a thread reads its elements before it writes them, and not by the read-only path.
// Bound: one read and one write of the tensor.
#include "dropout.cuh"

namespace dsalt {
namespace {

constexpr int kThreads = 256;

// A thread takes kBlocks blocks of eight elements (a counter's draws each), a CTA's
// width apart, with their loads out before the first draw: four for tensors that fill
// the device that way (16384 × 1024 bf16: 16 us, 18 with one, before the draws selected
// values), one for small tensors (613 × 1001 fp32: 2.4 us, 4.2 with four).  The large
// pass takes 12.9 us with x and y in L2 (a copy of the tensor 9.0; 14.2 with masks built and
// applied, before x was read by ordinary loads: 0.2) and 13.8 in a step's two passes over four tensors.
template <typename T, bool VEC, int kBlocks>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const DsaltDropoutParams p) {
  const int64_t first = ((int64_t)blockIdx.x * kBlocks * kThreads + threadIdx.x) * 8;
  Dropout dr;
  dr.init(p.seed, p.site, p.threshold);
  const T* x = reinterpret_cast<const T*>(p.x);
  T* y = reinterpret_cast<T*>(p.y);
  const f2 scale = pair(dr.scale, dr.scale);
  auto drop = [&](auto& raw, int64_t i) {
    float e[8];
    f2 v[4];
    raw.get(v);
#pragma unroll
    for (int j = 0; j < 4; ++j) unpair(mul2(v[j], scale), e[2 * j], e[2 * j + 1]);
    dr.select_block((uint64_t)i >> 3, e);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = pair(e[2 * j], e[2 * j + 1]);
    raw.set(v);
  };
  if (VEC && first + ((kBlocks - 1) * kThreads + 1) * 8 <= p.n) {
    Raw<T, true> raw[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) raw[b].load_in_place(x + first + b * kThreads * 8);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      drop(raw[b], first + b * kThreads * 8);
      raw[b].store(y + first + b * kThreads * 8, 8);
    }
    return;
  }
  for (int64_t i = first; i < p.n && i <= first + (kBlocks - 1) * kThreads * 8; i += kThreads * 8) {
    const int left = (int)min((int64_t)8, p.n - i);
    Raw<T, false> raw;
    raw.load(x + i, left);
    drop(raw, i);
    raw.store(y + i, left);
  }
}

template <typename T, int kBlocks>
cudaError_t launch_blocks(const DsaltDropoutParams& p, cudaStream_t st) {
  const bool vec = ((uintptr_t)p.x & 15) == 0 && ((uintptr_t)p.y & 15) == 0;
  const int64_t per_cta = 8 * kBlocks * kThreads;
  const unsigned grid = (unsigned)((p.n + per_cta - 1) / per_cta);
  if (vec) dropout_kernel<T, true, kBlocks><<<grid, kThreads, 0, st>>>(p);
  else dropout_kernel<T, false, kBlocks><<<grid, kThreads, 0, st>>>(p);
  return cudaGetLastError();
}

constexpr int64_t kLarge = (int64_t)8 * kThreads * 148 * 8;  // eight CTAs of one block for each of 148 SMs

template <typename T>
cudaError_t launch_t(const DsaltDropoutParams& p, cudaStream_t st) {
  return p.n >= kLarge ? launch_blocks<T, 4>(p, st) : launch_blocks<T, 1>(p, st);
}

}  // namespace

cudaError_t launch_dropout(const DsaltDropoutParams& p, cudaStream_t st) {
  switch (p.dtype) {
    case DSALT_BF16: return launch_t<__nv_bfloat16>(p, st);
    case DSALT_F16: return launch_t<__half>(p, st);
    case DSALT_F32: return launch_t<float>(p, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace dsalt

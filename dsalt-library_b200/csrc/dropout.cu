// Dropout whose mask is computed from (seed, site, element index) and never stored
// (dropout.cuh): y = keep ? x·65536 / (65536 − threshold) : 0.  The backward is the
// same pass over the gradient.  A dropped element is 0 whatever x holds there.
// Bound: one read and one write of the tensor.
#include "dropout.cuh"

namespace dsalt {
namespace {

constexpr int kThreads = 256;

// one thread per eight elements, a block of the generator
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const DsaltDropoutParams p) {
  const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 8;
  if (i >= p.n) return;
  Dropout dr;
  dr.init(p.seed, p.site, p.threshold);
  const T* x = reinterpret_cast<const T*>(p.x) + i;
  T* y = reinterpret_cast<T*>(p.y) + i;
  const int left = (int)min((int64_t)8, p.n - i);
  const uint32_t keep = dr.keep_block((uint64_t)i >> 3);
  float v[8];
  if (VEC && left == 8) {
    load8<T, true>(x, 8, v);
  } else {
    load8<T, false>(x, left, v);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (keep >> j & 1u) ? v[j] * dr.scale : 0.f;
  if (VEC && left == 8) {
    store8<T, true>(y, 8, v);
  } else {
    store8<T, false>(y, left, v);
  }
}

template <typename T>
cudaError_t launch_t(const DsaltDropoutParams& p, cudaStream_t st) {
  const bool vec = ((uintptr_t)p.x & 15) == 0 && ((uintptr_t)p.y & 15) == 0;
  const unsigned grid = (unsigned)((p.n + 8 * kThreads - 1) / (8 * kThreads));
  if (vec) dropout_kernel<T, true><<<grid, kThreads, 0, st>>>(p);
  else dropout_kernel<T, false><<<grid, kThreads, 0, st>>>(p);
  return cudaGetLastError();
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

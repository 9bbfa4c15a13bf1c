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
  uint32_t m[8];
  dr.masks_block((uint64_t)i >> 3, m);
  const f2 scale = pair(dr.scale, dr.scale);
  auto drop = [&](auto raw) {
    f2 v[4];
    raw.load(x, left);
    raw.get(v);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = mul2(and2(v[j], m[2 * j], m[2 * j + 1]), scale);
    raw.set(v);
    raw.store(y, left);
  };
  if (VEC && left == 8) drop(Raw<T, true>());
  else drop(Raw<T, false>());
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

// Dropout draws from a counter-based generator: the mask is a function of (seed,
// site, element index), so it is computed again wherever it is needed and never stored.
#pragma once

#include "common.cuh"

namespace dsalt {

// Philox4x32-10 of Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy
// as 1, 2, 3" (SC 2011): ten rounds of two 32 × 32 → 64 bit products with Weyl keys.
__device__ __forceinline__ uint4 philox(uint4 c, uint2 k) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)c.x * 0xD2511F53u, p1 = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(p1 >> 32) ^ c.y ^ k.x, (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c.w ^ k.y, (uint32_t)p0);
    k.x += 0x9E3779B9u;
    k.y += 0xBB67AE85u;
  }
  return c;
}

// One counter gives the 16-bit draws of eight consecutive elements: half the
// generator's work of 32-bit draws, which would cost more issue slots than the
// element's memory traffic leaves; a dropout rate is then a multiple of 2^-16.
struct Dropout {
  uint2 key;
  uint32_t site, threshold;
  float scale;  // 1 / share kept (0 when nothing is)

  __device__ __forceinline__ void init(const int64_t* seed, uint32_t site_, int threshold_) {
    threshold = (uint32_t)threshold_;
    site = site_;
    scale = threshold_ >= 65536 ? 0.f : 65536.f / (float)(65536 - threshold_);
    const uint64_t s = threshold_ > 0 ? (uint64_t)__ldg(seed) : 0;
    key = make_uint2((uint32_t)s, (uint32_t)(s >> 32));
  }
  // bit j: element 8·block + j is kept
  __device__ __forceinline__ uint32_t keep_block(uint64_t block) const {
    const uint4 w = philox(make_uint4((uint32_t)block, (uint32_t)(block >> 32), site, 0u), key);
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m |= (uint32_t)((v[j] & 0xffffu) >= threshold) << (2 * j);
      m |= (uint32_t)((v[j] >> 16) >= threshold) << (2 * j + 1);
    }
    return m;
  }
  // bit j: element i + j is kept, 0 ≤ j < 8, any i
  __device__ __forceinline__ uint32_t keep8(uint64_t i) const {
    const uint32_t o = (uint32_t)i & 7u;
    uint32_t m = keep_block(i >> 3);
    if (o) m = (m | keep_block((i >> 3) + 1) << 8) >> o;
    return m;
  }
};

// ------------------------------------------------- eight consecutive elements
// VEC: aligned 16-byte accesses and all eight inside; else element by element,
// those at or past n (counted from the first) left out and read as 0.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int n, float* v) {
  if constexpr (VEC && sizeof(T) == 2) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(e[j]);
  } else if constexpr (VEC) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? to_f32<T>(p[j]) : 0.f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int n, const float* v) {
  if constexpr (VEC && sizeof(T) == 2) {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = from_f32<T>(v[j]);
    *reinterpret_cast<uint4*>(p) = u;
  } else if constexpr (VEC) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = from_f32<T>(v[j]);
  }
}

}  // namespace dsalt

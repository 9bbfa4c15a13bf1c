// Dropout draws from a counter-based generator: the mask is a function of (seed,
// site, element index), so it is computed again wherever it is needed and never stored.
#pragma once

#include <type_traits>

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
  // the draws of elements 8·block … 8·block + 7
  __device__ __forceinline__ uint4 draws(uint64_t block) const {
    return philox(make_uint4((uint32_t)block, (uint32_t)(block >> 32), site, 0u), key);
  }
  // v, 8·block … 8·block + 7, with 0 where dropped
  __device__ __forceinline__ void select_block(uint64_t block, float* v) const {
    const uint4 w = draws(block);
    const uint32_t d[4] = {w.x, w.y, w.z, w.w};
    const uint32_t high = threshold << 16;
    const bool some = threshold < 65536;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = some && (d[j] << 16) >= high ? v[2 * j] : 0.f;
      v[2 * j + 1] = some && d[j] >= high ? v[2 * j + 1] : 0.f;
    }
  }
  // m[j] = all ones where element 8·block + j is kept, 0 where it is dropped
  __device__ __forceinline__ void masks_block(uint64_t block, uint32_t* m) const {
    const uint4 w = draws(block);
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    if (threshold >= 65536) {
#pragma unroll
      for (int j = 0; j < 8; ++j) m[j] = 0u;
      return;
    }
    const uint32_t high = threshold << 16;  // draw >= threshold, compared in the upper halves
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[2 * j] = (v[j] << 16) >= high ? 0xffffffffu : 0u;
      m[2 * j + 1] = v[j] >= high ? 0xffffffffu : 0u;
    }
  }
  // the masks of elements i … i + 7, any i: of two blocks as bits, shifted into place
  __device__ __forceinline__ void masks8(uint64_t i, uint32_t* m) const {
    const uint32_t o = (uint32_t)i & 7u;
    uint32_t bits = 0;
    masks_block(i >> 3, m);
#pragma unroll
    for (int j = 0; j < 8; ++j) bits |= m[j] & (1u << j);
    if (o) {
      masks_block((i >> 3) + 1, m);
#pragma unroll
      for (int j = 0; j < 8; ++j) bits |= m[j] & (256u << j);
    }
    bits >>= o;
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = (uint32_t)((int32_t)(bits << (31 - j)) >> 31);
  }
};

// Pairs of fp32 values for the packed fp32 instructions of sm_100.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pair(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 and2(f2 v, uint32_t m0, uint32_t m1) { return v & ((f2)m1 << 32 | m0); }

// ------------------------------------------------- eight consecutive elements
// As they lie in memory, so that they can be on their way in few registers.  VEC:
// aligned 16-byte accesses and all eight inside; else element by element, those at or
// past n (counted from the first) read as 0 and not written.
template <typename T, bool VEC>
struct Raw {
  T e[8];
  __device__ __forceinline__ void load(const T* p, int n) {
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = j < n ? p[j] : from_f32<T>(0.f);
  }
  __device__ __forceinline__ void zero() { load(nullptr, 0); }
  __device__ __forceinline__ void get(f2* v) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = pair(to_f32<T>(e[2 * j]), to_f32<T>(e[2 * j + 1]));
  }
  __device__ __forceinline__ void set(const f2* v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      unpair(v[j], a, b);
      e[2 * j] = from_f32<T>(a);
      e[2 * j + 1] = from_f32<T>(b);
    }
  }
  __device__ __forceinline__ void store(T* p, int n) const {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = e[j];
  }
};
template <typename T>
struct Raw<T, true> {
  uint32_t w[2 * sizeof(T)];
  // through the read-only path: no launch still running writes what it reads
  __device__ __forceinline__ void load(const T* p, int) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) put(i, __ldg(reinterpret_cast<const uint4*>(p) + i));
  }
  // of what this thread writes next
  __device__ __forceinline__ void load_in_place(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) put(i, reinterpret_cast<const uint4*>(p)[i]);
  }
  __device__ __forceinline__ void put(int i, uint4 u) {
    w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)(2 * sizeof(T)); ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void get(f2* v) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        v[j] = pair(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        v[j] = pair(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
      } else {
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        v[j] = pair(h.x, h.y);
      }
    }
  }
  __device__ __forceinline__ void set(const f2* v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      unpair(v[j], a, b);
      if constexpr (sizeof(T) == 4) {
        w[2 * j] = __float_as_uint(a);
        w[2 * j + 1] = __float_as_uint(b);
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(a, b);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
  __device__ __forceinline__ void store(T* p, int) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
};

}  // namespace dsalt

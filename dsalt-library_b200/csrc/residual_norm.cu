// Between a block and the next one, in one pass each way:
//   n  = f·rf·post (or f),  x' = R(x + D(scale⊙gate⊙n)),  h = R(x'·r·norm)
// with rf and r the inverse root mean squares of f and x', D the dropout of
// dropout.cuh and R the rounding to the tensors' type.  h is the norm of the
// rounded x', the tensor that the next residual add and the backward see (as in
// rmsnorm.cu's fused add).  Backward:
//   G = dx_new + r·(dh⊙norm − x'·r²·mean(dh⊙norm⊙x')),  dx = R(G),  dn = D(G)⊙scale⊙gate,
//   df = R(rf·(dn⊙post − f·rf²·mean(dn⊙post⊙f))),  dgate = D(G)⊙scale⊙n,
//   dscale = Σ_t D(G)⊙gate⊙n,  dpost = Σ_t dn⊙f·rf,  dnorm = Σ_t dh⊙x'·r.
// Everything between the loads and the stores is fp32.  Bound: the rows' bytes,
// once in and once out.
//
// A row belongs to a group of threads of eight consecutive columns each: 8, 16 or
// 32 lanes of a warp up to d = 256, else a whole CTA of ceil(d / 256) warps (two
// chunks of columns a thread past d = 8192).  A group walks rows of the grid's
// stride, its weights and column sums in registers; the sums of a group go to one
// partial row and a second kernel adds the partial rows in order.
#include "dropout.cuh"

namespace dsalt {
namespace {

constexpr int kSmallThreads = 128;  // CTA of several row groups (d <= 256)

struct Shape {
  int group;   // threads of a row
  int cta;     // threads of a CTA
  int chunks;  // 8-column chunks of a thread
};
inline Shape shape_of(int d) {
  const int units = (d + 7) / 8;
  if (units <= 8) return {8, kSmallThreads, 1};
  if (units <= 16) return {16, kSmallThreads, 1};
  if (units <= 32) return {32, kSmallThreads, 1};
  const int chunks = units <= 1024 ? 1 : 2;
  const int t = ((units + chunks - 1) / chunks + 31) / 32 * 32;
  return {t, t, chunks};
}

// Sums over the row group: NV values at once; every thread gets the totals.
template <int NV>
__device__ __forceinline__ void group_sum(float (&v)[NV], int group, float* red) {
#pragma unroll
  for (int k = 0; k < NV; ++k)
    for (int o = min(group, 32) / 2; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if (group <= 32) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = group >> 5;
  __syncthreads();  // the previous totals are read
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < NV; ++k) red[warp * NV + k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    float s = lane < nw ? red[lane * NV + k] : 0.f;
    v[k] = warp_sum(s);
  }
}

template <typename T>
__device__ __forceinline__ void load_weights(const void* w, bool f32, int c, int d, float* v) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    v[j] = c + j < d ? (f32 ? __ldg(reinterpret_cast<const float*>(w) + c + j)
                            : to_f32<T>(reinterpret_cast<const T*>(w)[c + j]))
                     : 0.f;
}

template <typename T, int CH, bool VEC>
__global__ void __launch_bounds__(1024) residual_fwd_kernel(const DsaltResidualNormParams p, int group) {
  __shared__ float red[32];
  const int gid = threadIdx.x / group, lane = threadIdx.x - gid * group;
  const int64_t groups = (int64_t)gridDim.x * (blockDim.x / group);
  const int64_t first = (int64_t)blockIdx.x * (blockDim.x / group) + gid;
  Dropout dr;
  dr.init(p.seed, p.site, p.threshold);
  const T* X = reinterpret_cast<const T*>(p.x);
  const T* Fv = reinterpret_cast<const T*>(p.f);
  const T* Gt = reinterpret_cast<const T*>(p.gate);
  // every group of a CTA makes the same number of rounds (the sums synchronise)
  const int64_t rounds = (p.T - (int64_t)blockIdx.x * (blockDim.x / group) + groups - 1) / groups;
  for (int64_t k = 0; k < rounds; ++k) {
    const int64_t t = first + k * groups;
    const bool on = t < p.T;
    float f[CH][8], x[CH][8];
    float s[1] = {0.f};
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (lane + ch * group) * 8;
      const bool in = on && c < p.d;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[ch][j] = x[ch][j] = 0.f;
      if (!in) continue;
      load8<T, VEC>(Fv + t * p.d + c, p.d - c, f[ch]);
      load8<T, VEC>(X + t * p.d + c, p.d - c, x[ch]);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] = fmaf(f[ch][j], f[ch][j], s[0]);
    }
    float rf = 1.f;
    if (p.post) {
      group_sum(s, group, red);
      rf = rsqrtf(s[0] / (float)p.d + p.eps);
      if (on && lane == 0 && p.rf) p.rf[t] = rf;
    }
    const float gt = p.gate_mode == DSALT_GATE_TOKEN && on ? to_f32<T>(Gt[t]) : 1.f;
    s[0] = 0.f;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (lane + ch * group) * 8;
      if (!(on && c < p.d)) continue;
      float w[8];
      if (p.post) {
        load_weights<T>(p.post, p.w_f32, c, p.d, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[ch][j] = f[ch][j] * rf * w[j];
      }
      if (p.scale) {
        load_weights<T>(p.scale, p.w_f32, c, p.d, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[ch][j] *= w[j];
      }
      if (p.gate_mode == DSALT_GATE_FULL) {
        load8<T, VEC>(Gt + t * p.d + c, p.d - c, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[ch][j] *= w[j];
      } else if (p.gate_mode == DSALT_GATE_TOKEN) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[ch][j] *= gt;
      }
      const uint32_t keep = p.threshold > 0 ? dr.keep8((uint64_t)(t * p.d + c)) : 0xffu;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[ch][j] = round_to<T>((keep >> j & 1u) ? fmaf(f[ch][j], dr.scale, x[ch][j]) : x[ch][j]);
        s[0] = fmaf(x[ch][j], x[ch][j], s[0]);
      }
      store8<T, VEC>(reinterpret_cast<T*>(p.x_new) + t * p.d + c, p.d - c, x[ch]);
    }
    if (p.norm) {
      group_sum(s, group, red);
      const float r = rsqrtf(s[0] / (float)p.d + p.eps);
      if (on && lane == 0 && p.r) p.r[t] = r;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const int c = (lane + ch * group) * 8;
        if (!(on && c < p.d)) continue;
        float w[8];
        load_weights<T>(p.norm, p.w_f32, c, p.d, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = x[ch][j] * r * w[j];
        store8<T, VEC>(reinterpret_cast<T*>(p.h) + t * p.d + c, p.d - c, w);
      }
    }
  }
}

template <typename T, int CH, bool VEC>
__global__ void __launch_bounds__(1024) residual_bwd_kernel(const DsaltResidualNormParams p, int group) {
  __shared__ float red[64];
  const int gid = threadIdx.x / group, lane = threadIdx.x - gid * group;
  const int64_t groups = (int64_t)gridDim.x * (blockDim.x / group);
  const int64_t first = (int64_t)blockIdx.x * (blockDim.x / group) + gid;
  Dropout dr;
  dr.init(p.seed, p.site, p.threshold);
  const T* Fv = reinterpret_cast<const T*>(p.f);
  const T* Xn = reinterpret_cast<const T*>(p.x_new);
  const T* Gt = reinterpret_cast<const T*>(p.gate);
  const bool with_h = p.norm && p.dh;
  float a_scale[CH][8], a_post[CH][8], a_norm[CH][8];
#pragma unroll
  for (int ch = 0; ch < CH; ++ch)
#pragma unroll
    for (int j = 0; j < 8; ++j) a_scale[ch][j] = a_post[ch][j] = a_norm[ch][j] = 0.f;
  const int64_t rounds = (p.T - (int64_t)blockIdx.x * (blockDim.x / group) + groups - 1) / groups;
  for (int64_t k = 0; k < rounds; ++k) {
    const int64_t t = first + k * groups;
    const bool on = t < p.T;
    float g[CH][8], x[CH][8];  // G in the end; x'
    const float r = with_h && on ? __ldg(p.r + t) : 0.f;
    const float rf = p.post && on ? __ldg(p.rf + t) : 1.f;
    if (with_h) {
      float s[1] = {0.f};
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const int c = (lane + ch * group) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) g[ch][j] = x[ch][j] = 0.f;
        if (!(on && c < p.d)) continue;
        float w[8];
        load8<T, VEC>(Xn + t * p.d + c, p.d - c, x[ch]);
        load8<T, VEC>(reinterpret_cast<const T*>(p.dh) + t * p.d + c, p.d - c, g[ch]);
        load_weights<T>(p.norm, p.w_f32, c, p.d, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          a_norm[ch][j] = fmaf(g[ch][j], x[ch][j] * r, a_norm[ch][j]);
          g[ch][j] *= w[j];
          s[0] = fmaf(g[ch][j], x[ch][j], s[0]);
        }
      }
      group_sum(s, group, red);
      const float m = r * r * s[0] / (float)p.d;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int j = 0; j < 8; ++j) g[ch][j] = r * fmaf(-x[ch][j], m, g[ch][j]);
    } else {
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int j = 0; j < 8; ++j) g[ch][j] = 0.f;
    }
    const float gt = p.gate_mode == DSALT_GATE_TOKEN && on ? to_f32<T>(Gt[t]) : 1.f;
    float f[CH][8];
    float s[2] = {0.f, 0.f};  // Σ dn·post·f, Σ D(G)·scale·n
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (lane + ch * group) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[ch][j] = 0.f;
      if (!(on && c < p.d)) continue;
      const int64_t at = t * p.d + c;
      float w[8], post[8], gate[8], scale[8];
      if (p.dx_new) {
        load8<T, VEC>(reinterpret_cast<const T*>(p.dx_new) + at, p.d - c, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[ch][j] += w[j];
      }
      store8<T, VEC>(reinterpret_cast<T*>(p.dx) + at, p.d - c, g[ch]);
      load8<T, VEC>(Fv + at, p.d - c, f[ch]);
      if (p.post) load_weights<T>(p.post, p.w_f32, c, p.d, post);
      if (p.scale) load_weights<T>(p.scale, p.w_f32, c, p.d, scale);
      if (p.gate_mode == DSALT_GATE_FULL) load8<T, VEC>(Gt + at, p.d - c, gate);
      const uint32_t keep = p.threshold > 0 ? dr.keep8((uint64_t)at) : 0xffu;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // a dropped element passes nothing back, whatever f holds there
        const bool kept = (keep >> j & 1u) && (VEC || c + j < p.d);
        const float da = kept ? g[ch][j] * dr.scale : 0.f;
        const float fr = f[ch][j] * rf;
        const float n = p.post ? fr * post[j] : fr;
        const float sc = p.scale ? scale[j] : 1.f;
        const float ga = p.gate_mode == DSALT_GATE_FULL ? gate[j] : gt;
        const float dn = da * sc * ga;
        const float dgn = kept ? da * n : 0.f;
        a_scale[ch][j] = fmaf(dgn, ga, a_scale[ch][j]);
        if (kept) a_post[ch][j] = fmaf(dn, fr, a_post[ch][j]);
        w[j] = dgn * sc;  // dgate of a full gate
        g[ch][j] = p.post ? dn * post[j] : dn;
        s[0] = fmaf(g[ch][j], f[ch][j], s[0]);
        s[1] += w[j];
      }
      if (p.gate_mode == DSALT_GATE_FULL) store8<T, VEC>(reinterpret_cast<T*>(p.dgate) + at, p.d - c, w);
    }
    if (p.post || p.gate_mode == DSALT_GATE_TOKEN) group_sum(s, group, red);
    if (p.gate_mode == DSALT_GATE_TOKEN && on && lane == 0) reinterpret_cast<T*>(p.dgate)[t] = from_f32<T>(s[1]);
    const float m = rf * rf * s[0] / (float)p.d;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (lane + ch * group) * 8;
      if (!(on && c < p.d)) continue;
      if (p.post) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[ch][j] = rf * fmaf(-f[ch][j], m, g[ch][j]);
      }
      store8<T, VEC>(reinterpret_cast<T*>(p.df) + t * p.d + c, p.d - c, g[ch]);
    }
  }
  // this group's sums: partial row `first` of [groups][3][d] (scale, post, norm)
  float* part = p.parts + first * 3 * p.d;
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
    const int c = (lane + ch * group) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (c + j >= p.d) continue;
      part[c + j] = a_scale[ch][j];
      part[p.d + c + j] = a_post[ch][j];
      part[2 * p.d + c + j] = a_norm[ch][j];
    }
  }
}

// Column sums of the partial rows in a fixed order: a CTA owns 32 columns of one of
// the three vectors; warp w adds rows w, w + 32, …, then the warps' sums in order.
template <typename T>
__global__ void __launch_bounds__(1024) residual_colsum_kernel(const DsaltResidualNormParams p, int64_t nparts) {
  void* out = blockIdx.y == 0 ? p.dscale : blockIdx.y == 1 ? p.dpost : p.dnorm;
  if (!out) return;
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float acc = 0.f;
  if (c < p.d)
#pragma unroll 8
    for (int64_t i = grp; i < nparts; i += 32) acc += __ldg(p.parts + (i * 3 + blockIdx.y) * p.d + c);
  s[grp][lane] = acc;
  __syncthreads();
  if (grp == 0 && c < p.d) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) v += s[w][lane];
    if (p.w_f32) reinterpret_cast<float*>(out)[c] = v;
    else reinterpret_cast<T*>(out)[c] = from_f32<T>(v);
  }
}

cudaError_t sm_count(int* out) {
  static int counts[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (counts[dev] <= 0) {
    e = cudaDeviceGetAttribute(&counts[dev], cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
  }
  *out = counts[dev];
  return cudaSuccess;
}

// CTAs of the backward: as many as run at once, no more than there are rows for
int bwd_ctas(int64_t T, const Shape& s, int sms) {
  const int per_cta = s.cta / s.group;
  const int64_t want = (T + per_cta - 1) / per_cta;
  const int64_t most = (int64_t)sms * (1024 / s.cta < 1 ? 1 : 1024 / s.cta);
  return (int)(want < most ? want : most);
}

template <typename T, int CH, bool VEC>
cudaError_t launch_v(const DsaltResidualNormParams& p, const Shape& s, bool bwd, cudaStream_t st) {
  int sms = 0;
  cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  const int per_cta = s.cta / s.group;
  if (!bwd) {
    const int64_t want = (p.T + per_cta - 1) / per_cta, most = (int64_t)sms * 2048 / s.cta;
    residual_fwd_kernel<T, CH, VEC><<<(unsigned)(want < most ? want : most), s.cta, 0, st>>>(p, s.group);
    return cudaGetLastError();
  }
  const int ctas = bwd_ctas(p.T, s, sms);
  residual_bwd_kernel<T, CH, VEC><<<ctas, s.cta, 0, st>>>(p, s.group);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if (p.dscale || p.dpost || p.dnorm) {
    residual_colsum_kernel<T><<<dim3((p.d + 31) / 32, 3), 1024, 0, st>>>(p, (int64_t)ctas * per_cta);
    e = cudaGetLastError();
  }
  return e;
}

template <typename T>
cudaError_t launch_t(const DsaltResidualNormParams& p, bool bwd, cudaStream_t st) {
  const Shape s = shape_of(p.d);
  bool vec = p.d % 8 == 0;
  for (const void* q : {p.x, p.f, (const void*)p.x_new, (const void*)p.h, p.dx_new, p.dh, (const void*)p.dx,
                        (const void*)p.df, p.gate_mode == DSALT_GATE_FULL ? p.gate : nullptr,
                        p.gate_mode == DSALT_GATE_FULL ? (const void*)p.dgate : nullptr})
    vec = vec && ((uintptr_t)q & 15) == 0;
  if (s.chunks == 1) return vec ? launch_v<T, 1, true>(p, s, bwd, st) : launch_v<T, 1, false>(p, s, bwd, st);
  return vec ? launch_v<T, 2, true>(p, s, bwd, st) : launch_v<T, 2, false>(p, s, bwd, st);
}

}  // namespace

cudaError_t residual_norm_parts(int64_t T, int d, int* out) {
  int sms = 0;
  const cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  const Shape s = shape_of(d);
  *out = bwd_ctas(T, s, sms) * (s.cta / s.group);
  return cudaSuccess;
}

cudaError_t launch_residual_norm(const DsaltResidualNormParams& p, bool bwd, cudaStream_t st) {
  switch (p.dtype) {
    case DSALT_BF16: return launch_t<__nv_bfloat16>(p, bwd, st);
    case DSALT_F16: return launch_t<__half>(p, bwd, st);
    case DSALT_F32: return launch_t<float>(p, bwd, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace dsalt

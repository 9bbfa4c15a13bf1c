// Between a block and the next one, in one pass each way:
//   n  = f·rf·post (or f),  s = x + D(scale⊙gate⊙n),  x' = R(s),  h = R(s·r·norm)
// with rf and r the inverse root mean squares of f and s, D the dropout of
// dropout.cuh and R the rounding to the tensors' type: h is the norm of the sum
// before its rounding, so that it is off by one rounding and not by two.  Backward, from
// the stored x' (rounded, with r of the sum before: dnorm and the projection in G see that
// rounding, a second one beside their own; s itself would be as many bytes again):
//   G = dx_new + r·(dh⊙norm − x'·r²·mean(dh⊙norm⊙x')),  dx = R(G),  dn = D(G)⊙scale⊙gate,
//   df = R(rf·(dn⊙post − f·rf²·mean(dn⊙post⊙f))),  dgate = D(G)⊙scale⊙n,
//   dscale = Σ_t D(G)⊙gate⊙n,  dpost = Σ_t dn⊙f·rf,  dnorm = Σ_t dh⊙x'·r.
// Everything between the loads and the stores is fp32.  Bound by the rows' bytes, once in
// and once out, and with dropout by issue slots (the generator's ten rounds a block of
// eight elements).  16384 × 1024 bf16 with every part, in replayed graphs: forward 41 us (31
// without dropout; 134 MB), backward with its column sums 65 us (53; 201 MB); fp32 forward
// 54 us (52), backward 76 us (72).  Under the profiler the bf16 kernels issue in 50 to 55 %
// of the cycles and use a quarter to two fifths of DRAM's rate: neither is full, the rest is
// latency, with 23 % (backward) and 43 % of an SM's warps resident.
//
// A row belongs to a group of threads of eight consecutive columns each: 8, 16 or
// 32 lanes of a warp up to d = 256, else a whole CTA (of one, two or four chunks of
// columns a thread).  A group walks rows of the grid's stride with the next row's loads
// on their way, its weights and column sums in registers; the sums of a CTA go to one
// partial row and a second kernel adds the partial rows in order.
//
// The backward works on the normed rows x̂ = x'·r and f̂ = f·rf, which stay near 1 whatever
// the rows' size: the cube of an inverse root mean square would leave fp32's range at rows
// of 1e13 (and, with a small eps, of 1e-13).  With q = dh⊙norm,
//   G = dx_new + r·(q − x̂·mean(q⊙x̂)),  df = rf·(dn⊙post − f̂·mean(dn⊙post⊙f̂)).
// It needs Σ q⊙x̂ before G, and Σ κ⊙G with κ = D⊙scale⊙post⊙f̂, times a full gate (for df
// and a token's dgate), after it.  G = u − e·x̂ with u = dx_new + r·q and e = r·mean(q⊙x̂)
// is linear in that first sum, so Σ κ⊙G = Σ κ⊙u − e·Σ κ⊙x̂: one round of three sums a row
// instead of two dependent rounds.  dscale and dpost share one sum over the rows,
// A = Σ_t D(G)⊙gate⊙f̂: dscale = post⊙A, dpost = scale⊙A.
#include <algorithm>

#include "device.cuh"
#include "dropout.cuh"

namespace dsalt {
namespace {

constexpr int kSmallThreads = 128;  // CTA of several row groups (d <= 256)

struct Shape {
  int group;   // threads of a row
  int cta;     // threads of a CTA
  int chunks;  // 8-column chunks of a thread
};
// Two chunks a thread past d = 4096, and from d = 512 on where rows are read element by
// element (16384 × 1001 bf16: 229 us instead of 276 with one, both before masks were shifted
// bits; 200 now); one elsewhere (16384 × 1024: 109 us instead of 117 with two, both before
// the forward selected instead of masking; 106 now).
inline Shape shape_of(int d, bool vec) {
  const int units = (d + 7) / 8;
  if (units <= 8) return {8, kSmallThreads, 1};
  if (units <= 16) return {16, kSmallThreads, 1};
  if (units <= 32) return {32, kSmallThreads, 1};
  const int chunks = units <= (vec ? 512 : 64) ? 1 : units <= 1024 ? 2 : 4;
  const int t = ((units + chunks - 1) / chunks + 31) / 32 * 32;
  return {t, t, chunks};
}

constexpr int kMaxWarps = 16;

// Sums over the row group, NV values at once; every thread gets the totals.  `red`: one
// of two halves that calls use in turn, so that a call needs one barrier: a half is
// written again only after the barrier of the call between.  A half has kMaxWarps
// entries of NV (3: 4) values; those past the group's warps stay 0.
template <int NV>
__device__ __forceinline__ void group_sum(float (&v)[NV], int group, float4* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < group)
#pragma unroll
      for (int k = 0; k < NV; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if (group <= 32) return;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    if constexpr (NV == 1) reinterpret_cast<float*>(red)[warp] = v[0];
    else red[warp] = make_float4(v[0], v[1], v[2], 0.f);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NV; ++k) v[k] = 0.f;
  for (int w = 0; w * 32 < group; w += 4) {
    if constexpr (NV == 1) {
      const float4 a = red[w / 4];
      v[0] += (a.x + a.y) + (a.z + a.w);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 a = red[w + i];
        v[0] += a.x;
        v[1] += a.y;
        v[2] += a.z;
      }
    }
  }
}

// weights of eight columns from c (1 without a vector, and past d)
template <typename T>
__device__ __forceinline__ void load_weights(const void* w, bool f32, int c, int d, float* v) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    v[j] = w && c + j < d ? (f32 ? __ldg(reinterpret_cast<const float*>(w) + c + j)
                                 : to_f32<T>(reinterpret_cast<const T*>(w)[c + j]))
                          : 1.f;
}
// post·scale·(1 / share kept) and norm of this thread's columns
template <typename T>
__device__ __forceinline__ void column_factors(const DsaltResidualNormParams& p, const Dropout& dr, int c, f2* branch,
                                               f2* norm) {
  float a[8], b[8];
  load_weights<T>(p.post, p.w_f32, c, p.d, a);
  load_weights<T>(p.scale, p.w_f32, c, p.d, b);
#pragma unroll
  for (int j = 0; j < 4; ++j) branch[j] = pair(a[2 * j] * b[2 * j] * dr.scale, a[2 * j + 1] * b[2 * j + 1] * dr.scale);
  load_weights<T>(p.norm, p.w_f32, c, p.d, a);
#pragma unroll
  for (int j = 0; j < 4; ++j) norm[j] = pair(a[2 * j], a[2 * j + 1]);
}
template <bool VEC, bool DROP>
__device__ __forceinline__ void row_masks(const Dropout& dr, int64_t at, uint32_t* m) {
  if constexpr (!DROP) {
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = 0xffffffffu;
  } else if constexpr (VEC) {
    dr.masks_block((uint64_t)at >> 3, m);
  } else {
    dr.masks8((uint64_t)at, m);
  }
}
__device__ __forceinline__ f2 dup(float v) { return pair(v, v); }
__device__ __forceinline__ float sum8(f2 s) {
  float a, b;
  unpair(s, a, b);
  return a + b;
}

// DROP, POST: the parts that cost most where they are not wanted.
template <typename T, int CH, bool VEC, int MAXT, bool DROP, bool POST>
__global__ void __launch_bounds__(MAXT, (CH == 1 ? 1024 : 512) / MAXT) residual_fwd_kernel(const DsaltResidualNormParams p, int group) {
  constexpr bool kHold = CH <= 2;  // weights in registers, the next row's loads early
  __shared__ float4 red[2][kMaxWarps / 4];
  if (threadIdx.x < 2 * kMaxWarps / 4) red[0][threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncthreads();
  const int gid = threadIdx.x / group, lane = threadIdx.x - gid * group, per_cta = blockDim.x / group;
  const int64_t stride = (int64_t)gridDim.x * per_cta;
  // every group of a CTA makes the same number of rounds (the sums synchronise)
  const int rounds = (int)((p.T - (int64_t)blockIdx.x * per_cta + stride - 1) / stride);
  Dropout dr;
  dr.init(p.seed, p.site, p.threshold);
  const T* X = reinterpret_cast<const T*>(p.x);
  const T* Fv = reinterpret_cast<const T*>(p.f);
  const T* Gt = reinterpret_cast<const T*>(p.gate);
  const float inv_d = 1.f / (float)p.d;
  f2 wbs[CH][4], wns[CH][4];
  if (kHold)
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) column_factors<T>(p, dr, (lane + ch * group) * 8, wbs[ch], wns[ch]);
  Raw<T, VEC> nx[CH], nf[CH];
  auto fetch = [&](int64_t t, int64_t row) {
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (lane + ch * group) * 8;
      if (t < p.T && c < p.d) {
        nx[ch].load(X + row + c, p.d - c);
        nf[ch].load(Fv + row + c, p.d - c);
      } else {
        nx[ch].zero();
        nf[ch].zero();
      }
    }
  };
  int64_t t = (int64_t)blockIdx.x * per_cta + gid;
  int64_t row = t * p.d;  // index of the row's first element
  fetch(t, row);
  for (int k = 0; k < rounds; ++k, t += stride, row += stride * p.d) {
    const bool on = t < p.T;
    f2 f[CH][4], x[CH][4], s2 = dup(0.f);
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      nf[ch].get(f[ch]);
      nx[ch].get(x[ch]);
#pragma unroll
      for (int j = 0; j < 4; ++j) s2 = fma2(f[ch][j], f[ch][j], s2);
    }
    if (kHold && k + 1 < rounds) fetch(t + stride, row + stride * p.d);
    float rf = 1.f;
    if (POST) {
      float s[1] = {sum8(s2)};
      group_sum(s, group, red[0]);
      rf = rsqrtf(fmaf(s[0], inv_d, p.eps));
      if (on && lane == 0 && p.rf) p.rf[t] = rf;
    }
    if (p.gate_mode == DSALT_GATE_TOKEN && on) rf *= to_f32<T>(Gt[t]);
    const f2 rf2 = dup(rf);
    s2 = dup(0.f);
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (lane + ch * group) * 8;
      if (!(on && c < p.d)) continue;
      const int64_t at = row + c;
      f2 (&wb)[4] = wbs[ch], (&wn)[4] = wns[ch];
      if (!kHold) column_factors<T>(p, dr, c, wb, wn);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[ch][j] = mul2(f[ch][j], wb[j]);
      if (p.gate_mode == DSALT_GATE_FULL) {
        Raw<T, VEC> raw;
        f2 g[4];
        raw.load(Gt + at, p.d - c);
        raw.get(g);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[ch][j] = mul2(f[ch][j], g[j]);
      }
      if constexpr (DROP && VEC) {
        float e[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) unpair(f[ch][j], e[2 * j], e[2 * j + 1]);
        dr.select_block((uint64_t)at >> 3, e);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[ch][j] = pair(e[2 * j], e[2 * j + 1]);
      } else if constexpr (DROP) {
        uint32_t m[8];
        dr.masks8((uint64_t)at, m);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[ch][j] = and2(f[ch][j], m[2 * j], m[2 * j + 1]);
      }
      Raw<T, VEC> out;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[ch][j] = fma2(f[ch][j], rf2, x[ch][j]);
      out.set(x[ch]);
      out.store(reinterpret_cast<T*>(p.x_new) + at, p.d - c);
#pragma unroll
      for (int j = 0; j < 4; ++j) s2 = fma2(x[ch][j], x[ch][j], s2);
    }
    if (p.norm) {
      float s[1] = {sum8(s2)};
      group_sum(s, group, red[1]);
      const float r = rsqrtf(fmaf(s[0], inv_d, p.eps));
      if (on && lane == 0 && p.r) p.r[t] = r;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const int c = (lane + ch * group) * 8;
        if (!(on && c < p.d)) continue;
        f2 (&wb)[4] = wbs[ch], (&wn)[4] = wns[ch];
      if (!kHold) column_factors<T>(p, dr, c, wb, wn);
        Raw<T, VEC> out;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[ch][j] = mul2(mul2(x[ch][j], dup(r)), wn[j]);
        out.set(x[ch]);
        out.store(reinterpret_cast<T*>(p.h) + row + c, p.d - c);
      }
    }
    if (!kHold && k + 1 < rounds) fetch(t + stride, row + stride * p.d);
    // with one sum a row the next row's would write what this row's may still read
    if (!(POST && p.norm) && group > 32) __syncthreads();
  }
}

template <typename T, int CH, bool VEC, int MAXT, bool DROP, bool POST>
__global__ void __launch_bounds__(MAXT, CH == 1 ? 512 / MAXT : 1) residual_bwd_kernel(const DsaltResidualNormParams p, int group) {
  constexpr bool kHold = CH <= 2;
  __shared__ float4 red[2][kMaxWarps];
  if (threadIdx.x < 2 * kMaxWarps) red[0][threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncthreads();
  const int gid = threadIdx.x / group, lane = threadIdx.x - gid * group, per_cta = blockDim.x / group;
  const int64_t stride = (int64_t)gridDim.x * per_cta, first = (int64_t)blockIdx.x * per_cta + gid;
  const int rounds = (int)((p.T - (int64_t)blockIdx.x * per_cta + stride - 1) / stride);
  Dropout dr;
  dr.init(p.seed, p.site, p.threshold);
  const T* Gt = reinterpret_cast<const T*>(p.gate);
  const bool with_h = p.norm && p.dh, full = p.gate_mode == DSALT_GATE_FULL;
  const bool sums = with_h || POST || p.gate_mode == DSALT_GATE_TOKEN;
  // without a norm, a scale or a gate on f nothing depends on its values
  const void* f_rows = POST || p.dscale || p.gate_mode != DSALT_GATE_NONE ? p.f : nullptr;
  const float inv_d = 1.f / (float)p.d;
  f2 wbs[CH][4], wns[CH][4], a_branch[CH][4], a_norm[CH][4];
  if (kHold)
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) column_factors<T>(p, dr, (lane + ch * group) * 8, wbs[ch], wns[ch]);
#pragma unroll
  for (int ch = 0; ch < CH; ++ch)
#pragma unroll
    for (int j = 0; j < 4; ++j) a_branch[ch][j] = a_norm[ch][j] = dup(0.f);
  Raw<T, VEC> nx[CH], nf[CH], nd[CH], nh[CH];  // x', f, dx_new, dh
  float nr = 0.f, nrf = 1.f, ngt = 1.f;
  auto fetch = [&](int64_t t, int64_t row) {
    const bool on = t < p.T;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (lane + ch * group) * 8;
      const bool in = on && c < p.d;
      const int64_t at = row + c;
      auto one = [&](Raw<T, VEC>& raw, const void* q) {
        if (in && q) raw.load(reinterpret_cast<const T*>(q) + at, p.d - c);
        else raw.zero();
      };
      one(nx[ch], with_h ? p.x_new : nullptr);
      one(nh[ch], with_h ? p.dh : nullptr);
      one(nf[ch], f_rows);
      one(nd[ch], p.dx_new);
    }
    nr = with_h && on ? __ldg(p.r + t) : 0.f;
    nrf = POST && on ? __ldg(p.rf + t) : 1.f;
    ngt = p.gate_mode == DSALT_GATE_TOKEN && on ? to_f32<T>(Gt[t]) : 1.f;
  };
  int64_t t = first;
  int64_t row = t * p.d;  // index of the row's first element
  fetch(t, row);
  for (int k = 0; k < rounds; ++k, t += stride, row += stride * p.d) {
    const bool on = t < p.T;
    const float r = nr, rf = nrf, gt = ngt;
    const f2 r2 = dup(r), rf2 = dup(rf);
    f2 u[CH][4], x[CH][4], f[CH][4];  // x̂, f̂
    uint32_t m[CH][8];
    f2 s0 = dup(0.f), s1 = dup(0.f), s2 = dup(0.f);
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (lane + ch * group) * 8;
      const int64_t at = row + c;
      f2 dh[4], g[4] = {dup(1.f), dup(1.f), dup(1.f), dup(1.f)};
      nx[ch].get(x[ch]);
      nf[ch].get(f[ch]);
      nd[ch].get(u[ch]);
      nh[ch].get(dh);
      f2 (&wb)[4] = wbs[ch], (&wn)[4] = wns[ch];
      if (!kHold) column_factors<T>(p, dr, c, wb, wn);
      row_masks<VEC, DROP>(dr, at, m[ch]);
      if (full && on && c < p.d) {
        Raw<T, VEC> raw;
        raw.load(Gt + at, p.d - c);
        raw.get(g);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[ch][j] = mul2(x[ch][j], r2);
        const f2 hx = mul2(dh[j], x[ch][j]);
        a_norm[ch][j] = add2(hx, a_norm[ch][j]);
        s0 = fma2(hx, wn[j], s0);
        u[ch][j] = fma2(mul2(dh[j], wn[j]), r2, u[ch][j]);
        if (POST) f[ch][j] = mul2(f[ch][j], rf2);
        // κ: a dropped element passes nothing back, whatever f holds there
        f2 kf = and2(f[ch][j], m[ch][2 * j], m[ch][2 * j + 1]);
        if (!POST) f[ch][j] = kf;
        kf = mul2(kf, wb[j]);
        if (full) kf = mul2(kf, g[j]);
        s1 = fma2(kf, u[ch][j], s1);
        s2 = fma2(kf, x[ch][j], s2);
      }
    }
    if (kHold && k + 1 < rounds) fetch(t + stride, row + stride * p.d);
    float s[3] = {sum8(s0), sum8(s1), sum8(s2)};
    if (sums) group_sum(s, group, red[k & 1]);
    const float e = r * (s[0] * inv_d);
    const float S = fmaf(-e, s[2], s[1]);  // Σ κ⊙G, without a token's gate
    if (p.gate_mode == DSALT_GATE_TOKEN && on && lane == 0) reinterpret_cast<T*>(p.dgate)[t] = from_f32<T>(S);
    const f2 ne = dup(-e), gt2 = dup(gt), al = dup(rf * gt), nm = dup(-(rf * gt) * (S * inv_d));
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (lane + ch * group) * 8;
      if (!(on && c < p.d)) continue;
      const int64_t at = row + c;
      f2 (&wb)[4] = wbs[ch], (&wn)[4] = wns[ch];
      if (!kHold) column_factors<T>(p, dr, c, wb, wn);
      Raw<T, VEC> out;
#pragma unroll
      for (int j = 0; j < 4; ++j) u[ch][j] = fma2(ne, x[ch][j], u[ch][j]);  // G
      out.set(u[ch]);
      out.store(reinterpret_cast<T*>(p.dx) + at, p.d - c);
      f2 df[4];
      if (full) {
        f2 g[4], dg[4];
        out.load(Gt + at, p.d - c);
        out.get(g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f2 G = and2(u[ch][j], m[ch][2 * j], m[ch][2 * j + 1]);
          const f2 Gw = mul2(G, wb[j]);
          dg[j] = mul2(Gw, f[ch][j]);
          df[j] = mul2(mul2(Gw, g[j]), al);
          a_branch[ch][j] = fma2(mul2(G, g[j]), f[ch][j], a_branch[ch][j]);
        }
        out.set(dg);
        out.store(reinterpret_cast<T*>(p.dgate) + at, p.d - c);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f2 G = and2(u[ch][j], m[ch][2 * j], m[ch][2 * j + 1]);
          df[j] = mul2(mul2(G, wb[j]), al);
          a_branch[ch][j] = fma2(mul2(G, f[ch][j]), gt2, a_branch[ch][j]);
        }
      }
      if (POST) {
#pragma unroll
        for (int j = 0; j < 4; ++j) df[j] = fma2(f[ch][j], nm, df[j]);
      }
      out.set(df);
      out.store(reinterpret_cast<T*>(p.df) + at, p.d - c);
    }
    if (!kHold && k + 1 < rounds) fetch(t + stride, row + stride * p.d);
  }
  // this CTA's sums: partial row blockIdx.x of [CTAs][2][d] (Σ G⊙gate⊙f̂ where kept,
  // Σ dh⊙x̂); several groups' sums are added in order first
  float* part = p.parts + (int64_t)blockIdx.x * 2 * p.d;
  if (per_cta > 1) {
    __shared__ float group_sums[CH == 1 && MAXT == 256 ? 2 * kSmallThreads * 8 : 1];
    if constexpr (CH == 1 && MAXT == 256) {
      float* mine = group_sums + gid * 2 * group * 8 + lane * 8;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unpair(a_branch[0][j], mine[2 * j], mine[2 * j + 1]);
        unpair(a_norm[0][j], mine[group * 8 + 2 * j], mine[group * 8 + 2 * j + 1]);
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * p.d; i += blockDim.x) {
        const int at = i < p.d ? i : group * 8 + i - p.d;
        float v = 0.f;
        for (int g = 0; g < per_cta; ++g) v += group_sums[g * 2 * group * 8 + at];
        part[i] = v;
      }
    }
    return;
  }
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
    const int c = (lane + ch * group) * 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b, n0, n1;
      unpair(a_branch[ch][j], a, b);
      unpair(a_norm[ch][j], n0, n1);
      if (c + 2 * j < p.d) part[c + 2 * j] = a, part[p.d + c + 2 * j] = n0;
      if (c + 2 * j + 1 < p.d) part[c + 2 * j + 1] = b, part[p.d + c + 2 * j + 1] = n1;
    }
  }
}

// Column sums of the partial rows in a fixed order: a CTA owns 32 columns of one of
// the two sums; warp w adds rows w, w + 32, …, then the warps' sums in order.  The first
// sum, times 1 / share kept, gives dscale with post's weights and dpost with scale's.
template <typename T>
__global__ void __launch_bounds__(1024) residual_colsum_kernel(const DsaltResidualNormParams p, int64_t nparts) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float acc = 0.f;
  if (c < p.d)
#pragma unroll 8
    for (int64_t i = grp; i < nparts; i += 32) acc += __ldg(p.parts + (i * 2 + blockIdx.y) * p.d + c);
  s[grp][lane] = acc;
  __syncthreads();
  if (grp != 0 || c >= p.d) return;
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < 32; ++w) v += s[w][lane];
  auto weight = [&](const void* w) {
    return !w ? 1.f : p.w_f32 ? __ldg(reinterpret_cast<const float*>(w) + c) : to_f32<T>(reinterpret_cast<const T*>(w)[c]);
  };
  auto put = [&](void* out, float x) {
    if (!out) return;
    if (p.w_f32) reinterpret_cast<float*>(out)[c] = x;
    else reinterpret_cast<T*>(out)[c] = from_f32<T>(x);
  };
  if (blockIdx.y == 1) {
    put(p.dnorm, v);
    return;
  }
  v *= p.threshold >= 65536 ? 0.f : 65536.f / (float)(65536 - p.threshold);
  put(p.dscale, v * weight(p.post));
  put(p.dpost, v * weight(p.scale));
}

// CTAs that run at once: 16 warps an SM for the backward's registers, 32 for the
// forward's, half as many with more than one chunk; no more than there are rows for
int64_t ctas_of(int64_t T, const Shape& s, bool bwd, int sms) {
  const int per_cta = s.cta / s.group, threads_per_sm = (bwd ? 512 : 1024) / (s.chunks > 1 ? 2 : 1);
  const int64_t want = (T + per_cta - 1) / per_cta, most = (int64_t)sms * (threads_per_sm < s.cta ? 1 : threads_per_sm / s.cta);
  return want < most ? want : most;
}

template <typename T, int CH, bool VEC, int MAXT>
cudaError_t launch_v(const DsaltResidualNormParams& p, const Shape& s, bool bwd, cudaStream_t st) {
  int sms = 0;
  cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  const unsigned ctas = (unsigned)ctas_of(p.T, s, bwd, sms);
  auto run = [&](auto drop, auto post) {
    if (bwd) residual_bwd_kernel<T, CH, VEC, MAXT, drop.value, post.value><<<ctas, s.cta, 0, st>>>(p, s.group);
    else residual_fwd_kernel<T, CH, VEC, MAXT, drop.value, post.value><<<ctas, s.cta, 0, st>>>(p, s.group);
  };
  using Yes = std::true_type;
  using No = std::false_type;
  if (p.threshold > 0) p.post ? run(Yes(), Yes()) : run(Yes(), No());
  else p.post ? run(No(), Yes()) : run(No(), No());
  if (!bwd) return cudaGetLastError();
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if (p.dscale || p.dpost || p.dnorm) {
    residual_colsum_kernel<T><<<dim3((p.d + 31) / 32, p.dnorm ? 2 : 1), 1024, 0, st>>>(p, ctas);
    e = cudaGetLastError();
  }
  return e;
}
template <typename T, bool VEC>
cudaError_t launch_s(const DsaltResidualNormParams& p, const Shape& s, bool bwd, cudaStream_t st) {
  if (s.chunks == 4) return launch_v<T, 4, VEC, 512>(p, s, bwd, st);
  if (s.chunks == 2) return s.cta > 256 ? launch_v<T, 2, VEC, 512>(p, s, bwd, st) : launch_v<T, 2, VEC, 256>(p, s, bwd, st);
  return s.cta > 256 ? launch_v<T, 1, VEC, 512>(p, s, bwd, st) : launch_v<T, 1, VEC, 256>(p, s, bwd, st);
}

template <typename T>
cudaError_t launch_t(const DsaltResidualNormParams& p, bool bwd, cudaStream_t st) {
  bool vec = p.d % 8 == 0;
  for (const void* q : {p.x, p.f, (const void*)p.x_new, (const void*)p.h, p.dx_new, p.dh, (const void*)p.dx,
                        (const void*)p.df, p.gate_mode == DSALT_GATE_FULL ? p.gate : nullptr,
                        p.gate_mode == DSALT_GATE_FULL ? (const void*)p.dgate : nullptr})
    vec = vec && ((uintptr_t)q & 15) == 0;
  const Shape s = shape_of(p.d, vec);
  return vec ? launch_s<T, true>(p, s, bwd, st) : launch_s<T, false>(p, s, bwd, st);
}

}  // namespace

cudaError_t residual_norm_parts(int64_t T, int d, int* out) {
  int sms = 0;
  const cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  *out = 0;
  for (const bool vec : {false, true}) {
    const Shape s = shape_of(d, vec);
    *out = std::max(*out, (int)ctas_of(T, s, true, sms));
  }
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

// Forward of the gated feed-forward block for up to 16 tokens (serving: one token a
// sequence): g = x·Wgᵀ, u = x·Wuᵀ, h = act(g)⊙u, then y = h·Wdᵀ, as two launches.
// Bound: the weights' bytes (3·d·F), and at these sizes the latency of getting them.
//
// A CTA owns 16 weight rows (features, or output columns) and splits K over its eight
// warps, and over the CTAs of a cluster where there are too few rows to fill the
// device; the partial sums are added in the order of K through shared memory, so
// results do not change from run to run.  The products are mma.sync m16n8k16 with the
// weight rows as M and 8 or 16 tokens as N: a tile of the 5th-generation pipe would
// have 128 weight rows, a fifth of the SMs would get one, and it would wait for the
// bytes all the same.  Weights go from global memory straight to the fragments: a lane
// reads 16 contiguous bytes of a row (8 consecutive k), and since a sum over k does not
// care for its order, those 8 serve as the fragment's k of two MMA steps, in A and B
// alike.  The second product takes h as two 16-bit words, the rounded value and the
// rounding's rest, at no cost beside the weights' bytes: y is off by its own rounding
// only.  The second launch starts early (programmatic dependent launch): it fetches
// its first weights before it waits for h.
#include <algorithm>

#include "device.cuh"
#include "ffn.cuh"
#include "ffn_act.cuh"

namespace dsalt {
namespace ffn {
namespace {

constexpr int kWarps = 8, kRows = 16, kBlockK = 32;

struct FewArgs {
  const uint16_t* w[2];  // [M, K] stride ld_w: gate and up, or down
  int64_t ld_w[2];
  const uint16_t* in;    // [T, K] stride ld_in
  uint16_t* h_lo;        // what h's rounding leaves, rounded: written beside h, read with it
  int64_t ld_in;
  uint16_t* out;         // [T, M] stride ld_out: h, or y
  uint16_t *a, *b, *ab;  // with `out`'s stride, or null
  int64_t ld_out;
  int64_t T;
  int M, K, split;       // split: CTAs of the cluster along K
  bool bf16;
};

// 8 consecutive elements, or zeros.  RO: through the read-only path, for what no launch
// still running writes.
template <bool RO>
__device__ __forceinline__ uint4 load_k8(const uint16_t* p, bool on) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (on) v = RO ? __ldg(reinterpret_cast<const uint4*>(p)) : __ldcg(reinterpret_cast<const uint4*>(p));
  return v;
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: groups of 8 tokens of a CTA.  NM: weight matrices, 2 (gate and up) or 1 (down).
template <int NT, int NM, bool BF16, int ACT>
__global__ void __launch_bounds__(kWarps * 32, 2) ffn_few_kernel(const FewArgs p) {
  constexpr int kAhead = 4;  // K blocks whose weights a warp requests at once
  constexpr int kTok = NT * 8, kSums = NM * kRows * kTok;
  extern __shared__ float red[];  // [kWarps][NM][kRows][kTok], then the CTA's sums in the first
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const uint32_t rank = p.split > 1 ? sm100::cluster_rank() : 0;
  const int row0 = (int)(blockIdx.x / p.split) * kRows;
  const int64_t t0 = (int64_t)blockIdx.y * kTok;
  const int nkb = (p.K + kBlockK - 1) / kBlockK, parts = kWarps * p.split, part = (int)rank * kWarps + warp;
  const int kb_end = (int)((int64_t)nkb * (part + 1) / parts);
  int kb = (int)((int64_t)nkb * part / parts);

  float c[NM][NT][4];
#pragma unroll
  for (int m = 0; m < NM; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[m][n][i] = 0.f;

  uint4 wr[kAhead][NM][2];
  auto load_weights = [&](int from) {
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
      for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = row0 + g + 8 * i, k = (from + s) * kBlockK + 8 * q;
          wr[s][m][i] = load_k8<true>(p.w[m] + row * p.ld_w[m] + k, row < p.M && from + s < kb_end && k < p.K);
        }
  };
  load_weights(kb);
  if constexpr (NM == 2) asm volatile("griddepcontrol.launch_dependents;");
  else asm volatile("griddepcontrol.wait;" ::: "memory");  // h is complete
  while (kb < kb_end) {
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      // h comes from the launch before, which was still running when this one began
      auto products = [&](const uint16_t* in) {
        uint4 x[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int64_t t = t0 + n * 8 + g;
          const int k = (kb + s) * kBlockK + 8 * q;
          x[n] = load_k8<NM == 2>(in + t * p.ld_in + k, t < p.T && kb + s < kb_end && k < p.K);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int m = 0; m < NM; ++m) {
            const uint4 lo = wr[s][m][0], hi = wr[s][m][1];
            mma16816<BF16>(c[m][n], lo.x, hi.x, lo.y, hi.y, x[n].x, x[n].y);
            mma16816<BF16>(c[m][n], lo.z, hi.z, lo.w, hi.w, x[n].z, x[n].w);
          }
      };
      products(p.in);
      if constexpr (NM == 1) products(p.h_lo);
    }
    kb += kAhead;
    if (kb < kb_end) load_weights(kb);
  }

  // c[m][n]: rows g (0, 1) and g + 8 (2, 3), tokens 8·n + 2·q and the next
  float* mine = red + warp * kSums;
#pragma unroll
  for (int m = 0; m < NM; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<float2*>(mine + (m * kRows + g + 8 * i) * kTok + n * 8 + 2 * q) =
            make_float2(c[m][n][2 * i], c[m][n][2 * i + 1]);
  __syncthreads();
  for (int i = threadIdx.x; i < kSums; i += kWarps * 32) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += red[w * kSums + i];
    red[i] = s;  // read and written by this thread alone
  }
  if (p.split > 1) sm100::cluster_sync();
  else __syncthreads();

  // the cluster's sums: each CTA finishes its share of the 16 × kTok results
  const int share = (kRows * kTok + p.split - 1) / p.split;
  const int last = min((int)(rank + 1) * share, kRows * kTok);
  for (int i = (int)rank * share + threadIdx.x; i < last; i += kWarps * 32) {
    const int r = i % kRows, tok = i / kRows, row = row0 + r;
    const int64_t t = t0 + tok;
    if (row >= p.M || t >= p.T) continue;
    float v[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      const int at = (m * kRows + r) * kTok + tok;
      v[m] = 0.f;
      if (p.split == 1) {
        v[m] = red[at];
      } else {
        const uint32_t addr = sm100::smem_u32(red + at);
        for (int k = 0; k < p.split; ++k) {
          float x;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(sm100::map_rank(addr, k)) : "memory");
          v[m] += x;
        }
      }
    }
    const int64_t at = t * p.ld_out + row;
    float result = v[0];
    if constexpr (NM == 2) {
      float a, da;
      act_pair<ACT>(v[0], a, da);
      result = a * v[1];
      if (p.a) {
        const float b = da * v[1];
        p.a[at] = (uint16_t)(__float_as_uint(a) >> 16);
        p.b[at] = (uint16_t)(__float_as_uint(b) >> 16);
        p.ab[at] = (uint16_t)(next8(a, b, a, b));
      }
    }
    const uint32_t word = sm100::pack2(result, result, BF16);
    p.out[at] = (uint16_t)(word & 0xffffu);
    if constexpr (NM == 2) {
      const float rest =
          rounding_rest(result, BF16 ? __uint_as_float(word << 16) : __half2float(__ushort_as_half((uint16_t)word)));
      p.h_lo[at] = (uint16_t)(sm100::pack2(rest, rest, BF16) & 0xffffu);
    }
  }
  if (p.split > 1) sm100::cluster_sync();  // no CTA leaves while its sums are read
}

template <int NT, int NM, bool BF16, int ACT>
cudaError_t launch_kernel(FewArgs a, cudaStream_t st) {
  auto kernel = ffn_few_kernel<NT, NM, BF16, ACT>;
  const size_t smem = (size_t)kWarps * NM * kRows * NT * 8 * sizeof(float);
  cudaError_t e = ensure_smem((const void*)kernel, smem);
  if (e != cudaSuccess) return e;
  int sms = 0;
  if ((e = sm_count(&sms)) != cudaSuccess) return e;
  const int64_t tiles = (a.M + kRows - 1) / kRows, chunks = (a.T + NT * 8 - 1) / (NT * 8);
  // clusters along K while two CTAs an SM stay enough and every warp keeps a K block
  a.split = 1;
  while (a.split < 8 && tiles * chunks * a.split * 2 <= 2 * sms && (a.K + kBlockK - 1) / kBlockK >= 2 * kWarps * a.split)
    a.split *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * a.split), (unsigned)chunks);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)a.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = NM == 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int NT, int NM, int ACT>
cudaError_t launch_type(const FewArgs& a, cudaStream_t st) {
  return a.bf16 ? launch_kernel<NT, NM, true, ACT>(a, st) : launch_kernel<NT, NM, false, ACT>(a, st);
}
template <int NM, int ACT>
cudaError_t launch_tokens(const FewArgs& a, cudaStream_t st) {
  return a.T <= 8 ? launch_type<1, NM, ACT>(a, st) : launch_type<2, NM, ACT>(a, st);
}

}  // namespace
}  // namespace ffn

cudaError_t launch_ffn_few(const DsaltGatedFfnParams& p, cudaStream_t st) {
  using namespace ffn;
  FewArgs a = {};
  a.w[0] = (const uint16_t*)p.w_gate;
  a.w[1] = (const uint16_t*)p.w_up;
  a.ld_w[0] = p.ld_wg;
  a.ld_w[1] = p.ld_wu;
  a.in = (const uint16_t*)p.x;
  a.ld_in = p.ld_x;
  a.out = (uint16_t*)p.h;
  a.h_lo = (uint16_t*)p.h_lo;
  a.a = (uint16_t*)p.a;
  a.b = (uint16_t*)p.b;
  a.ab = (uint16_t*)p.ab;
  a.ld_out = p.ld_f;
  a.T = p.T;
  a.M = p.F;
  a.K = p.d;
  a.bf16 = p.dtype == DSALT_BF16;
  cudaError_t e = p.activation == DSALT_ACT_SILU   ? launch_tokens<2, DSALT_ACT_SILU>(a, st)
                  : p.activation == DSALT_ACT_GELU ? launch_tokens<2, DSALT_ACT_GELU>(a, st)
                                                   : launch_tokens<2, DSALT_ACT_GELU_TANH>(a, st);
  if (e != cudaSuccess) return e;
  a.w[0] = (const uint16_t*)p.w_down;
  a.ld_w[0] = p.ld_wd;
  a.in = (const uint16_t*)p.h;
  a.ld_in = p.ld_f;
  a.out = (uint16_t*)p.y;
  a.a = a.b = a.ab = nullptr;
  a.ld_out = p.d_out;
  a.M = p.d_out;
  a.K = p.F;
  return launch_tokens<1, 0>(a, st);
}

}  // namespace dsalt

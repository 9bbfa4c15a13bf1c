// Forward of the gated feed-forward block for a batch of tokens that is still short of
// a tile of ffn_tc.cu (17 to 384: a step of many sequences, a short prompt), as two
// launches.  Bound: the weights' bytes and the latency of the way to them; with tiles of
// 256 tokens × 128 features a handful of SM pairs would fetch all weights.
//
// The roles are swapped: weight rows are M (128 TMEM lanes: 64 rows of gate and the same
// 64 of up, or rows of down), tokens are N, and K is split over the CTAs of a cluster,
// so that the weights stream into every SM.  Each CTA multiplies its share of K
// (TMA ring, tcgen05.mma, one accumulator in TMEM), writes the fp32 partial sums to its
// shared memory, and after a cluster barrier finishes a share of the tokens: the
// partials are added in the order of K (the same bits every run), then the activation
// and the product.  Up to 64 tokens the second product takes h as two 16-bit words (two
// MMAs a step), as in ffn_few.cu.  The second launch is a programmatic dependent: it
// requests its first weights before it waits for h.  Every wait is bounded.
//   warp 0  TMA loads      warp 1  TMEM owner, MMA issuer      all 8: sums and results
#include <algorithm>
#include <cstring>

#include "device.cuh"
#include "ffn.cuh"
#include "ffn_act.cuh"

namespace dsalt {
namespace ffn {
namespace {

constexpr int kThreads = 256, BK = 64, kHalf = 64 * BK * 2;  // 64 weight rows of a K block
constexpr int kMaxSplit = 8;

// NT: tokens (N).  NB: B operands of a K block, 2 with h's low words.
template <int NT, int NB>
struct Cfg {
  static constexpr int kStageBytes = 2 * kHalf + NB * NT * BK * 2;
  static constexpr int kStages = NT * NB > 64 ? 3 : 4;  // two CTAs an SM: 112 KB at most
  static constexpr int FULL = 0, EMPTY = kStages, ACC = 2 * kStages, NB_BARS = ACC + 1;
  static constexpr int kRing = kStages * kStageBytes, kSums = 128 * NT * 4;
  struct alignas(1024) Smem {
    uint8_t ring[kRing > kSums ? kRing : kSums];  // after the products: partial sums [token][128 rows]
    uint64_t bars[NB_BARS];
    uint32_t tmem_base;
    int abort_flag;
  };
};

struct alignas(64) MidArgs {
  CUtensorMap mw[2];  // gate and up, or down twice: 64-row boxes
  CUtensorMap mx[2];  // x, or h and its low words: NT-row boxes
  uint16_t *out, *out_lo, *a, *b, *ab;  // h (a, b, ab or null), or y
  int64_t ld_out;
  int T, M, K, split;   // tokens: NT of them from blockIdx.y · NT on
  int rows;           // weight rows of a tile: 64 (hidden: of each of gate and up), or 128
  bool bf16, vec;     // vec: 8-byte stores of four results fit
  int32_t* status;
};

__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr)
               : "memory");
  return v;
}

template <int NT, int NB, bool HIDDEN, int ACT>
__global__ void __launch_bounds__(kThreads) ffn_mid_kernel(const __grid_constant__ MidArgs p) {
  using namespace sm100;
  using C = Cfg<NT, NB>;
  extern __shared__ uint8_t smem_raw[];
  auto& sm = *reinterpret_cast<typename C::Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = p.split > 1 ? cluster_rank() : 0;
  const int row0 = (int)(blockIdx.x / p.split) * p.rows;
  const int nkb = (p.K + BK - 1) / BK;
  const int kb0 = nkb * (int)rank / p.split, kb1 = nkb * ((int)rank + 1) / p.split;
  const BarArray bar{smem_u32(&sm.bars[0])};
  if (HIDDEN) asm volatile("griddepcontrol.launch_dependents;");
  if (tid == 0) {
    prefetch_tmap(&p.mw[0]);
    if (HIDDEN) prefetch_tmap(&p.mw[1]);
    for (int i = 0; i < NB; ++i) prefetch_tmap(&p.mx[i]);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar[C::FULL + s], 1);
      mbar_init(bar[C::EMPTY + s], 1);
    }
    mbar_init(bar[C::ACC], 1);
    fence_mbar_init();
    sm.abort_flag = 0;
  }
  if (warp == 1) tmem_alloc(smem_u32(&sm.tmem_base), NT);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  volatile int* abort_flag = &sm.abort_flag;

  if (warp == 0 && lane == 0) {
    // ------------------------------------------------------------ loads
    auto stage = [&](int g) { return smem_u32(sm.ring) + (uint32_t)(g % C::kStages) * C::kStageBytes; };
    auto load_w = [&](int g) {
      const uint32_t full = bar[C::FULL + g % C::kStages];
      const bool both = HIDDEN || p.rows == 128;  // else lanes 64 to 127 multiply what lies there, unread
      mbar_expect_tx(full, C::kStageBytes - (both ? 0 : kHalf));
      tma_load_3d(stage(g), &p.mw[0], full, (kb0 + g) * BK, row0, 0);
      if (both) tma_load_3d(stage(g) + kHalf, &p.mw[1], full, (kb0 + g) * BK, HIDDEN ? row0 : row0 + 64, 0);
    };
    auto load_x = [&](int g) {
      const uint32_t full = bar[C::FULL + g % C::kStages];
#pragma unroll
      for (int i = 0; i < NB; ++i)
        tma_load_3d(stage(g) + 2 * kHalf + i * NT * BK * 2, &p.mx[i], full, (kb0 + g) * BK, (int)blockIdx.y * NT, 0);
    };
    const int n = kb1 - kb0, ahead = min(n, C::kStages);
    for (int g = 0; g < ahead; ++g) load_w(g);
    if (!HIDDEN) asm volatile("griddepcontrol.wait;" ::: "memory");  // h is complete
    for (int g = 0; g < ahead; ++g) load_x(g);
    int g = ahead;
    for (; g < n; ++g) {
      if (!mbar_wait(bar[C::EMPTY + g % C::kStages], (g / C::kStages - 1) & 1, abort_flag, p.status)) break;
      load_w(g);
      load_x(g);
    }
    // never leave a copy in flight into shared memory
    for (int gg = max(0, g - C::kStages); gg < g; ++gg) mbar_drain(bar[C::FULL + gg % C::kStages], (gg / C::kStages) & 1);
  } else if (warp == 1 && lane == 0) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t idesc = idesc_f16(p.bf16, 128, NT, false, false);
    for (int g = 0; g < kb1 - kb0; ++g) {
      const int st = g % C::kStages;
      if (!mbar_wait(bar[C::FULL + st], (g / C::kStages) & 1, abort_flag, p.status)) break;
      tc_fence_after();
      const uint32_t a = smem_u32(sm.ring) + st * C::kStageBytes;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk)
          mma_f16(tmem, sdesc_sw128(a + kk * 32, 16, 1024), sdesc_sw128(a + 2 * kHalf + i * NT * BK * 2 + kk * 32, 16, 1024),
                  idesc, (g > 0 || i > 0 || kk > 0) ? 1u : 0u);
      mma_commit(bar[C::EMPTY + st]);
    }
    mma_commit(bar[C::ACC]);
  }
  __syncwarp();
  // -------------------------------------------------------- partial sums
  // (also after a wait that gave up: the cluster's barriers are met by all its CTAs)
  const bool ok = mbar_wait(bar[C::ACC], 0, abort_flag, p.status);
  __syncwarp();  // the lanes' waits may end apart; the TMEM loads want them together
  tc_fence_after();
  __syncthreads();  // every product and copy of this CTA is done: the ring becomes the sums
  float* sums = reinterpret_cast<float*>(sm.ring);
  const int q4 = warp & 3;
#pragma unroll
  for (int c = (warp >> 2) * 16; c < NT; c += 32) {
    float v[16];
    tmem_ld16(tmem + ((uint32_t)(32 * q4) << 16) + c, v);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) sums[(c + j) * 128 + 32 * q4 + lane] = ok ? v[j] : 0.f;
  }
  tc_fence_before();
  if (p.split > 1) cluster_sync();
  else __syncthreads();

  // ------------------------------------------------------------- results
  // four rows a thread, this CTA's share of the tokens
  const int t0 = (int)blockIdx.y * NT, share = (NT + p.split - 1) / p.split;
  const int t_end = min(min((int)(rank + 1) * share, NT), p.T - t0);
  const int quads = p.rows / 4;
  const uint32_t base = smem_u32(sums);
  uint32_t peer[kMaxSplit];
#pragma unroll
  for (int s = 0; s < kMaxSplit; ++s) peer[s] = p.split > 1 ? map_rank(base, min(s, p.split - 1)) : base;
  for (int i = tid; i < (t_end - (int)rank * share) * quads; i += kThreads) {
    const int t = (int)rank * share + i / quads, r = i % quads * 4, row = row0 + r;
    if (row >= p.M) continue;
    // every load on its way before the first sum; added in the order of K
    float4 xg[kMaxSplit], xu[kMaxSplit];
#pragma unroll
    for (int s = 0; s < kMaxSplit; ++s)
      if (s < p.split) {
        xg[s] = cluster_load4(peer[s] + (uint32_t)(t * 128 + r) * 4);
        if (HIDDEN) xu[s] = cluster_load4(peer[s] + (uint32_t)(t * 128 + 64 + r) * 4);
      }
    float4 g4 = xg[0], u4 = xu[0];
#pragma unroll
    for (int s = 1; s < kMaxSplit; ++s)
      if (s < p.split) {
        g4.x += xg[s].x; g4.y += xg[s].y; g4.z += xg[s].z; g4.w += xg[s].w;
        if (HIDDEN) u4.x += xu[s].x, u4.y += xu[s].y, u4.z += xu[s].z, u4.w += xu[s].w;
      }
    float v[4] = {g4.x, g4.y, g4.z, g4.w};
    const int64_t at = (int64_t)(t0 + t) * p.ld_out + row;
    auto put = [&](uint16_t* dst, uint32_t lo, uint32_t hi) {
      if (p.vec) {  // rows in fours: M is a multiple of 4 there
        *reinterpret_cast<uint2*>(dst + at) = make_uint2(lo, hi);
      } else {
        const uint32_t w[2] = {lo, hi};
        for (int k = 0; k < 4 && row + k < p.M; ++k) dst[at + k] = (uint16_t)(w[k / 2] >> (16 * (k & 1)));
      }
    };
    if constexpr (HIDDEN) {
      const float u[4] = {u4.x, u4.y, u4.z, u4.w};
      float a[4], b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        act_pair<ACT>(v[k], a[k], b[k]);
        v[k] = a[k] * u[k];
        b[k] *= u[k];
      }
      if (p.a) {
        put(p.a, upper16(a[0], a[1]), upper16(a[2], a[3]));
        put(p.b, upper16(b[0], b[1]), upper16(b[2], b[3]));
        put(p.ab, next8(a[0], b[0], a[1], b[1]), next8(a[2], b[2], a[3], b[3]));
      }
    }
    const uint32_t w0 = pack2(v[0], v[1], p.bf16), w1 = pack2(v[2], v[3], p.bf16);
    put(p.out, w0, w1);
    if (HIDDEN && p.out_lo) {
      const float2 f0 = unpack2(w0, p.bf16), f1 = unpack2(w1, p.bf16);
      put(p.out_lo, pack2(rounding_rest(v[0], f0.x), rounding_rest(v[1], f0.y), p.bf16),
          pack2(rounding_rest(v[2], f1.x), rounding_rest(v[3], f1.y), p.bf16));
    }
  }
  __syncwarp();  // the loop above ends lane by lane; the barriers and the release of TMEM want whole warps
  if (p.split > 1) cluster_sync();  // no CTA leaves while its sums are read
  else __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, NT);
}

bool encode(CUtensorMap* m, int dtype, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  return encode_tensor_map_3d(m, dtype == DSALT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base,
                              (uint64_t)cols, (uint64_t)rows, 1, (uint64_t)ld * 2, (uint64_t)ld * 2, BK, box_rows,
                              1) == CUDA_SUCCESS;
}

template <int NT, int NB, bool HIDDEN, int ACT>
cudaError_t launch_kernel(const MidArgs& a, int64_t tiles, cudaStream_t st) {
  auto kernel = ffn_mid_kernel<NT, NB, HIDDEN, ACT>;
  const size_t smem = sizeof(typename Cfg<NT, NB>::Smem) + 1024;
  cudaError_t e = ensure_smem((const void*)kernel, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * a.split), (unsigned)((a.T + NT - 1) / NT));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)a.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = HIDDEN ? 1 : 2;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

// CTAs of a cluster along K: what runs at once at two CTAs an SM (a GPC's odd SMs leave
// out a tenth at clusters of 8), and two K blocks a CTA at least.
int split_of(int64_t ctas, int K, int sms) {
  int s = 1;
  while (s < kMaxSplit && ctas * s * 2 <= (s < 4 ? 2 * sms - 12 : 2 * sms - 32) && (K + BK - 1) / BK >= 4 * s) s *= 2;
  return s;
}

template <int NT, int NB>
cudaError_t launch_both(const DsaltGatedFfnParams& p, int sms, cudaStream_t st) {
  MidArgs a;
  memset(&a, 0, sizeof(a));
  a.T = (int)p.T;
  a.bf16 = p.dtype == DSALT_BF16;
  a.status = p.status;
  // h
  a.M = p.F;
  a.K = p.d;
  a.rows = 64;
  a.out = (uint16_t*)p.h;
  a.out_lo = NB == 2 ? (uint16_t*)p.h_lo : nullptr;
  a.a = (uint16_t*)p.a;
  a.b = (uint16_t*)p.b;
  a.ab = (uint16_t*)p.ab;
  a.ld_out = p.ld_f;
  a.vec = p.F % 4 == 0;
  if (!encode(&a.mw[0], p.dtype, p.w_gate, p.F, p.d, p.ld_wg, 64) || !encode(&a.mw[1], p.dtype, p.w_up, p.F, p.d, p.ld_wu, 64) ||
      !encode(&a.mx[0], p.dtype, p.x, p.T, p.d, p.ld_x, NT))
    return cudaErrorInvalidValue;
  const int64_t chunks = (p.T + NT - 1) / NT;
  int64_t tiles = (p.F + 63) / 64;
  a.split = split_of(tiles * chunks, a.K, sms);
  cudaError_t e = p.activation == DSALT_ACT_SILU   ? launch_kernel<NT, 1, true, DSALT_ACT_SILU>(a, tiles, st)
                  : p.activation == DSALT_ACT_GELU ? launch_kernel<NT, 1, true, DSALT_ACT_GELU>(a, tiles, st)
                                                   : launch_kernel<NT, 1, true, DSALT_ACT_GELU_TANH>(a, tiles, st);
  if (e != cudaSuccess) return e;
  // y: tiles of 64 rows (half the lanes idle) where tiles of 128 would leave SMs without one
  a.M = p.d_out;
  a.K = p.F;
  a.rows = (p.d_out + 127) / 128 * chunks * kMaxSplit >= sms ? 128 : 64;
  a.out = (uint16_t*)p.y;
  a.out_lo = a.a = a.b = a.ab = nullptr;
  a.ld_out = p.d_out;
  a.vec = p.d_out % 4 == 0 && ((uintptr_t)p.y & 7) == 0;
  if (!encode(&a.mw[0], p.dtype, p.w_down, p.d_out, p.F, p.ld_wd, 64) || !encode(&a.mx[0], p.dtype, p.h, p.T, p.F, p.ld_f, NT) ||
      (NB == 2 && !encode(&a.mx[1], p.dtype, p.h_lo, p.T, p.F, p.ld_f, NT)))
    return cudaErrorInvalidValue;
  a.mw[1] = a.mw[0];
  tiles = (p.d_out + a.rows - 1) / a.rows;
  a.split = split_of(tiles * chunks, a.K, sms);
  return launch_kernel<NT, NB, false, 0>(a, tiles, st);
}

}  // namespace
}  // namespace ffn

cudaError_t launch_ffn_mid(const DsaltGatedFfnParams& p, cudaStream_t st) {
  using namespace ffn;
  // the tensor maps need the device's context current on this thread (see launch_ffn_tc)
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaSetDevice(dev);
  if (e == cudaSuccess) e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  if (p.T <= 32) return launch_both<32, 2>(p, sms, st);
  if (p.T <= 64) return launch_both<64, 2>(p, sms, st);
  return launch_both<128, 1>(p, sms, st);
}

}  // namespace dsalt

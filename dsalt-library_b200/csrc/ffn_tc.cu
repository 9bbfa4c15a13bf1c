// Gated feed-forward block on the tensor cores (sm_100a):
//   g = x·Wgᵀ,  u = x·Wuᵀ,  h = act(g)⊙u,  y = h·Wdᵀ
// and its gradients
//   dh = dy·Wd,  dg = dh⊙u⊙act'(g),  du = dh⊙act(g),
//   dx = dg·Wg + du·Wu,  dWg = dgᵀ·x,  dWu = duᵀ·x,  dWd = dyᵀ·h.
// One persistent kernel template runs the five products; they differ in the
// operands' major order (read in place through the descriptors: nothing is
// transposed or stacked in memory), in the list of K segments and problems, and
// in what the epilogue does with the fp32 accumulator:
//   hidden      gate and up tiles side by side in one accumulator, so that the
//               activation and the product run on registers; a training forward
//               also stores a = act(g) and b = u⊙act'(g), each rounded once from
//               fp32, which is all the backward needs of g and u: du = dh⊙a and
//               dg = dh⊙b need no exponential and do not depend on the activation;
//   out, dx, dW the accumulator rounded once to the result's type;
//   dhidden     dh stays in fp32 and is multiplied with the a and b tiles.
// Bound: the tensor pipe for long batches (6·T·d·F flops forward, 12·T·d·F
// backward), the weights' bytes for few tokens.
//
// A tile is 128 tokens × 256 columns, K in steps of 64 through a TMA ring; the
// accumulators are double-buffered in TMEM (2 × 256 columns), so that a tile's
// epilogue runs beside the next tile's products.
//   warp 0      TMA loads (128-byte swizzle)
//   warp 1      TMEM owner, single-thread MMA issuer
//   warps 2-9   epilogue: TMEM lane quadrant warp % 4, column half (warp − 2) / 4
// Every wait is bounded (sm100::mbar_wait).
#include <algorithm>
#include <cstring>

#include "ffn.cuh"
#include "sm100.cuh"

namespace dsalt {
namespace ffn {

constexpr int BM = 128, BN = 256, BK = 64;
constexpr int kPiece = 128 * BK * 2;       // 128 rows (or columns) × 64 K of one operand
constexpr int kStageBytes = 3 * kPiece;    // A, and B's two halves
constexpr int kStages = 4;
constexpr int kEpiWarps = 8;
constexpr int kThreads = (2 + kEpiWarps) * 32;
constexpr int kWarpStage = 4096;           // epilogue staging of one warp
constexpr int kMaxProb = 3;
enum { FULL = 0, EMPTY = FULL + kStages, ACC_FULL = EMPTY + kStages, ACC_EMPTY = ACC_FULL + 2, FINAL = ACC_EMPTY + 2,
       NB = FINAL + 1 };
enum Epi { EPI_STORE = 0, EPI_HIDDEN = 1, EPI_DHIDDEN = 2 };

struct alignas(1024) Smem {
  uint8_t ring[kStages][kStageBytes];
  uint8_t stage[kEpiWarps][kWarpStage];
  uint64_t bars[NB];
  uint32_t tmem_base;
  int abort_flag;
};

// One product D[M, N] = Σ over its K segments; out_cols: columns of D.
struct Problem {
  int M, N, m_tiles, n_tiles, tile_end;
  void* out;
  int64_t ld_out;
};

struct alignas(64) Args {
  CUtensorMap ma[kMaxProb], mb[kMaxProb];  // per problem, or per K segment of the only problem
  Problem prob[kMaxProb];
  int n_prob, n_seg, K, n_tiles;
  bool bf16, out_f32;
  int act;
  void *h, *a, *b;        // hidden: outputs (a, b may be null); dhidden: a, b inputs
  void *dg, *du;          // dhidden outputs
  int64_t ld_f;
  int32_t* status;
};

struct Tile { int prob, m0, nt; };
__device__ __forceinline__ Tile decode(const Args& a, int t) {
  Tile r;
  r.prob = 0;
  int begin = 0;
  while (r.prob + 1 < a.n_prob && t >= a.prob[r.prob].tile_end) begin = a.prob[r.prob++].tile_end;
  const int nt = a.prob[r.prob].n_tiles;
  r.m0 = (t - begin) / nt * BM;
  r.nt = (t - begin) % nt;
  return r;
}

// ---------------------------------------------------------------- activation
// act(g) and act'(g).  exp and the reciprocal are the fast ones (relative error
// below 2^-20 over the range where the result is not rounded to 0 or g): the
// results are rounded to 16 bits next.
__device__ __forceinline__ void act_pair(int act, float g, float& a, float& da) {
  if (act == DSALT_ACT_SILU) {
    const float sig = __fdividef(1.f, 1.f + __expf(-g));
    a = g * sig;
    da = sig * (1.f + g - a);
  } else if (act == DSALT_ACT_GELU) {
    const float cdf = normcdff(g);
    a = g * cdf;
    da = fmaf(g * 0.3989422804f, __expf(-0.5f * g * g), cdf);
  } else {
    // ½(1 + tanh z) = σ(2z), ½(1 − tanh² z) = 2σ(1 − σ), z = √(2/π)(g + 0.044715 g³)
    const float g2 = g * g;
    const float z2 = 1.5957691216f * g * fmaf(0.044715f, g2, 1.f);
    const float sig = __fdividef(1.f, 1.f + __expf(-z2));
    const float w = sig * (1.f - sig);
    a = g * sig;
    da = sig + (w > 0.f ? g * w * 1.5957691216f * fmaf(0.134145f, g2, 1.f) : 0.f);
  }
}

// ------------------------------------------------------------------- staging
// A warp's 32 rows × ROWB bytes, in 16-byte units XORed so that a row's owner
// and a row-contiguous copy both touch all banks.
template <int ROWB>
__device__ __forceinline__ uint32_t stage_off(int row, int u) {
  if constexpr (ROWB == 128) return row * 128 + ((u ^ (row & 7)) << 4);
  return row * 64 + ((u ^ ((row >> 1) & 3)) << 4);
}
// staged rows → global rows r0 … (at most `rows`), columns c0 … below N
template <int ROWB, typename E>
__device__ __forceinline__ void stage_to_global(const uint8_t* st, E* out, int64_t ld, int rows, int c0, int N, bool vec) {
  constexpr int kU = ROWB / 16, kE = 16 / sizeof(E);
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kU; ++i) {
    const int idx = i * 32 + lane, row = idx / kU, u = idx % kU;
    const int c = c0 + u * kE;
    if (row >= rows || c >= N) continue;
    const uint4 v = *reinterpret_cast<const uint4*>(st + stage_off<ROWB>(row, u));
    E* dst = out + row * ld + c;
    if (vec && c + kE <= N) {
      *reinterpret_cast<uint4*>(dst) = v;
    } else {
      const E* e = reinterpret_cast<const E*>(&v);
      for (int k = 0; k < kE && c + k < N; ++k) dst[k] = e[k];
    }
  }
}
// global rows → staging (units past the bounds as zeros); 16-byte aligned rows
template <int ROWB>
__device__ __forceinline__ void global_to_stage(uint8_t* st, const uint16_t* in, int64_t ld, int rows, int c0, int N) {
  constexpr int kU = ROWB / 16;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kU; ++i) {
    const int idx = i * 32 + lane, row = idx / kU, u = idx % kU;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < rows && c0 + u * 8 < N) v = *reinterpret_cast<const uint4*>(in + row * ld + c0 + u * 8);
    *reinterpret_cast<uint4*>(st + stage_off<ROWB>(row, u)) = v;
  }
}
// this lane's row of 32 values → 4 units of the staged 16-bit rows
__device__ __forceinline__ void stage_row16(uint8_t* st, int lane, const float* v, bool bf16) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    uint4 w;
    w.x = sm100::pack2(v[8 * u + 0], v[8 * u + 1], bf16);
    w.y = sm100::pack2(v[8 * u + 2], v[8 * u + 3], bf16);
    w.z = sm100::pack2(v[8 * u + 4], v[8 * u + 5], bf16);
    w.w = sm100::pack2(v[8 * u + 6], v[8 * u + 7], bf16);
    *reinterpret_cast<uint4*>(st + stage_off<64>(lane, u)) = w;
  }
}
__device__ __forceinline__ float2 unpack2(uint32_t w, bool bf16) {
  if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// ------------------------------------------------------------------- kernel
// AMN / BMN: the operand's K is the strided dimension (MN-major) instead of the
// contiguous one.  A 128-wide piece of an operand at K offset k0:
//   K-major   one box of 64 k × 128 rows; MMA step k at +32·k bytes
//   MN-major  two boxes of 64 columns × 64 k; MMA step k at +2048·k bytes
template <bool MN>
__device__ __forceinline__ void load_piece(uint32_t dst, const CUtensorMap* map, uint32_t bar, int mn0, int k0) {
  if constexpr (MN) {
    sm100::tma_load_3d(dst, map, bar, mn0, k0, 0);
    sm100::tma_load_3d(dst + kPiece / 2, map, bar, mn0 + 64, k0, 0);
  } else {
    sm100::tma_load_3d(dst, map, bar, k0, mn0, 0);
  }
}
template <bool MN>
__device__ __forceinline__ uint64_t piece_desc(uint32_t addr, int kk) {
  return MN ? sm100::sdesc_sw128(addr + kk * 2048, kPiece / 2, 1024) : sm100::sdesc_sw128(addr + kk * 32, 16, 1024);
}

template <bool AMN, bool BMN, int EPI>
__global__ void __launch_bounds__(kThreads, 1) ffn_gemm_kernel(const __grid_constant__ Args a) {
  using namespace sm100;
  extern __shared__ uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const BarArray bar{smem_u32(&sm.bars[0])};
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar[FULL + s], 1);
      mbar_init(bar[EMPTY + s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar[ACC_FULL + b], 1);
      mbar_init(bar[ACC_EMPTY + b], kEpiWarps);
    }
    mbar_init(bar[FINAL], 1);
    fence_mbar_init();
    sm.abort_flag = 0;
  }
  if (warp == 1) tmem_alloc(smem_u32(&sm.tmem_base), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  volatile int* abort_flag = &sm.abort_flag;
  const int k_tiles = (a.K + BK - 1) / BK;
  const int steps = k_tiles * a.n_seg;

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      int g = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < a.n_tiles; t += gridDim.x) {
        const Tile tl = decode(a, t);
        for (int s = 0; ok && s < steps; ++s, ++g) {
          const int st = g % kStages;
          if (g >= kStages && !mbar_wait(bar[EMPTY + st], (g / kStages - 1) & 1, abort_flag, a.status)) {
            ok = false;
            break;
          }
          const int seg = s / k_tiles, k0 = (s - seg * k_tiles) * BK;
          const int im = a.n_prob > 1 ? tl.prob : seg;
          const uint32_t base = smem_u32(sm.ring[st]);
          mbar_expect_tx(bar[FULL + st], kStageBytes);
          load_piece<AMN>(base, &a.ma[im], bar[FULL + st], tl.m0, k0);
          if constexpr (EPI == EPI_HIDDEN) {  // the same 128 columns of gate and up
            load_piece<BMN>(base + kPiece, &a.mb[0], bar[FULL + st], tl.nt * 128, k0);
            load_piece<BMN>(base + 2 * kPiece, &a.mb[1], bar[FULL + st], tl.nt * 128, k0);
          } else {
            load_piece<BMN>(base + kPiece, &a.mb[im], bar[FULL + st], tl.nt * BN, k0);
            load_piece<BMN>(base + 2 * kPiece, &a.mb[im], bar[FULL + st], tl.nt * BN + 128, k0);
          }
        }
      }
      // never leave a copy in flight into shared memory
      for (int gg = max(0, g - kStages); gg < g; ++gg) mbar_drain(bar[FULL + gg % kStages], (gg / kStages) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t idesc = idesc_f16(a.bf16, BM, BN, AMN, BMN);
      int g = 0, li = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < a.n_tiles; t += gridDim.x, ++li) {
        const int acc = li & 1;
        if (li >= 2) ok = mbar_wait(bar[ACC_EMPTY + acc], ((li >> 1) - 1) & 1, abort_flag, a.status);
        tc_fence_after();
        for (int s = 0; ok && s < steps; ++s, ++g) {
          const int st = g % kStages;
          if (!mbar_wait(bar[FULL + st], (g / kStages) & 1, abort_flag, a.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t base = smem_u32(sm.ring[st]);
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk)
            mma_f16(tmem + acc * BN, piece_desc<AMN>(base, kk), piece_desc<BMN>(base + kPiece, kk), idesc,
                    (s > 0 || kk > 0) ? 1u : 0u);
          mma_commit(bar[EMPTY + st]);
        }
        if (ok) mma_commit(bar[ACC_FULL + acc]);
      }
      mma_commit(bar[FINAL]);
      mbar_drain(bar[FINAL], 0);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int q4 = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_addr = (uint32_t)(32 * q4) << 16;
    uint8_t* st0 = sm.stage[warp - 2];
    int li = 0;
    for (int t = blockIdx.x; t < a.n_tiles; t += gridDim.x, ++li) {
      const Tile tl = decode(a, t);
      const Problem& pr = a.prob[tl.prob];
      const int acc = li & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(bar[ACC_FULL + acc], (li >> 1) & 1, abort_flag, a.status))) break;
      tc_fence_after();
      const uint32_t tacc = tmem + acc * BN + lane_addr;
      const int row0 = tl.m0 + 32 * q4, rows = pr.M - row0;  // rows of this warp (may be <= 0)
      if constexpr (EPI == EPI_HIDDEN) {
#pragma unroll 1
        for (int c = half * 64; c < half * 64 + 64; c += 32) {
          float g[32], u[32];
          tmem_ld32(tacc + c, g);
          tmem_ld32(tacc + 128 + c, u);
          tmem_wait_ld();
          const int col = tl.nt * 128 + c;
          const int64_t at = (int64_t)row0 * a.ld_f;
          float b[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            float av, da;
            act_pair(a.act, g[j], av, da);
            g[j] = av;
            b[j] = u[j] * da;
            u[j] *= av;
          }
          stage_row16(st0, lane, u, a.bf16);
          stage_row16(st0 + 2048, lane, g, a.bf16);
          __syncwarp();
          stage_to_global<64>(st0, (uint16_t*)a.h + at, a.ld_f, rows, col, pr.N, true);
          if (a.a) {
            stage_to_global<64>(st0 + 2048, (uint16_t*)a.a + at, a.ld_f, rows, col, pr.N, true);
            __syncwarp();
            stage_row16(st0, lane, b, a.bf16);
            __syncwarp();
            stage_to_global<64>(st0, (uint16_t*)a.b + at, a.ld_f, rows, col, pr.N, true);
          }
          __syncwarp();
        }
      } else if constexpr (EPI == EPI_DHIDDEN) {
#pragma unroll 1
        for (int c = half * 128; c < half * 128 + 128; c += 32) {
          const int col = tl.nt * BN + c;
          const int64_t at = (int64_t)row0 * a.ld_f;
          global_to_stage<64>(st0, (const uint16_t*)a.a + at, a.ld_f, rows, col, pr.N);
          global_to_stage<64>(st0 + 2048, (const uint16_t*)a.b + at, a.ld_f, rows, col, pr.N);
          float v[32];
          tmem_ld32(tacc + c, v);
          tmem_wait_ld();
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint4* pa = reinterpret_cast<uint4*>(st0 + stage_off<64>(lane, u));
            uint4* pb = reinterpret_cast<uint4*>(st0 + 2048 + stage_off<64>(lane, u));
            uint32_t wa[4], wb[4];
            *reinterpret_cast<uint4*>(wa) = *pa;
            *reinterpret_cast<uint4*>(wb) = *pb;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float d0 = v[8 * u + 2 * k], d1 = v[8 * u + 2 * k + 1];
              const float2 fa = unpack2(wa[k], a.bf16), fb = unpack2(wb[k], a.bf16);
              wa[k] = pack2(d0 * fa.x, d1 * fa.y, a.bf16);
              wb[k] = pack2(d0 * fb.x, d1 * fb.y, a.bf16);
            }
            *pa = *reinterpret_cast<uint4*>(wa);
            *pb = *reinterpret_cast<uint4*>(wb);
          }
          __syncwarp();
          stage_to_global<64>(st0, (uint16_t*)a.du + at, a.ld_f, rows, col, pr.N, true);
          stage_to_global<64>(st0 + 2048, (uint16_t*)a.dg + at, a.ld_f, rows, col, pr.N, true);
          __syncwarp();
        }
      } else {
        const int esz = a.out_f32 ? 4 : 2;
        const bool vec = ((uintptr_t)pr.out & 15) == 0 && (pr.ld_out * esz) % 16 == 0;
#pragma unroll 1
        for (int c = half * 128; c < half * 128 + 128; c += 32) {
          float v[32];
          tmem_ld32(tacc + c, v);
          tmem_wait_ld();
          const int col = tl.nt * BN + c;
          const int64_t at = (int64_t)row0 * pr.ld_out;
          if (a.out_f32) {
#pragma unroll
            for (int u = 0; u < 8; ++u)
              *reinterpret_cast<float4*>(st0 + stage_off<128>(lane, u)) =
                  make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
            __syncwarp();
            stage_to_global<128>(st0, (float*)pr.out + at, pr.ld_out, rows, col, pr.N, vec);
          } else {
            stage_row16(st0, lane, v, a.bf16);
            __syncwarp();
            stage_to_global<64>(st0, (uint16_t*)pr.out + at, pr.ld_out, rows, col, pr.N, vec);
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      if (lane == 0) mbar_arrive(bar[ACC_EMPTY + acc]);  // read: the MMA warp may reuse it
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// --------------------------------------------------------------------- host
// 2-D row-major tensor [rows, cols] with row stride ld (elements), as an operand
// whose 64 × 128 (K-major) or 64 × 64 (MN-major) boxes the kernel loads.
bool encode(CUtensorMap* m, int dtype, const void* base, int64_t rows, int64_t cols, int64_t ld, bool mn) {
  const CUtensorMapDataType dt = dtype == DSALT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode_tensor_map_3d(m, dt, base, (uint64_t)cols, (uint64_t)rows, 1, (uint64_t)ld * 2, (uint64_t)ld * 2, 64,
                              mn ? 64 : 128, 1) == CUDA_SUCCESS;
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

void add_problem(Args& a, int64_t M, int64_t N, int tile_n, void* out, int64_t ld_out) {
  Problem& p = a.prob[a.n_prob];
  p.M = (int)M;
  p.N = (int)N;
  p.m_tiles = (int)((M + BM - 1) / BM);
  p.n_tiles = (int)((N + tile_n - 1) / tile_n);
  p.out = out;
  p.ld_out = ld_out;
  a.n_tiles += p.m_tiles * p.n_tiles;
  p.tile_end = a.n_tiles;
  ++a.n_prob;
}

template <bool AMN, bool BMN, int EPI>
cudaError_t launch(const Args& a, cudaStream_t st) {
  auto kernel = ffn_gemm_kernel<AMN, BMN, EPI>;
  const size_t smem = sizeof(Smem) + 1024;
  cudaError_t e = ensure_smem((const void*)kernel, smem);
  if (e != cudaSuccess) return e;
  int sms = 0;
  if ((e = sm_count(&sms)) != cudaSuccess) return e;
  kernel<<<(unsigned)std::min(a.n_tiles, sms), kThreads, smem, st>>>(a);
  return cudaGetLastError();
}

Args base_args(const DsaltGatedFfnParams& p) {
  Args a;
  memset(&a, 0, sizeof(a));
  a.bf16 = p.dtype == DSALT_BF16;
  a.n_seg = 1;
  a.act = p.activation;
  a.ld_f = p.ld_f;
  a.status = p.status;
  return a;
}

}  // namespace ffn

cudaError_t launch_ffn(int stage, const DsaltGatedFfnParams& p, cudaStream_t st) {
  using namespace ffn;
  Args a = base_args(p);
  const int dt = p.dtype;
  bool ok = true;
  switch (stage) {
    case FFN_HIDDEN:
      ok = encode(&a.ma[0], dt, p.x, p.T, p.d, p.ld_x, false) && encode(&a.mb[0], dt, p.w_gate, p.F, p.d, p.ld_wg, false) &&
           encode(&a.mb[1], dt, p.w_up, p.F, p.d, p.ld_wu, false);
      if (!ok) return cudaErrorInvalidValue;
      a.K = p.d;
      a.h = p.h;
      a.a = p.a;
      a.b = p.b;
      add_problem(a, p.T, p.F, 128, nullptr, 0);
      return launch<false, false, EPI_HIDDEN>(a, st);
    case FFN_OUT:
      ok = encode(&a.ma[0], dt, p.h, p.T, p.F, p.ld_f, false) && encode(&a.mb[0], dt, p.w_down, p.d_out, p.F, p.ld_wd, false);
      if (!ok) return cudaErrorInvalidValue;
      a.K = p.F;
      add_problem(a, p.T, p.d_out, BN, p.y, p.d_out);
      return launch<false, false, EPI_STORE>(a, st);
    case FFN_BWD_HIDDEN:
      ok = encode(&a.ma[0], dt, p.dy, p.T, p.d_out, p.ld_dy, false) && encode(&a.mb[0], dt, p.w_down, p.d_out, p.F, p.ld_wd, true);
      if (!ok) return cudaErrorInvalidValue;
      a.K = p.d_out;
      a.a = p.a;
      a.b = p.b;
      a.dg = p.dg;
      a.du = p.du;
      add_problem(a, p.T, p.F, BN, nullptr, 0);
      return launch<false, true, EPI_DHIDDEN>(a, st);
    case FFN_BWD_INPUT:
      ok = encode(&a.ma[0], dt, p.dg, p.T, p.F, p.ld_f, false) && encode(&a.ma[1], dt, p.du, p.T, p.F, p.ld_f, false) &&
           encode(&a.mb[0], dt, p.w_gate, p.F, p.d, p.ld_wg, true) && encode(&a.mb[1], dt, p.w_up, p.F, p.d, p.ld_wu, true);
      if (!ok) return cudaErrorInvalidValue;
      a.K = p.F;
      a.n_seg = 2;
      add_problem(a, p.T, p.d, BN, p.dx, p.d);
      return launch<false, true, EPI_STORE>(a, st);
    case FFN_BWD_WEIGHTS: {
      a.K = (int)p.T;
      a.out_f32 = p.w_grad_f32 != 0;
      struct { const void* l; int64_t nl, ldl; const void* r; int64_t nr, ldr; void* out; } job[3] = {
          {p.dg, p.F, p.ld_f, p.x, p.d, p.ld_x, p.dw_gate},
          {p.du, p.F, p.ld_f, p.x, p.d, p.ld_x, p.dw_up},
          {p.dy, p.d_out, p.ld_dy, p.h, p.F, p.ld_f, p.dw_down}};
      for (const auto& j : job) {
        if (!j.out) continue;
        const int i = a.n_prob;
        if (!encode(&a.ma[i], dt, j.l, p.T, j.nl, j.ldl, true) || !encode(&a.mb[i], dt, j.r, p.T, j.nr, j.ldr, true))
          return cudaErrorInvalidValue;
        add_problem(a, j.nl, j.nr, BN, j.out, j.nr);
      }
      if (a.n_prob == 0) return cudaSuccess;
      return launch<true, true, EPI_STORE>(a, st);
    }
  }
  return cudaErrorInvalidValue;
}

}  // namespace dsalt

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
//               also stores a = act(g) and b = u⊙act'(g), which is all the backward
//               needs of g and u: du = dh⊙a and dg = dh⊙b need no exponential and do
//               not depend on the activation.  a and b are kept to 24 bits (fp32
//               without its last byte, cut and not rounded, so up to 2^-15 of the value
//               towards 0: two 16-bit words and a word of the two next bytes): rounded
//               to 16 bits they would add a third rounding to dx, dWg and dWu beside
//               those of dg or du and of the result (error against 64 bits 1.73
//               roundings instead of 1.41);
//   out, dx, dW the accumulator rounded once to the result's type;
//   dhidden     dh stays in fp32 and is multiplied with the a and b tiles.
// Bound: the tensor pipe (6·T·d·F flops forward, 12·T·d·F backward).  T = 16384,
// d = 1024, F = 2816, bf16: 648 us of kernels for the step in a replayed graph (1,312
// TFLOP/s; 0.80 of the measured burst rate), in a long loop 790 us at 1.35 to 1.5 GHz under
// the power cap.  Where two times stand beside a choice below, both were taken at the step
// that made it.
//
// A tile is 256 rows × BN columns worked on by a pair of CTAs (a cluster of 2,
// cta_group::2): each holds 128 rows of A, half of B's columns and the accumulator of
// its rows, so that an SM fetches two thirds of what a tile of its own would need.
// K in steps of 64 through a TMA ring; two accumulators in TMEM (2 × BN columns), so
// that a tile's epilogue runs beside the next tile's products.
//   warp 0      TMA loads of this CTA's halves (128-byte swizzle); the leader's FULL
//               barrier counts both CTAs' bytes
//   warp 1      TMEM owner; in the leader the single-thread MMA issuer
//   warps 2-…   epilogue: TMEM lane quadrant warp % 4, 32-column chunks in turn;
//               a lane owns a row, so results are staged in shared memory and copied
//               with row-contiguous 16-byte accesses (TMA stores of the same 64-byte
//               rows shared the TMA unit with the operands' loads: hidden 175 us
//               instead of 163 at T = 16384, d = 1024, F = 2816)
// Every wait is bounded (sm100::mbar_wait).  Launches after the first of a call are
// programmatic dependents: they set up their barriers and TMEM beside the end of the
// launch before, and wait for its completion before they touch memory.
#include <algorithm>
#include <cstring>
#include <initializer_list>

#include "device.cuh"
#include "ffn.cuh"
#include "ffn_act.cuh"

namespace dsalt {
namespace ffn {

constexpr int BM = 256, BK = 64;
constexpr int kPiece = 128 * BK * 2;       // 128 rows (or columns) × 64 K of one operand
constexpr int kBox = 2048;                 // staged box: 32 rows × 64 bytes
constexpr int kMaxProb = 3;
enum Epi { EPI_STORE = 0, EPI_HIDDEN = 1, EPI_DHIDDEN = 2 };

template <int BN, int EPI>
struct Cfg {
  static constexpr int kStageBytes = kPiece + BN / 2 * BK * 2;  // A's and B's halves of this CTA
  // dhidden reads three boxes a chunk from memory: twice the warps keep enough of them on
  // the way (115 us; 129 with 8 warps and a fifth stage).  The others take the stage that
  // the smaller staging leaves (hidden 158 us; 166 with 16 warps and 5 stages).
  static constexpr int kEpiWarps = EPI == EPI_DHIDDEN ? 16 : 8;
  static constexpr int kThreads = (2 + kEpiWarps) * 32;
  static constexpr int kColStep = kEpiWarps / 4 * 32;           // columns from a warp's chunk to its next
  static constexpr int kBoxes = EPI == EPI_DHIDDEN ? 3 : 2;     // staged boxes of a warp
  static constexpr int kStages = EPI == EPI_DHIDDEN || BN == 512 ? 4 : 6;
  // 512 columns fill TMEM with one accumulator: the epilogue waits beside nothing, which
  // only a long K forgives
  static constexpr int kAcc = BN == 512 ? 1 : 2;
  static constexpr int kMmaN = BN == 512 ? 256 : BN, kMmas = BN / kMmaN;
  static constexpr int FULL = 0, EMPTY = kStages, ACC_FULL = 2 * kStages, ACC_EMPTY = ACC_FULL + 2,
                       FINAL = ACC_EMPTY + 2, NB = FINAL + 1;
  struct alignas(1024) Smem {
    uint8_t ring[kStages][kStageBytes];
    uint8_t stage[kEpiWarps][kBoxes * kBox];
    uint64_t bars[NB];
    uint32_t tmem_base;
    int abort_flag;
  };
};

// One product D[M, N] = Σ over its K segments.
struct Problem {
  int M, N, m_tiles, n_tiles, tile_end;
  void* out;
  int64_t ld_out;
};

struct alignas(64) Args {
  CUtensorMap ma[kMaxProb], mb[kMaxProb];  // per problem, or per K segment of the only problem
  Problem prob[kMaxProb];
  int n_prob, n_seg, K, n_tiles;
  bool bf16, out_f32, out_vec, keep;
  bool early;      // launched beside its predecessor in the stream, one of these kernels
  uint16_t* f[5];  // [T, F] stride ld_f: hidden writes h, a, b, ab; dhidden reads a, b, ab, writes du, dg
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

// ------------------------------------------------------------------- staging
// A box of 32 rows × 64 bytes, its 16-byte units XORed with row / 2 % 4: a row's owner
// writes or reads its four units, and four lanes copy a row, without bank conflicts.
__device__ __forceinline__ uint32_t box_off(int row, int u) { return row * 64 + ((u ^ ((row >> 1) & 3)) << 4); }

__device__ __forceinline__ void stage_words(uint8_t* box, int lane, const uint32_t* w) {
#pragma unroll
  for (int u = 0; u < 4; ++u)
    *reinterpret_cast<uint4*>(box + box_off(lane, u)) = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
}
// A staged box → global rows [0, rows) at `out`, `cols` columns: 16-byte accesses, of
// which the last may reach past `cols` (the rows' padding to 8 elements).
template <typename E>
__device__ __forceinline__ void box_to_rows(const uint8_t* box, E* out, int64_t ld, int rows, int cols) {
  constexpr int kE = 16 / sizeof(E);
  const int lane = threadIdx.x & 31, r = lane >> 2, u = lane & 3;
  if (u * kE >= cols) return;
  out += r * ld + u * kE;
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    if (r + i < rows) *reinterpret_cast<uint4*>(out + i * ld) = *reinterpret_cast<const uint4*>(box + box_off(r + i, u));
}
// the same element by element, for results whose rows are not 16-byte aligned
template <typename E>
__device__ __forceinline__ void box_to_elements(const uint8_t* box, E* out, int64_t ld, int rows, int cols) {
  constexpr int kCols = 64 / sizeof(E);
  for (int i = threadIdx.x & 31; i < 32 * kCols; i += 32) {
    const int row = i / kCols, c = i % kCols;
    if (row < rows && c < cols)
      out[row * ld + c] = *reinterpret_cast<const E*>(box + box_off(row, c * (int)sizeof(E) / 16) + c * sizeof(E) % 16);
  }
}
// global rows → a box, asynchronously (zeros outside); cp_async_wait before reading it
__device__ __forceinline__ void rows_to_box(uint32_t box, const uint16_t* in, int64_t ld, int rows, int cols) {
  const int lane = threadIdx.x & 31, r = lane >> 2, u = lane & 3;
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const bool on = r + i < rows && u * 8 < cols;
    const uint16_t* src = on ? in + (r + i) * ld + u * 8 : in;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(box + box_off(r + i, u)), "l"(src), "r"(on ? 16 : 0)
                 : "memory");
  }
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// ------------------------------------------------------------------- kernel
// AMN / BMN: the operand's K is the strided dimension (MN-major) instead of the
// contiguous one.  A piece of W rows (or columns) of an operand at K offset k0:
//   K-major   one box of 64 k × W rows; MMA step k at +32·k bytes
//   MN-major  W / 64 boxes of 64 columns × 64 k; MMA step k at +2048·k bytes
template <bool MN, int W>
__device__ __forceinline__ void load_piece(uint32_t dst, const CUtensorMap* map, uint32_t bar, int mn0, int k0) {
  if constexpr (MN) {
#pragma unroll
    for (int c = 0; c < W; c += 64) sm100::tma_load_3d_pair(dst + c * 128, map, bar, mn0 + c, k0, 0);
  } else {
    sm100::tma_load_3d_pair(dst, map, bar, k0, mn0, 0);
  }
}
template <bool MN>
__device__ __forceinline__ uint64_t piece_desc(uint32_t addr, int kk) {
  return MN ? sm100::sdesc_sw128(addr + kk * 2048, 64 * 128, 1024) : sm100::sdesc_sw128(addr + kk * 32, 16, 1024);
}

template <bool AMN, bool BMN, int EPI, int BN, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Cfg<BN, EPI>::kThreads, 1) ffn_gemm_kernel(const __grid_constant__ Args a) {
  using namespace sm100;
  using C = Cfg<BN, EPI>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  auto& sm = *reinterpret_cast<typename C::Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const BarArray bar{smem_u32(&sm.bars[0])};
  // the next launch may set itself up beside this one; it waits for this one's results
  asm volatile("griddepcontrol.launch_dependents;");
  if (tid == 64) {
    for (int i = 0; i < kMaxProb; ++i) {
      if (i > 0 && i >= a.n_prob && i >= a.n_seg && !(EPI == EPI_HIDDEN && i == 1)) break;
      if (i == 0 || EPI != EPI_HIDDEN) prefetch_tmap(&a.ma[i]);
      prefetch_tmap(&a.mb[i]);
    }
  }
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar[C::FULL + s], 1);
      mbar_init(bar[C::EMPTY + s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar[C::ACC_FULL + b], 1);
      mbar_init(bar[C::ACC_EMPTY + b], 2 * C::kEpiWarps);
    }
    mbar_init(bar[C::FINAL], 1);
    fence_mbar_init();
    sm.abort_flag = 0;
  }
  if (warp == 1) tmem_alloc_pair(smem_u32(&sm.tmem_base), C::kAcc * BN);
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before either signals the other's
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the launch before has written its results
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  volatile int* abort_flag = &sm.abort_flag;
  const int k_tiles = (a.K + BK - 1) / BK;
  const int steps = k_tiles * a.n_seg;
  const int t0 = blockIdx.x >> 1, t_step = gridDim.x >> 1;

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      int g = 0;
      bool ok = true;
      for (int t = t0; ok && t < a.n_tiles; t += t_step) {
        const Tile tl = decode(a, t);
        for (int s = 0; s < steps; ++s, ++g) {
          const int st = g % kStages;
          if (g >= kStages && !mbar_wait(bar[C::EMPTY + st], (g / kStages - 1) & 1, abort_flag, a.status)) {
            ok = false;
            break;
          }
          const int seg = s / k_tiles, k0 = (s - seg * k_tiles) * BK;
          const int im = a.n_prob > 1 ? tl.prob : seg;
          const uint32_t base = smem_u32(sm.ring[st]), full = map_rank(bar[C::FULL + st], 0);
          if (rank == 0) mbar_expect_tx(bar[C::FULL + st], 2 * C::kStageBytes);
          load_piece<AMN, 128>(base, &a.ma[im], full, tl.m0 + 128 * rank, k0);
          if constexpr (EPI == EPI_HIDDEN)  // the same columns of gate (leader) and up (its peer)
            load_piece<BMN, BN / 2>(base + kPiece, &a.mb[rank], full, tl.nt * (BN / 2), k0);
          else  // this CTA's half of each MMA's columns
#pragma unroll
            for (int j = 0; j < C::kMmas; ++j)
              load_piece<BMN, C::kMmaN / 2>(base + kPiece + j * C::kMmaN / 2 * BK * 2, &a.mb[im], full,
                                            tl.nt * BN + j * C::kMmaN + (C::kMmaN / 2) * (int)rank, k0);
        }
      }
      // the last products have read this CTA's shared memory, and their signals have come
      for (int gg = max(0, g - kStages); gg < g; ++gg) mbar_drain(bar[C::EMPTY + gg % kStages], (gg / kStages) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = idesc_f16(a.bf16, BM, C::kMmaN, AMN, BMN);
      int g = 0, li = 0;
      bool ok = true;
      for (int t = t0; ok && t < a.n_tiles; t += t_step, ++li) {
        const int acc = li % C::kAcc;
        if (li >= C::kAcc) ok = mbar_wait(bar[C::ACC_EMPTY + acc], (li / C::kAcc - 1) & 1, abort_flag, a.status);
        tc_fence_after();
        for (int s = 0; ok && s < steps; ++s, ++g) {
          const int st = g % kStages;
          if (!mbar_wait(bar[C::FULL + st], (g / kStages) & 1, abort_flag, a.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t base = smem_u32(sm.ring[st]);
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk)
#pragma unroll
            for (int j = 0; j < C::kMmas; ++j)
              mma_f16_pair(tmem + acc * BN + j * C::kMmaN, piece_desc<AMN>(base, kk),
                           piece_desc<BMN>(base + kPiece + j * C::kMmaN / 2 * BK * 2, kk), idesc, (s > 0 || kk > 0) ? 1u : 0u);
          mma_commit_pair(bar[C::EMPTY + st]);
        }
        if (ok) mma_commit_pair(bar[C::ACC_FULL + acc]);
      }
      mma_commit_pair(bar[C::FINAL]);
    }
    if (lane == 0) mbar_drain(bar[C::FINAL], 0);
  } else {
    // ------------------------------------------------------------ epilogue
    const int q4 = warp & 3, cg = (warp - 2) >> 2;
    const uint32_t lane_addr = (uint32_t)(32 * q4) << 16;
    uint8_t* box = sm.stage[warp - 2];
    const uint32_t box_u32 = smem_u32(box);
    constexpr int kCols = EPI == EPI_HIDDEN ? BN / 2 : BN;  // result columns of a tile
    int li = 0;
    for (int t = t0; t < a.n_tiles; t += t_step, ++li) {
      const Tile tl = decode(a, t);
      const Problem& pr = a.prob[tl.prob];
      const int acc = li % C::kAcc;
      const int row0 = tl.m0 + 128 * (int)rank + 32 * q4, rows = pr.M - row0;  // rows of this warp (may be <= 0)
      const int col0 = tl.nt * kCols, cols = pr.N - col0;
      const int64_t at = EPI == EPI_STORE ? row0 * pr.ld_out + col0 : row0 * a.ld_f + col0;
      auto load_ab = [&](int c) {  // the a, b and ab boxes of columns c (dhidden)
#pragma unroll
        for (int i = 0; i < 3; ++i) rows_to_box(box_u32 + i * kBox, rows > 0 ? a.f[i] + at + c : a.f[i], a.ld_f, rows, cols - c);
        cp_async_commit();
      };
      if constexpr (EPI == EPI_DHIDDEN)  // on the way while the products finish
        if (cg * 32 < kCols) load_ab(cg * 32);
      if (!__all_sync(0xffffffffu, mbar_wait(bar[C::ACC_FULL + acc], (li / C::kAcc) & 1, abort_flag, a.status))) break;
      tc_fence_after();
      const uint32_t tacc = tmem + acc * BN + lane_addr;
      auto release = [&]() {  // this warp has read its part: the products may reuse the accumulator
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_rank(bar[C::ACC_EMPTY + acc], 0));
      };
#pragma unroll 1
      for (int c = cg * 32; c < kCols; c += C::kColStep) {
        const bool last = c + C::kColStep >= kCols;
        if constexpr (EPI == EPI_HIDDEN) {
          uint32_t wh[16], wa[16], wb[16], wl[16];
#pragma unroll
          for (int c2 = 0; c2 < 32; c2 += 16) {  // 16 columns at a time: the values fit the registers
            float g[16], u[16];
            tmem_ld16(tacc + c + c2, g);
            tmem_ld16(tacc + BN / 2 + c + c2, u);
            tmem_wait_ld();
            if (last && c2 == 16) release();
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              float a0, a1, d0, d1;
              act_pair<ACT>(g[j], a0, d0);
              act_pair<ACT>(g[j + 1], a1, d1);
              d0 *= u[j];
              d1 *= u[j + 1];
              const int k = (c2 + j) / 2;
              wh[k] = pack2(u[j] * a0, u[j + 1] * a1, a.bf16);
              wa[k] = upper16(a0, a1);
              wb[k] = upper16(d0, d1);
              wl[k] = next8(a0, d0, a1, d1);
            }
          }
          stage_words(box, lane, wh);
          stage_words(box + kBox, lane, wa);
          __syncwarp();
          box_to_rows(box, a.f[0] + at + c, a.ld_f, rows, cols - c);
          if (a.keep) {
            box_to_rows(box + kBox, a.f[1] + at + c, a.ld_f, rows, cols - c);
            __syncwarp();
            stage_words(box, lane, wb);
            stage_words(box + kBox, lane, wl);
            __syncwarp();
            box_to_rows(box, a.f[2] + at + c, a.ld_f, rows, cols - c);
            box_to_rows(box + kBox, a.f[3] + at + c, a.ld_f, rows, cols - c);
          }
          __syncwarp();
        } else if constexpr (EPI == EPI_DHIDDEN) {
          float v[32];
          tmem_ld32(tacc + c, v);
          cp_async_wait();
          tmem_wait_ld();
          if (last) release();
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint4* pa = reinterpret_cast<uint4*>(box + box_off(lane, u));
            uint4* pb = reinterpret_cast<uint4*>(box + kBox + box_off(lane, u));
            const uint4 va = *pa, vb = *pb, vl = *reinterpret_cast<const uint4*>(box + 2 * kBox + box_off(lane, u));
            uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
            const uint32_t wl[4] = {vl.x, vl.y, vl.z, vl.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float d0 = v[8 * u + 2 * k], d1 = v[8 * u + 2 * k + 1];
              // upper half in bytes 2 and 3, low byte in byte 1, byte 0 cleared
              const uint32_t lo = wl[k];
              const float a0 = __uint_as_float(__byte_perm(wa[k], lo, 0x1040) & 0xffffff00u);
              const float a1 = __uint_as_float(__byte_perm(wa[k], lo, 0x3260) & 0xffffff00u);
              const float b0 = __uint_as_float(__byte_perm(wb[k], lo, 0x1050) & 0xffffff00u);
              const float b1 = __uint_as_float(__byte_perm(wb[k], lo, 0x3270) & 0xffffff00u);
              wa[k] = pack2(d0 * a0, d1 * a1, a.bf16);
              wb[k] = pack2(d0 * b0, d1 * b1, a.bf16);
            }
            *pa = make_uint4(wa[0], wa[1], wa[2], wa[3]);
            *pb = make_uint4(wb[0], wb[1], wb[2], wb[3]);
          }
          __syncwarp();
          box_to_rows(box, a.f[3] + at + c, a.ld_f, rows, cols - c);
          box_to_rows(box + kBox, a.f[4] + at + c, a.ld_f, rows, cols - c);
          __syncwarp();
          if (!last) load_ab(c + C::kColStep);
        } else {
          float v[32];
          tmem_ld32(tacc + c, v);
          tmem_wait_ld();
          if (last) release();
          if (a.out_f32) {  // two boxes of 16 columns
#pragma unroll
            for (int u = 0; u < 8; ++u)
              *reinterpret_cast<float4*>(box + (u >> 2) * kBox + box_off(lane, u & 3)) =
                  make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
            __syncwarp();
            float* out = (float*)pr.out + at + c;
            if (a.out_vec) {
              box_to_rows(box, out, pr.ld_out, rows, cols - c);
              box_to_rows(box + kBox, out + 16, pr.ld_out, rows, cols - c - 16);
            } else {
              box_to_elements(box, out, pr.ld_out, rows, cols - c);
              box_to_elements(box + kBox, out + 16, pr.ld_out, rows, cols - c - 16);
            }
          } else {
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = pack2(v[2 * j], v[2 * j + 1], a.bf16);
            stage_words(box, lane, w);
            __syncwarp();
            uint16_t* out = (uint16_t*)pr.out + at + c;
            if (a.out_vec) box_to_rows(box, out, pr.ld_out, rows, cols - c);
            else box_to_elements(box, out, pr.ld_out, rows, cols - c);
          }
          __syncwarp();
        }
      }
      if (cg * 32 >= kCols) release();
    }
    cp_async_wait();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the peer's products, copies and signals for this CTA are done
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, C::kAcc * BN);
}

// --------------------------------------------------------------------- host
CUtensorMapDataType map_type(int dtype) {
  return dtype == DSALT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}
// 2-D row-major tensor [rows, cols] with row stride ld (elements), as an operand
// whose 64 × W (K-major) or 64 × 64 (MN-major) boxes the kernel loads.
bool encode(CUtensorMap* m, int dtype, const void* base, int64_t rows, int64_t cols, int64_t ld, bool mn, int w) {
  return encode_tensor_map_3d(m, map_type(dtype), base, (uint64_t)cols, (uint64_t)rows, 1, (uint64_t)ld * 2, (uint64_t)ld * 2,
                              64, mn ? 64 : w, 1) == CUDA_SUCCESS;
}
// The products of one launch, before the tile width is chosen.
struct Job { int64_t M, N; void* out; int64_t ld_out; };
struct Jobs {
  const Job* first;
  int n;
  const Job* begin() const { return first; }
  const Job* end() const { return first + n; }
};

int tiles_of(const Jobs& jobs, int cols) {
  int64_t n = 0;
  for (const Job& j : jobs) n += (j.M + BM - 1) / BM * ((j.N + cols - 1) / cols);
  return (int)n;
}

// Tile columns by estimated time: waves of tiles over the pairs × K steps × a step's
// cycles, and the first loads and the last epilogue.  The numbers fit kernels measured
// alone at T = 65 … 16384, d = 512 and 1024, e.g. (us with 256, 128, 64 columns) out at
// T = 512, d = 1024, F = 2816: 18.8, 16.7, 16.2; hidden there: 15.5, 16.8, 19.8; out at
// T = 16384: 75, 90, 165.
int pick_bn(const Jobs& jobs, int steps, bool halves, bool b_mn, int pairs, bool wide = false) {
  struct Width { int bn, step, ends; };
  int best = 256;
  int64_t best_cost = INT64_MAX;
  // 512 columns: a quarter less to fetch for the same products, one accumulator (us with
  // 256 and 512: the weight gradients at T = 16384, d = 1024, F = 2816: 246, 224; at
  // T = 8192, d = 2048, F = 5632: 489, 452)
  if (wide) {
    const int64_t waves = (tiles_of(jobs, 512) + pairs - 1) / pairs;
    best = 512;
    best_cost = waves * (steps * 1150 + 16000);
  }
  for (const Width w : {Width{256, 680, 9500}, Width{128, 590, 4750}, Width{64, 550, 2850}}) {
    if (w.bn == 64 && b_mn) break;  // an MN-major half tile is 64 columns at least
    const int64_t waves = (tiles_of(jobs, halves ? w.bn / 2 : w.bn) + pairs - 1) / pairs;
    const int64_t cost = waves * steps * w.step + w.ends;
    if (cost < best_cost) best = w.bn, best_cost = cost;
  }
  return best;
}

void set_jobs(Args& a, const Jobs& jobs, int cols) {
  for (const Job& j : jobs) {
    Problem& p = a.prob[a.n_prob++];
    p.M = (int)j.M;
    p.N = (int)j.N;
    p.m_tiles = (int)((j.M + BM - 1) / BM);
    p.n_tiles = (int)((j.N + cols - 1) / cols);
    p.out = j.out;
    p.ld_out = j.ld_out;
    a.n_tiles += p.m_tiles * p.n_tiles;
    p.tile_end = a.n_tiles;
  }
}

template <bool AMN, bool BMN, int EPI, int BN, int ACT = 0>
cudaError_t launch_bn(const Args& a, int pairs, cudaStream_t st) {
  auto kernel = ffn_gemm_kernel<AMN, BMN, EPI, BN, ACT>;
  const size_t smem = sizeof(typename Cfg<BN, EPI>::Smem) + 1024;
  cudaError_t e = ensure_smem((const void*)kernel, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min(a.n_tiles, pairs)));
  cfg.blockDim = dim3(Cfg<BN, EPI>::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}
template <bool AMN, bool BMN, int EPI, int ACT = 0>
cudaError_t launch(const Args& a, int bn, int pairs, cudaStream_t st) {
  if (bn == 256) return launch_bn<AMN, BMN, EPI, 256, ACT>(a, pairs, st);
  if constexpr (BMN && EPI == EPI_STORE)
    if (bn == 512) return launch_bn<AMN, BMN, EPI, 512, ACT>(a, pairs, st);
  if constexpr (!BMN)
    if (bn == 64) return launch_bn<AMN, BMN, EPI, 64, ACT>(a, pairs, st);
  return launch_bn<AMN, BMN, EPI, 128, ACT>(a, pairs, st);
}

Args base_args(const DsaltGatedFfnParams& p) {
  Args a;
  memset(&a, 0, sizeof(a));
  a.bf16 = p.dtype == DSALT_BF16;
  a.n_seg = 1;
  a.ld_f = p.ld_f;
  a.status = p.status;
  return a;
}
void set_f(Args& a, std::initializer_list<void*> f) {
  int i = 0;
  for (void* q : f) a.f[i++] = reinterpret_cast<uint16_t*>(q);
}
// the type of the plain products' results, and whether their rows take 16-byte stores
void set_out(Args& a, bool f32) {
  a.out_f32 = f32;
  a.out_vec = true;
  for (int i = 0; i < a.n_prob; ++i)
    a.out_vec = a.out_vec && ((uintptr_t)a.prob[i].out & 15) == 0 && a.prob[i].ld_out * (f32 ? 4 : 2) % 16 == 0;
}

}  // namespace ffn

cudaError_t launch_ffn_tc(int stage, const DsaltGatedFfnParams& p, bool early, cudaStream_t st) {
  using namespace ffn;
  // the tensor maps need the device's context current on this thread, which a thread
  // that has only allocated (a backward's first call) need not have: setting the device does it
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaSetDevice(dev);
  if (e != cudaSuccess) return e;
  int sms = 0;
  if ((e = sm_count(&sms)) != cudaSuccess) return e;
  const int pairs = sms / 2;
  Args a = base_args(p);
  a.early = early;
  const int dt = p.dtype;
  const cudaError_t bad = cudaErrorInvalidValue;
  auto steps = [](int64_t k) { return (int)((k + BK - 1) / BK); };
  switch (stage) {
    case FFN_HIDDEN: {
      a.K = p.d;
      a.keep = p.a != nullptr;
      const Job job = {p.T, p.F, nullptr, 0};
      const Jobs jobs = {&job, 1};
      const int bn = pick_bn(jobs, steps(a.K), true, false, pairs);
      set_jobs(a, jobs, bn / 2);
      set_f(a, {p.h, p.a, p.b, p.ab});
      if (!encode(&a.ma[0], dt, p.x, p.T, p.d, p.ld_x, false, 128) ||
          !encode(&a.mb[0], dt, p.w_gate, p.F, p.d, p.ld_wg, false, bn / 2) ||
          !encode(&a.mb[1], dt, p.w_up, p.F, p.d, p.ld_wu, false, bn / 2))
        return bad;
      if (p.activation == DSALT_ACT_SILU) return launch<false, false, EPI_HIDDEN, DSALT_ACT_SILU>(a, bn, pairs, st);
      if (p.activation == DSALT_ACT_GELU) return launch<false, false, EPI_HIDDEN, DSALT_ACT_GELU>(a, bn, pairs, st);
      return launch<false, false, EPI_HIDDEN, DSALT_ACT_GELU_TANH>(a, bn, pairs, st);
    }
    case FFN_OUT: {
      a.K = p.F;
      const Job job = {p.T, p.d_out, p.y, p.d_out};
      const Jobs jobs = {&job, 1};
      const int bn = pick_bn(jobs, steps(a.K), false, false, pairs);
      set_jobs(a, jobs, bn);
      set_out(a, false);
      if (!encode(&a.ma[0], dt, p.h, p.T, p.F, p.ld_f, false, 128) ||
          !encode(&a.mb[0], dt, p.w_down, p.d_out, p.F, p.ld_wd, false, bn / 2))
        return bad;
      return launch<false, false, EPI_STORE>(a, bn, pairs, st);
    }
    case FFN_BWD_HIDDEN: {
      a.K = p.d_out;
      const Job job = {p.T, p.F, nullptr, 0};
      const Jobs jobs = {&job, 1};
      const int bn = pick_bn(jobs, steps(a.K), false, true, pairs);
      set_jobs(a, jobs, bn);
      set_f(a, {p.a, p.b, p.ab, p.du, p.dg});
      if (!encode(&a.ma[0], dt, p.dy, p.T, p.d_out, p.ld_dy, false, 128) ||
          !encode(&a.mb[0], dt, p.w_down, p.d_out, p.F, p.ld_wd, true, 0))
        return bad;
      return launch<false, true, EPI_DHIDDEN>(a, bn, pairs, st);
    }
    case FFN_BWD_INPUT: {
      a.K = p.F;
      a.n_seg = 2;
      const Job job = {p.T, p.d, p.dx, p.d};
      const Jobs jobs = {&job, 1};
      const int bn = pick_bn(jobs, 2 * steps(a.K), false, true, pairs, true);
      set_jobs(a, jobs, bn);
      set_out(a, false);
      if (!encode(&a.ma[0], dt, p.dg, p.T, p.F, p.ld_f, false, 128) || !encode(&a.ma[1], dt, p.du, p.T, p.F, p.ld_f, false, 128) ||
          !encode(&a.mb[0], dt, p.w_gate, p.F, p.d, p.ld_wg, true, 0) || !encode(&a.mb[1], dt, p.w_up, p.F, p.d, p.ld_wu, true, 0))
        return bad;
      return launch<false, true, EPI_STORE>(a, bn, pairs, st);
    }
    case FFN_BWD_WEIGHTS: {
      a.K = (int)p.T;
      struct { const void* l; int64_t nl, ldl; const void* r; int64_t nr, ldr; void* out; } all[3] = {
          {p.dg, p.F, p.ld_f, p.x, p.d, p.ld_x, p.dw_gate},
          {p.du, p.F, p.ld_f, p.x, p.d, p.ld_x, p.dw_up},
          {p.dy, p.d_out, p.ld_dy, p.h, p.F, p.ld_f, p.dw_down}};
      Job job[3];
      int n = 0;
      for (const auto& j : all) {
        if (!j.out) continue;
        if (!encode(&a.ma[n], dt, j.l, p.T, j.nl, j.ldl, true, 0) || !encode(&a.mb[n], dt, j.r, p.T, j.nr, j.ldr, true, 0))
          return bad;
        job[n++] = Job{j.nl, j.nr, j.out, j.nr};
      }
      if (n == 0) return cudaSuccess;
      const Jobs jobs = {job, n};
      const int bn = pick_bn(jobs, steps(a.K), false, true, pairs, true);
      set_jobs(a, jobs, bn);
      set_out(a, p.w_grad_f32 != 0);
      return launch<true, true, EPI_STORE>(a, bn, pairs, st);
    }
  }
  return bad;
}

}  // namespace dsalt

// W8A8: 8-bit rows (a token's codes and its scale) times 8-bit weights (a
// channel's codes and its scale), exact 32-bit integer sums:
//
//   y[t][c] = fp16(x_scale[t] w_scale[c] sum_k x[t][k] w[c][k] + bias[c] + residual[t][c])
//   gated:   y[t][c] = fp16(silu(g) u) with g from weight row c, u from row n + c
//
// The sum of up to 131071 products of codes fits 32 bits; everything after it
// is fp32 and rounded once.  Three kernels, by the number of tokens:
//   * gemv_kernel: dp4a, a warp per channel; the weights' bytes are all there is;
//   * split_kernel: tcgen05 with 128 weight rows as the MMA's M and the tokens
//     as its N, K shared out over a thread-block cluster that adds the integer
//     sums through distributed shared memory (any order gives the same);
//   * pair_kernel: tcgen05 over CTA pairs, 256 tokens x 256 weight rows a
//     tile, persistent, the epilogue of a tile under the products of the next.
// Every wait on the device is bounded (error flag, no hang).
#include "common.cuh"
#include "tcgen05.cuh"

namespace lmps {
namespace w8 {

constexpr int kMaxK = 131071;  // 2^31 / 2^14: codes of -128 included

struct Args {
  const int8_t* x;
  size_t ldx;
  const float* xs;
  const int8_t* w;
  size_t ldw;
  const float* ws;
  const __half* bias;
  const __half* residual;
  size_t ldr;
  __half* y;
  size_t ldy;
  int m, n, k, swiglu;
};

// y[t][c] from the integer sum(s) and the scales.
__device__ __forceinline__ float linear_value(int acc, float xs, float ws) { return static_cast<float>(acc) * xs * ws; }

// A warp per output channel and four tokens, lanes over K, four products a
// dp4a: for single tokens, where the weights' bytes are all there is.
constexpr int kTokens = 4;
constexpr int kGemvWarps = 4;

template <bool GATED>
__global__ void __launch_bounds__(kGemvWarps* kWarp) gemv_kernel(const Args A) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  const int c = blockIdx.x * kGemvWarps + static_cast<int>(threadIdx.x / kWarp), lane = threadIdx.x % kWarp;
  const int t0 = blockIdx.y * kTokens;
  if (c >= A.n) return;
  const int8_t* w0 = A.w + static_cast<size_t>(c) * A.ldw;
  const int8_t* w1 = w0 + static_cast<size_t>(A.n) * A.ldw;
  const int whole = A.k / 16;
  int acc[2][kTokens] = {};
  for (int j = lane; j < whole; j += kWarp) {
    const int4 a = *reinterpret_cast<const int4*>(w0 + 16 * j);
    const int4 b = GATED ? *reinterpret_cast<const int4*>(w1 + 16 * j) : make_int4(0, 0, 0, 0);
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      if (t0 + t >= A.m) break;
      const int4 v = *reinterpret_cast<const int4*>(A.x + static_cast<size_t>(t0 + t) * A.ldx + 16 * j);
      acc[0][t] = __dp4a(a.x, v.x, __dp4a(a.y, v.y, __dp4a(a.z, v.z, __dp4a(a.w, v.w, acc[0][t]))));
      if (GATED) acc[1][t] = __dp4a(b.x, v.x, __dp4a(b.y, v.y, __dp4a(b.z, v.z, __dp4a(b.w, v.w, acc[1][t]))));
    }
  }
  if (16 * whole + lane < A.k) {  // the last k % 16 elements
    const int i = 16 * whole + lane;
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      if (t0 + t >= A.m) break;
      const int v = A.x[static_cast<size_t>(t0 + t) * A.ldx + i];
      acc[0][t] += w0[i] * v;
      if (GATED) acc[1][t] += w1[i] * v;
    }
  }
#pragma unroll
  for (int t = 0; t < kTokens; ++t) {
    if (t0 + t >= A.m) break;
    const int a = __reduce_add_sync(0xffffffffu, acc[0][t]);
    const int b = GATED ? __reduce_add_sync(0xffffffffu, acc[1][t]) : 0;
    if (lane != 0) continue;
    const size_t row = static_cast<size_t>(t0 + t);
    float v = linear_value(a, A.xs[row], A.ws[c]);
    if (GATED) v = silu_mul(v, linear_value(b, A.xs[row], A.ws[A.n + c]));
    if (A.bias) v += __half2float(A.bias[c]);
    if (A.residual) v += __half2float(A.residual[row * A.ldr + c]);
    A.y[row * A.ldy + c] = __float2half_rn(v);
  }
}


// ---------------------------------------------------------------------------
// tcgen05: kind::i8, signed operands, 32-bit integer accumulators
// ---------------------------------------------------------------------------
using namespace tc;

constexpr int kBK = 128;  // codes a K step: one 128-byte swizzle row

// Instruction descriptor: D s32 (2 at bit 4), A and B signed (1 at bits 7 and 10), both K-major.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
template <int GROUP>
__device__ __forceinline__ void mma_i8(uint32_t tmem, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
  if (GROUP == 2)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(
            tmem),
        "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(
            tmem),
        "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
        : "memory");
}
// Completion of this thread's MMAs so far, to the barrier at this offset in both CTAs of the pair.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The shared::cluster address of `p` in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 2-D TMA load into this CTA's shared memory that reports to a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, "
      "%3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, const void* src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_u32(src))
               : "memory");
}

struct __align__(64) Params {
  CUtensorMap tx;  // codes [m, k], box 128 x (tokens of a CTA)
  CUtensorMap tw;  // weight codes [n or 2n, k], box 128 x (weight rows of a CTA's load)
  CUtensorMap ty;  // y [m, n] fp16, box 64 x 32, 128-byte swizzle (pair_kernel, aligned y)
  Args a;
  int tma_y;    // y goes out by TMA (ty is set)
  int xrows;    // split_kernel: tokens of a tile
  int stages;   // split_kernel: K steps in flight
  int ksteps;   // split_kernel: K steps of each CTA of a cluster
  int tiles_n, tiles;  // pair_kernel: tiles along n, all tiles
  int* error;
};

__device__ __forceinline__ float silu_product(float g, float u) {
  // e^-g past 2^126 makes the quotient 0, which fp16 makes of it anyway
  return __fdividef(g, 1.0f + __expf(-g)) * u;
}

// Shared-memory ring position (slot and the parity of its fill).
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++slot == n) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// --- split_kernel -------------------------------------------------------------
// One tile of 128 weight rows (gated: 64 gate and their 64 up rows) and xrows
// tokens a cluster; CTA z of the cluster multiplies K steps z * ksteps .. .
//   warp 0 lane 0: TMA loads; warp 1 lane 0: MMAs; warps 2-5: sums out of TMEM.
// The int32 partial sums go to the CTA that finishes their channels, [split]
// [rows of the CTA][xrows + 4] in the (by then idle) ring.
constexpr int kSplitThreads = 192;
constexpr int kSplitStages = 8;  // at most
constexpr int kWBytes = 128 * kBK;

template <bool GATED>
__global__ void __launch_bounds__(kSplitThreads) split_kernel(const __grid_constant__ Params P) {
  extern __shared__ unsigned char smem_raw[];
  const Args& A = P.a;
  const int S = P.stages, xbytes = P.xrows * kBK;
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* wt = base;
  unsigned char* xt = base + static_cast<size_t>(S) * kWBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(xt + static_cast<size_t>(S) * xbytes);
  uint64_t* empty = full + kSplitStages;
  uint64_t* done = empty + kSplitStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* abort_v = abort_flag;
  constexpr int kOut = GATED ? 64 : 128;  // channels of a tile

  lmps_pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int c0 = blockIdx.x * kOut, t0 = blockIdx.y * P.xrows;
  const int splits = gridDim.z;
  const int all = (A.k + kBK - 1) / kBK, kbeg = blockIdx.z * P.ksteps;
  const int ksteps = max(0, min(P.ksteps, all - kbeg));
  const uint32_t tcols = P.xrows <= 32 ? 32u : P.xrows <= 64 ? 64u : P.xrows <= 128 ? 128u : 256u;

  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(tcols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;

  if (tid == 0) {
    lmps_pdl_wait();  // both operands may be the previous kernel's output
    Ring r;
    int issued = 0;
    for (int kt = 0; kt < ksteps; ++kt, r.next(S)) {
      if (kt >= S && !mbar_wait(&empty[r.slot], r.phase ^ 1u, P.error, abort_v)) break;
      mbar_expect_tx(&full[r.slot], static_cast<uint32_t>(kWBytes + xbytes));
      unsigned char* w = wt + static_cast<size_t>(r.slot) * kWBytes;
      const int kx = (kbeg + kt) * kBK;
      if (GATED) {
        tma_load_2d(w, &P.tw, kx, c0, &full[r.slot]);
        tma_load_2d(w + kWBytes / 2, &P.tw, kx, A.n + c0, &full[r.slot]);
      } else {
        tma_load_2d(w, &P.tw, kx, c0, &full[r.slot]);
      }
      tma_load_2d(xt + static_cast<size_t>(r.slot) * xbytes, &P.tx, kx, t0, &full[r.slot]);
      issued = kt + 1;
    }
    for (int kt = max(0, issued - S); kt < issued; ++kt) {  // every issued copy lands before the ring is reused
      const uint64_t since = globaltimer();
      while (!mbar_try(&full[kt % S], (kt / S) & 1))
        if (globaltimer() - since > kTimeoutNs) break;
    }
  } else if (warp == 1 && lane == 0) {
    lmps_pdl_wait();  // (bounded waits begin when the work does)
    const uint32_t idesc = idesc_i8(128, P.xrows);
    Ring r;
    for (int kt = 0; kt < ksteps; ++kt, r.next(S)) {
      if (!mbar_wait(&full[r.slot], r.phase, P.error, abort_v)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t wd = sw128_desc(smem_u32(wt + static_cast<size_t>(r.slot) * kWBytes));
      const uint64_t xd = sw128_desc(smem_u32(xt + static_cast<size_t>(r.slot) * xbytes));
#pragma unroll
      for (int j = 0; j < kBK / 32; ++j)  // K = 32 a MMA: 32 bytes further into the swizzle row
        mma_i8<1>(tmem, wd + 2 * j, xd + 2 * j, idesc, (kt > 0 || j > 0) ? 1u : 0u);
      mma_commit(&empty[r.slot]);
    }
    mma_commit(done);
    const uint64_t since = globaltimer();  // the tensor memory and the ring are free once these finish
    while (!mbar_try(done, 0u))
      if (globaltimer() - since > kTimeoutNs) break;
  }
  __syncwarp();
  lmps_pdl_wait();  // before any read of scales and residual, or write of y
  const bool epi = warp >= 2;
  bool ok = false;
  if (epi) {
    ok = mbar_wait(done, 0, P.error, abort_v) && ksteps > 0 && *abort_v == 0;
    ok = __all_sync(0xffffffffu, ok);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  }
  // Every CTA of the cluster is past its products: the rings may receive sums.
  __syncthreads();
  if (splits > 1) cluster_sync();
  int* red = reinterpret_cast<int*>(base);
  const int rs = P.xrows + 4, rows = 128 / splits, outs = kOut / splits;  // sums and channels a CTA finishes
  const uint32_t rank = splits > 1 ? cluster_rank() : 0u;
  if (epi) {
    const int q = warp & 3, row = 32 * q + lane;  // TMEM lane = row of the tile
    const int half = GATED ? row / 64 : 0, c = row % kOut;
    const int slot = static_cast<int>(rank) * rows + half * outs + c % outs;
    const uint32_t to = cluster_addr(red + static_cast<size_t>(slot) * rs, static_cast<uint32_t>(c / outs));
    const uint32_t tl = tmem + (static_cast<uint32_t>(32 * q) << 16);
    for (int j0 = 0; j0 < P.xrows; j0 += 32) {
      uint32_t v[32];
      if (ok) {
        tmem_ld32(tl + j0, v);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = 0u;
      }
#pragma unroll
      for (int j = 0; j < 32; j += 4)
        if (j0 + j < P.xrows)
          asm volatile("st.shared::cluster.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to + (j0 + j) * 4), "r"(v[j]),
                       "r"(v[j + 1]), "r"(v[j + 2]), "r"(v[j + 3])
                       : "memory");
    }
  }
  if (splits > 1) cluster_sync();
  __syncthreads();
  const int tok = min(P.xrows, A.m - t0), tok4 = (tok + 3) / 4;
  const int cbase = c0 + static_cast<int>(rank) * outs;
  for (int i = tid; i < outs * tok4; i += kSplitThreads) {
    const int lc = i % outs, j = 4 * (i / outs), c = cbase + lc;
    if (c >= A.n) continue;
    int g[4] = {0, 0, 0, 0}, u[4] = {0, 0, 0, 0};
    for (int z = 0; z < splits; ++z) {
      const int4 v = *reinterpret_cast<const int4*>(red + static_cast<size_t>(z * rows + lc) * rs + j);
      g[0] += v.x, g[1] += v.y, g[2] += v.z, g[3] += v.w;
      if (GATED) {
        const int4 b = *reinterpret_cast<const int4*>(red + static_cast<size_t>(z * rows + outs + lc) * rs + j);
        u[0] += b.x, u[1] += b.y, u[2] += b.z, u[3] += b.w;
      }
    }
    const float ws = A.ws[c], wu = GATED ? A.ws[A.n + c] : 0.0f, bias = A.bias ? __half2float(A.bias[c]) : 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (j + e >= tok) break;
      const size_t row = static_cast<size_t>(t0 + j + e);
      const float xs = A.xs[row];
      float v = linear_value(g[e], xs, ws);
      if (GATED) v = silu_product(v, linear_value(u[e], xs, wu));
      v += bias;
      if (A.residual) v += __half2float(A.residual[row * A.ldr + c]);
      A.y[row * A.ldy + c] = __float2half_rn(v);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tcols) : "memory");
}

static size_t split_smem(int stages, int xrows) {
  return static_cast<size_t>(stages) * (kWBytes + xrows * kBK) + 1024 + (2 * kSplitStages + 1) * sizeof(uint64_t) + 16;
}

// --- pair_kernel ----------------------------------------------------------------
// A tile: 256 tokens (128 for each CTA of the pair) x BN weight rows (each CTA
// loads BN / 2 of them; gated: the first CTA gate rows, the second their up
// rows, so that a CTA's accumulator holds a token's gates in columns 0 .. and
// their up values BN / 2 further).  One elected thread of the first CTA issues
// the MMAs of both.  Each pair walks tiles pair, + pairs, ..; two accumulators
// in tensor memory.
//   warp 0 lane 0: TMA loads of this CTA's half of both operands
//   warp 1 lane 0 of the first CTA: MMAs
//   warps 2-9: epilogue (TMEM lanes 32 (w % 4) .., half of the columns each)
constexpr int kPairThreads = 320;
constexpr int kEpiWarps = 8;
constexpr int kPairStages = 5;

template <int BN>
struct PairShape {
  static constexpr int kX = 128 * kBK, kW = BN / 2 * kBK;
  static constexpr int kStage = kX + kW;
  static constexpr int kStore = kEpiWarps * 32 * 128;  // 32 rows x 64 fp16 a warp
  static constexpr int kCols = kEpiWarps * BN * 4;  // a warp's BN / 2 scales and biases (gated: BN / 4 gate and up scales)
  static constexpr size_t kSmem = static_cast<size_t>(kPairStages) * kStage + kStore + kCols + 1024 +
                                  (2 * kPairStages + 5) * sizeof(uint64_t) + 16;
};

// Bounded wait for a barrier that threads of both CTAs arrive at.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, int* err, volatile int* abort_flag) {
  const uint64_t t0 = globaltimer();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if (*abort_flag) return false;
    if (globaltimer() - t0 > kTimeoutNs) {
      atomicExch(err, 1);
      *abort_flag = 1;
      return false;
    }
  }
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <int BN, bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1) pair_kernel(const __grid_constant__ Params P) {
  using Sh = PairShape<BN>;
  constexpr int S = kPairStages;
  constexpr int kOut = GATED ? BN / 2 : BN;  // channels of a tile
  constexpr uint32_t kTmem = BN > 128 ? 512u : 256u;
  constexpr uint32_t kAcc = kTmem / 2;  // columns from one accumulator to the other
  extern __shared__ unsigned char smem_raw[];
  const Args& A = P.a;
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* stage = base;  // [S] codes tile, weight tile
  unsigned char* store = base + static_cast<size_t>(S) * Sh::kStage;
  float* cols = reinterpret_cast<float*>(store + Sh::kStore);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<unsigned char*>(cols) + Sh::kCols);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;   // [2] accumulator complete
  uint64_t* tempty = tfull + 2;  // [2] accumulator read by both CTAs' epilogues (the first CTA's counts)
  uint64_t* done = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* abort_v = abort_flag;

  lmps_pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int ksteps = (A.k + kBK - 1) / kBK;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 2 * kEpiWarps);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      lmps_pdl_wait();  // both operands may be the previous kernel's output
      Ring r;
      int issued = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < P.tiles; tile += pairs) {
        const int c0 = (tile % P.tiles_n) * kOut, t0 = (tile / P.tiles_n) * 256 + static_cast<int>(rank) * 128;
        const int w0 = GATED ? static_cast<int>(rank) * A.n + c0 : c0 + static_cast<int>(rank) * (BN / 2);
        for (int kt = 0; kt < ksteps; ++kt, r.next(S)) {
          if (issued >= S && !mbar_wait(&empty[r.slot], r.phase ^ 1u, P.error, abort_v)) {
            ok = false;
            break;
          }
          // the first CTA's barrier counts the bytes of both
          if (rank == 0) mbar_expect_tx(&full[r.slot], 2u * Sh::kStage);
          const uint32_t bar = cluster_addr(&full[r.slot], 0);
          unsigned char* x = stage + static_cast<size_t>(r.slot) * Sh::kStage;
          tma_load_pair(x, &P.tx, kt * kBK, t0, bar);
          tma_load_pair(x + Sh::kX, &P.tw, kt * kBK, w0, bar);
          ++issued;
        }
      }
      // every copy has landed and every release of a stage has reached this CTA before it leaves
      for (int g = max(0, issued - S); g < issued; ++g) {
        const uint64_t since = globaltimer();
        while (!mbar_try(&empty[g % S], (g / S) & 1))
          if (globaltimer() - since > kTimeoutNs) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      lmps_pdl_wait();  // (bounded waits begin when the work does)
      constexpr uint32_t idesc = idesc_i8(256, BN);
      Ring r;
      uint32_t uses[2] = {0u, 0u};
      int buf = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < P.tiles; tile += pairs, buf ^= 1) {
        if (!mbar_wait_cluster(&tempty[buf], (uses[buf] & 1u) ^ 1u, P.error, abort_v)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t acc = tmem + static_cast<uint32_t>(buf) * kAcc;
        for (int kt = 0; kt < ksteps; ++kt, r.next(S)) {
          if (!mbar_wait(&full[r.slot], r.phase, P.error, abort_v)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t x = smem_u32(stage + static_cast<size_t>(r.slot) * Sh::kStage);
          const uint64_t xd = sw128_desc(x), wd = sw128_desc(x + Sh::kX);
#pragma unroll
          for (int j = 0; j < kBK / 32; ++j)
            mma_i8<2>(acc, xd + 2 * j, wd + 2 * j, idesc, (kt > 0 || j > 0) ? 1u : 0u);
          commit_pair(&empty[r.slot]);
        }
        if (!ok) break;
        commit_pair(&tfull[buf]);
        ++uses[buf];
      }
      commit_pair(done);
    }
  } else {
    lmps_pdl_wait();  // before any read of scales and residual, or write of y
    const int e = warp - 2, q = warp & 3, part = e / 4;  // part: which half of the columns
    unsigned char* mine = store + e * (32 * 128);
    float* ws = cols + e * BN;  // this warp's scales and biases (gated: gate and up scales)
    float* bs = ws + BN / 2;
    uint32_t uses[2] = {0u, 0u};
    int buf = 0;
    for (int tile = pair; tile < P.tiles; tile += pairs, buf ^= 1) {
      const int c0 = (tile % P.tiles_n) * kOut, t0 = (tile / P.tiles_n) * 256 + static_cast<int>(rank) * 128;
      constexpr int kMine = kOut / 2;  // channels of this warp's half, from first on
      const int first = part * kMine;
      __syncwarp();
      for (int i = lane; i < kMine; i += 32) {
        const int c = c0 + first + i;
        const bool in = c < A.n;
        ws[i] = in ? A.ws[c] : 0.0f;
        bs[i] = GATED ? (in ? A.ws[A.n + c] : 0.0f) : (in && A.bias ? __half2float(A.bias[c]) : 0.0f);
      }
      const int row = t0 + 32 * q + lane;
      const bool live = row < A.m;
      const float xs = live ? A.xs[row] : 0.0f;
      __syncwarp();
      if (!__all_sync(0xffffffffu, mbar_wait(&tfull[buf], uses[buf] & 1u, P.error, abort_v))) break;
      ++uses[buf];
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t tl = tmem + static_cast<uint32_t>(buf) * kAcc + (static_cast<uint32_t>(32 * q) << 16);
#pragma unroll 1
      for (int o = first; o < first + kMine; o += 32) {  // 32 channels a time, half a store box
        uint32_t packed[16];
        if (GATED) {
          uint32_t g[32], u[32];
          tmem_ld32(tl + o, g);
          tmem_ld32(tl + kOut + o, u);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float a = silu_product(linear_value(static_cast<int>(g[j]), xs, ws[o - first + j]),
                                         linear_value(static_cast<int>(u[j]), xs, bs[o - first + j]));
            const float b = silu_product(linear_value(static_cast<int>(g[j + 1]), xs, ws[o - first + j + 1]),
                                         linear_value(static_cast<int>(u[j + 1]), xs, bs[o - first + j + 1]));
            const __half2 h = __floats2half2_rn(a, b);
            packed[j / 2] = *reinterpret_cast<const uint32_t*>(&h);
          }
        } else {
          uint32_t g[32];
          tmem_ld32(tl + o, g);
          float res[32];
          if (A.residual) {
            const __half* rr = A.residual + static_cast<size_t>(row) * A.ldr + c0 + o;
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              if (P.tma_y && live && c0 + o + j + 8 <= A.n) {  // (then residual rows are 16-byte aligned)
                const uint4 v = *reinterpret_cast<const uint4*>(rr + j);
                const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 f = __half22float2(h[i]);
                  res[j + 2 * i] = f.x, res[j + 2 * i + 1] = f.y;
                }
              } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) res[j + i] = live && c0 + o + j + i < A.n ? __half2float(rr[j + i]) : 0.0f;
              }
            }
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float a = linear_value(static_cast<int>(g[j]), xs, ws[o - first + j]) + bs[o - first + j];
            float b = linear_value(static_cast<int>(g[j + 1]), xs, ws[o - first + j + 1]) + bs[o - first + j + 1];
            if (A.residual) a += res[j], b += res[j + 1];
            const __half2 h = __floats2half2_rn(a, b);
            packed[j / 2] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
        if (P.tma_y) {
          const int box = o & 32;  // first or second half of a 64-column box
          if (box == 0) {          // the box's last store has left the buffer
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4*>(mine + lane * 128 + (((box / 8 + j) ^ (lane & 7)) << 4)) =
                make_uint4(packed[4 * j], packed[4 * j + 1], packed[4 * j + 2], packed[4 * j + 3]);
          if (box != 0) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0 && c0 + o - 32 < A.n && t0 + 32 * q < A.m) {
              tma_store_2d(&P.ty, c0 + o - 32, t0 + 32 * q, mine);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          }
        } else if (live) {
          __half* y = A.y + static_cast<size_t>(row) * A.ldy + c0 + o;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c0 + o + j < A.n) y[j] = reinterpret_cast<const __half*>(packed)[j];
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive_cluster(cluster_addr(&tempty[buf], 0));
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    if (lane == 0) {  // every MMA is finished before the tensor memory is freed (the commit reaches both CTAs)
      const uint64_t since = globaltimer();
      while (!mbar_try(done, 0u))
        if (globaltimer() - since > 2 * kTimeoutNs) break;
    }
    __syncwarp();
  }
  cluster_sync();  // neither CTA leaves while the other reads or signals its memory
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem) : "memory");
}

// --- host side ---------------------------------------------------------------------
static int device_sms(int* sms) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
  return static_cast<int>(e);
}

static bool encode_codes(CUtensorMap* map, const int8_t* p, int k, size_t rows, size_t ld, int box_rows) {
  return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, p, static_cast<uint64_t>(k), rows, ld, kBK,
                   static_cast<uint32_t>(box_rows), CU_TENSOR_MAP_SWIZZLE_128B);
}

static int launch_gemv(const Args& A, cudaStream_t st) {
  const dim3 grid((A.n + kGemvWarps - 1) / kGemvWarps, (A.m + kTokens - 1) / kTokens);
  return lmps_launch_pdl(A.swiglu ? gemv_kernel<true> : gemv_kernel<false>, grid, dim3(kGemvWarps * kWarp), 0, st, A);
}

static int launch_split(const Args& A, int* error, cudaStream_t st) {
  Params P{};
  P.a = A;
  P.error = error;
  P.xrows = A.m >= 128 ? 128 : (A.m + 15) / 16 * 16;
  const int out = A.swiglu ? 64 : 128;
  const int tiles = (A.n + out - 1) / out, ty = (A.m + P.xrows - 1) / P.xrows, steps = (A.k + kBK - 1) / kBK;
  int sms = 148;
  if (const int e = device_sms(&sms)) return e;
  int splits = 1;  // about two CTAs an SM, at least two K steps each
  while (2 * splits <= 8 && 2 * splits * tiles * ty <= 2 * sms && 4 * splits <= steps) splits *= 2;
  P.ksteps = (steps + splits - 1) / splits;
  int stages = P.ksteps < 6 ? P.ksteps : 6;
  while (stages > 2 && split_smem(stages, P.xrows) > 113 * 1024) --stages;
  // the ring also holds the sums: 128 rows of xrows + 4
  while (static_cast<size_t>(stages) * (kWBytes + P.xrows * kBK) < static_cast<size_t>(128) * (P.xrows + 4) * 4) ++stages;
  P.stages = stages;
  const size_t w_rows = static_cast<size_t>(A.n) * (A.swiglu ? 2 : 1);
  if (!encode_codes(&P.tx, A.x, A.k, static_cast<size_t>(A.m), A.ldx, P.xrows) ||
      !encode_codes(&P.tw, A.w, A.k, w_rows, A.ldw, out))
    return LMPS_ERR_INVALID_ARGUMENT;
  const size_t smem = split_smem(stages, P.xrows);
  const int attr = A.swiglu ? lmps_max_dyn_smem<split_kernel<true>>(static_cast<int>(smem))
                            : lmps_max_dyn_smem<split_kernel<false>>(static_cast<int>(smem));
  if (attr != LMPS_OK) return attr;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles, ty, splits);
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 1;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = static_cast<unsigned>(splits);
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, A.swiglu ? split_kernel<true> : split_kernel<false>, P);
  return e == cudaSuccess ? lmps_launch_status() : static_cast<int>(e);
}

template <int BN, bool GATED>
static int launch_pair(const Args& A, int* error, cudaStream_t st) {
  Params P{};
  P.a = A;
  P.error = error;
  constexpr int kOut = GATED ? BN / 2 : BN;
  P.tiles_n = (A.n + kOut - 1) / kOut;
  const long long tiles = static_cast<long long>(P.tiles_n) * ((A.m + 255) / 256);
  if (tiles > (1ll << 30)) return LMPS_ERR_UNSUPPORTED;
  P.tiles = static_cast<int>(tiles);
  const size_t w_rows = static_cast<size_t>(A.n) * (GATED ? 2 : 1);
  if (!encode_codes(&P.tx, A.x, A.k, static_cast<size_t>(A.m), A.ldx, 128) ||
      !encode_codes(&P.tw, A.w, A.k, w_rows, A.ldw, BN / 2))
    return LMPS_ERR_INVALID_ARGUMENT;
  P.tma_y = A.ldy % 8 == 0 && lmps_aligned(A.y, 16) &&
            (!A.residual || (A.ldr % 8 == 0 && lmps_aligned(A.residual, 16)));
  if (P.tma_y && !encode_2d(&P.ty, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, A.y, static_cast<uint64_t>(A.n),
                            static_cast<uint64_t>(A.m), A.ldy * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B))
    return LMPS_ERR_INVALID_ARGUMENT;
  constexpr int kBytes = static_cast<int>(PairShape<BN>::kSmem);
  const int attr = lmps_max_dyn_smem<pair_kernel<BN, GATED>>(kBytes);
  if (attr != LMPS_OK) return attr;
  int sms = 148;
  if (const int e = device_sms(&sms)) return e;
  const int pairs = P.tiles < sms / 2 ? P.tiles : sms / 2;
  return lmps_launch_pdl(pair_kernel<BN, GATED>, dim3(2 * pairs), dim3(kPairThreads), kBytes, st, P);
}

}  // namespace w8
}  // namespace lmps

using namespace lmps;

extern "C" int lmps_w8a8_gemm(const int8_t* x, int ldx, const float* x_scales, const int8_t* w, int ldw,
                              const float* w_scales, const uint16_t* bias, const uint16_t* residual, int ldr,
                              uint16_t* y, int ldy, int m, int n, int k, int swiglu, int32_t* error, void* stream) {
  LMPS_CHECK_ARG(x && x_scales && w && w_scales && y && error);
  LMPS_CHECK_ARG(m >= 1 && n >= 1 && k >= 1 && (swiglu == 0 || swiglu == 1));
  LMPS_CHECK_ARG(ldx >= k && ldx % 16 == 0 && ldw >= k && ldw % 16 == 0 && ldy >= n);
  LMPS_CHECK_ARG(!residual || ldr >= n);
  LMPS_CHECK_ARG(!swiglu || (!bias && !residual));
  LMPS_CHECK_ARG(lmps_aligned(x, 16) && lmps_aligned(w, 16) && lmps_aligned(x_scales, 4) && lmps_aligned(w_scales, 4));
  LMPS_CHECK_ARG(lmps_aligned(y, 2) && lmps_aligned(bias, 2) && lmps_aligned(residual, 2) && lmps_aligned(error, 4));
  if (k > w8::kMaxK || n > (1 << 30)) return LMPS_ERR_UNSUPPORTED;
  w8::Args A{};
  A.x = x;
  A.ldx = static_cast<size_t>(ldx);
  A.xs = x_scales;
  A.w = w;
  A.ldw = static_cast<size_t>(ldw);
  A.ws = w_scales;
  A.bias = reinterpret_cast<const __half*>(bias);
  A.residual = reinterpret_cast<const __half*>(residual);
  A.ldr = static_cast<size_t>(residual ? ldr : 0);
  A.y = reinterpret_cast<__half*>(y);
  A.ldy = static_cast<size_t>(ldy);
  A.m = m;
  A.n = n;
  A.k = k;
  A.swiglu = swiglu;
  cudaStream_t st = lmps_stream(stream);
  if (m <= w8::kTokens) return w8::launch_gemv(A, st);
  if (m <= 256) return w8::launch_split(A, error, st);
  return swiglu ? w8::launch_pair<256, true>(A, error, st) : w8::launch_pair<256, false>(A, error, st);
}

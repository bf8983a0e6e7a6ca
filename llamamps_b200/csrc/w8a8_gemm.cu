// W8A8: 8-bit rows (a token's codes and its scale) times 8-bit weights (a
// channel's codes and its scale), exact 32-bit integer sums:
//
//   y[t][c] = fp16(x_scale[t] w_scale[c] sum_k x[t][k] w[c][k] + bias[c] + residual[t][c])
//   gated:   y[t][c] = fp16(silu(g) u) with g from weight row c, u from row n + c
//
// The sum of up to 131071 products of codes fits 32 bits; everything after it
// is fp32 and rounded once.  Four kernels, by the number of tokens:
//   * few_kernel: mma.sync on weights straight from global memory; their bytes are all there is;
//   * split_kernel: tcgen05 with 128 weight rows as the MMA's M and the tokens
//     as its N, K shared out over a thread-block cluster that adds the integer
//     sums through distributed shared memory (any order gives the same);
//   * whole_kernel: tcgen05 with the tokens as rows, for wide outputs;
//   * pair_kernel: tcgen05 over CTA pairs, 256 tokens x 256 or 128 weight rows
//     a tile, persistent, the epilogue of a tile under the products of the
//     next; with few tiles, several pairs share a tile's K out.
// Every wait on the device is bounded (error flag, no hang).
#include <type_traits>

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
  int m, n, k;
};

// The scaled sum, and the bias in the rounding of the second product.  Every kernel goes through the same roundings
// (this, then the residual), so a token's result does not depend on the other tokens of its call.  Where there is no
// residual, nothing is added or kNone, which leaves a zero's sign as well.
constexpr float kNone = -0.0f;
__device__ __forceinline__ float linear_value(int acc, float xs, float ws, float bias = 0.0f) {
  return fmaf(__fmul_rn(static_cast<float>(acc), xs), ws, bias);
}

// 2^x and 1 / x to some 2^-22, results below 2^-126 as zero: e^-g past 2^126 makes silu(g) 0, and so the product with
// any up value below some 2^94, which fp16 would round to 0.  (Codes and scales of fp16 rows give less than 2^64: a sum
// of 2^31, scales below 2^10 and, behind a norm, 2^18.)
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kMinusLog2e = -1.4426950408889634f;
__device__ __forceinline__ float silu_product(float g, float u) {
  return __fmul_rn(__fmul_rn(g, rcp_fast(__fadd_rn(exp2_fast(__fmul_rn(g, kMinusLog2e)), 1.0f))), u);
}

// --- few_kernel -----------------------------------------------------------------
// A CTA per 16 channels (gated: 16 gate rows and their up rows) and all of up
// to 8 NT tokens; its warps share K out in chunks of 64 codes and add their
// sums through shared memory.  mma.sync with the weights as the 16 rows: the
// order of k within a product is free as long as both operands have the same,
// so lane l holds codes 16 (l % 4) .. of the chunk of its rows, 16 bytes of
// global memory each, as they come; nothing is staged.  Bound by the weights'
// bytes behind a kernel's start: 1 x 8960 x 1536 gated 7.0 us out of DRAM (3.9
// TB/s), 5.4 out of L2; 1 x 2048 x 1536 2.4 us.
__device__ __forceinline__ uint4 load_codes(const int8_t* p, int left) {  // 16 codes, those from `left` on zero
  if (left >= 16) return *reinterpret_cast<const uint4*>(p);
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (left > 0) {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 15; ++i)
      if (i < left) w[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(p[i])) << (8 * (i % 4));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

template <int NT, bool GATED, int WARPS>
__global__ void __launch_bounds__(WARPS* kWarp) few_kernel(const Args A) {
  constexpr int kRows = 16, kToks = 8 * NT, kW = GATED ? 2 : 1;
  // chunks a warp has on their way: the more warps an SM holds the fewer (64 x 8960 gated rows, 8 warps a CTA: 7.1 us
  // with one, 9.1 with two; 1536 x 8960, 32 warps: 5.3 with three, 6.6 with one)
  constexpr int kAhead = WARPS == 32 ? (NT * kW == 1 ? 3 : 1) : 2 / kW;
  constexpr int kPitch = kRows + 4;                                // (the four token pairs of a row: other banks)
  __shared__ int red[WARPS][kW][kToks][kPitch];
  lmps_pdl_trigger();
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
  const int r = lane / 4, at = 16 * (lane % 4);
  const int c0 = blockIdx.x * kRows, chunks = (A.k + 63) / 64;
  const int8_t* w[kW][2];  // this lane's two weight rows (gated: and their up rows)
  bool in[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = c0 + r + 8 * h;
    in[h] = c < A.n;
#pragma unroll
    for (int z = 0; z < kW; ++z)
      w[z][h] = A.w + static_cast<size_t>(z * A.n + (in[h] ? c : 0)) * A.ldw + at;
  }
  for (int i = warp; i < chunks; i += WARPS)  // the weights come nearer while the kernel before ends
    if (64 * i + at < A.k)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int z = 0; z < kW; ++z)
          if (in[h]) prefetch_l2(w[z][h] + 64 * i);
  lmps_pdl_wait();
  int acc[kW][NT][4] = {};
  for (int i0 = warp; i0 < chunks; i0 += kAhead * WARPS) {
    uint4 wv[kAhead][kW][2], xv[kAhead][NT];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int k0 = 64 * (i0 + j * WARPS), left = A.k - k0 - at;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int z = 0; z < kW; ++z) wv[j][z][h] = load_codes(w[z][h] + k0, in[h] ? left : 0);
#pragma unroll
      for (int t = 0; t < NT; ++t)
        xv[j][t] = load_codes(A.x + static_cast<size_t>(8 * t + r) * A.ldx + at + k0, 8 * t + r < A.m ? left : 0);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int z = 0; z < kW; ++z) {
          const uint4 &lo = wv[j][z][0], &hi = wv[j][z][1], &x = xv[j][t];
          mma_s8(acc[z][t], lo.x, hi.x, lo.y, hi.y, x.x, x.y);
          mma_s8(acc[z][t], lo.z, hi.z, lo.w, hi.w, x.z, x.w);
        }
  }
  // what the sums meet, on its way before they do: output o = 16 token + channel
  constexpr int kOuts = kRows * kToks, kMine = (kOuts + WARPS * kWarp - 1) / (WARPS * kWarp);
  float ws[kMine], wu[kMine], xs[kMine], bias[kMine], res[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int o = static_cast<int>(threadIdx.x) + i * WARPS * kWarp, t = o / kRows, c = c0 + o % kRows;
    const bool live = o < kOuts && t < A.m && c < A.n;
    ws[i] = live ? A.ws[c] : 0.0f;
    wu[i] = GATED && live ? A.ws[A.n + c] : 0.0f;
    xs[i] = live ? A.xs[t] : 0.0f;
    bias[i] = live && A.bias ? __half2float(A.bias[c]) : 0.0f;
    res[i] = live && A.residual ? __half2float(A.residual[static_cast<size_t>(t) * A.ldr + c]) : kNone;
  }
#pragma unroll
  for (int z = 0; z < kW; ++z)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[warp][z][8 * t + 2 * (lane % 4) + (e & 1)][r + 8 * (e >> 1)] = acc[z][t][e];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int o = static_cast<int>(threadIdx.x) + i * WARPS * kWarp, t = o / kRows, row = o % kRows;
    if (o >= kOuts || t >= A.m || c0 + row >= A.n) continue;
    int g = 0, u = 0;
#pragma unroll
    for (int v = 0; v < WARPS; ++v) {
      g += red[v][0][t][row];
      if (GATED) u += red[v][kW - 1][t][row];
    }
    float v = linear_value(g, xs[i], ws[i], bias[i]);
    if (GATED) v = silu_product(v, linear_value(u, xs[i], wu[i]));
    A.y[static_cast<size_t>(t) * A.ldy + c0 + row] = __float2half_rn(v + res[i]);
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
// Issued by the lane with `lead`, inside uniform code of the whole warp: descriptors then stay in uniform registers
// (a branch to one lane moved each there, 16384 x 8960 x 1536 gated 324 us instead of 308).
template <int GROUP>
__device__ __forceinline__ void mma_i8(uint32_t tmem, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc,
                                       uint32_t lead) {
  if (GROUP == 2)
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(tmem),
        "l"(ad), "l"(bd), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(tmem),
        "l"(ad), "l"(bd), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
// Completion of this thread's MMAs so far, to the barrier at this offset in both CTAs of the pair.
__device__ __forceinline__ void commit_pair(uint64_t* bar, uint32_t first_cta, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
      " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3u << first_cta)), "r"(lead)
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
// All CTAs of the cluster have come here.  Relaxed: the barriers' own fence publishes them, sums and tiles are published
// by the barriers that count them, and a release took half a microsecond.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 2-D TMA load into this CTA's shared memory that reports to a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar,
                                              uint32_t lead) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %5, 0;\n"
      " @q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
      "{%2, %3}], [%4];\n}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, const void* src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_u32(src))
               : "memory");
}

// Two fp32 operations at once.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ float2 both(uint64_t p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// silu_product and linear_value of two channels.
__device__ __forceinline__ uint64_t silu2(uint64_t g, uint64_t u) {
  const float2 e = both(mul2(g, pair2(kMinusLog2e, kMinusLog2e)));
  const float2 d = both(add2(pair2(exp2_fast(e.x), exp2_fast(e.y)), pair2(1.0f, 1.0f)));
  return mul2(mul2(g, pair2(rcp_fast(d.x), rcp_fast(d.y))), u);
}
__device__ __forceinline__ uint64_t linear2(uint32_t a0, uint32_t a1, uint64_t xs, uint64_t ws, uint64_t bias) {
  return fma2(mul2(pair2(static_cast<float>(static_cast<int>(a0)), static_cast<float>(static_cast<int>(a1))), xs), ws, bias);
}

// 32 accumulator columns of this thread's TMEM lane on their way; tmem_arrived ends the wait for all such loads.
__device__ __forceinline__ void tmem_start32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_start16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_arrived(uint32_t (&r)[32]) {  // (the operands keep uses behind the wait)
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

struct __align__(64) Params {
  CUtensorMap tx;  // codes [m, k], box 128 x (tokens of a CTA)
  CUtensorMap tw;  // weight codes [n or 2n, k], box 128 x (weight rows of a CTA's load)
  CUtensorMap ty;  // pair_kernel, aligned rows: y [m, n] fp16, box (64 or 32) x 32, swizzled by its row length
  CUtensorMap tr;  // residual, the same
  Args a;
  int tma_y;    // y goes out, and the residual comes in, by TMA (ty and tr are set)
  int xrows;    // split_kernel: tokens, rounded up to 16
  int stages;   // split_kernel: K steps in flight
  int ksteps;   // split_kernel: K steps of each CTA of a cluster
  int tiles_n, tiles;  // pair_kernel: tiles along n, all tiles
  int* error;
};

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

// Bounded wait for a barrier that other CTAs of the cluster report to.
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
// The wait of a whole warp (one that runs out does so for all of its lanes).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, abort_flag));
}
// (relaxed: what it reports, loads out of tensor memory, is complete; a release took 1000 cycles of the epilogue)
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// --- split_kernel -------------------------------------------------------------
// One tile of 128 weight rows (gated: 64 gate and their 64 up rows) and all
// tokens (up to 128, in 16s) a cluster; CTA z of the cluster multiplies K steps z * ksteps .. .
//   warp 0 lane 0: TMA loads; warp 1 lane 0: MMAs; warps 2-17: sums out of
//   TMEM, 32 tokens of 32 rows each; all warps: finish the CTA's rows.
// Each CTA finishes 128 / splits of the tile's rows: all CTAs store their sums
// of these rows into its shared memory ([tokens / 4][split][row][4], so that a
// warp's stores and loads are contiguous), counted in bytes by its barrier.
// Latency: 64 x 1536 x 8960 6.7 us, of it start and barriers 1, loads 2.5 (some
// 50 B a clock and SM), the sums' exchange 1.2 (25 B a clock), the rest 1.
constexpr int kSplitThreads = 64 + 512;
constexpr int kSplitStages = 8;   // at most
constexpr int kSplitTokens = 128;  // of a tile at most
constexpr int kWBytes = 128 * kBK;

// 16 bytes into the shared memory of a CTA of the cluster, reported to a barrier there.
__device__ __forceinline__ void store_cluster(uint32_t to, const uint32_t* v, uint32_t bar) {
  asm volatile(
      "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(bar)
      : "memory");
}

template <bool GATED>
__global__ void __launch_bounds__(kSplitThreads, 2) split_kernel(const __grid_constant__ Params P) {
  extern __shared__ unsigned char smem_raw[];
  const Args& A = P.a;
  const int S = P.stages, xbytes = P.xrows * kBK;
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* wt = base;
  unsigned char* xt = base + static_cast<size_t>(S) * kWBytes;
  int4* red = reinterpret_cast<int4*>(xt + static_cast<size_t>(S) * xbytes);
  float* xs = reinterpret_cast<float*>(red + 32 * P.xrows);  // [kSplitTokens] token scales
  float* cs = xs + kSplitTokens;                             // [3][128] channel scales, up scales, biases
  uint64_t* full = reinterpret_cast<uint64_t*>(cs + 3 * 128);
  uint64_t* empty = full + kSplitStages;
  uint64_t* done = empty + kSplitStages;
  uint64_t* sums = done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sums + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* abort_v = abort_flag;
  constexpr int kOut = GATED ? 64 : 128;  // channels of a tile

  lmps_pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int c0 = blockIdx.x * kOut;
  const int splits = gridDim.z;
  const int all = (A.k + kBK - 1) / kBK, kbeg = blockIdx.z * P.ksteps;
  const int ksteps = max(0, min(P.ksteps, all - kbeg));
  const uint32_t tcols = P.xrows <= 32 ? 32u : P.xrows <= 64 ? 64u : 128u;
  const uint32_t rank = cluster_rank();  // = blockIdx.z

  if (warp == 0) {  // a lane per barrier
    if (lane < S) {
      mbar_init(&full[lane], 1);
      mbar_init(&empty[lane], 1);
    } else if (lane == 30) {
      mbar_init(done, 1);
      *abort_flag = 0;
    } else if (lane == 31) {
      mbar_init(sums, 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (lane == 31) mbar_expect_tx(sums, static_cast<uint32_t>(128 * P.xrows * 4));
    __syncwarp();
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
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // (the barriers exist; waited for before the sums go out)
  const uint32_t tmem = *tmem_slot;
  const int rows = 128 / splits, outs = kOut / splits;  // sums and channels that this CTA finishes
  const int cbase = c0 + static_cast<int>(rank) * outs;
  const int log_outs = __ffs(outs) - 1;

  if (warp == 0) {
    if (lane == 0) {
      lmps_pdl_wait();  // both operands may be the previous kernel's output
      Ring r;
      int issued = 0;
      for (int kt = 0; kt < ksteps; ++kt, r.next(S)) {
        if (kt >= S && !mbar_wait(&empty[r.slot], r.phase ^ 1u, P.error, abort_v)) break;
        mbar_expect_tx(&full[r.slot], static_cast<uint32_t>(kWBytes + xbytes));
        unsigned char* w = wt + static_cast<size_t>(r.slot) * kWBytes;
        const int kx = (kbeg + kt) * kBK;
        tma_load_2d(w, &P.tw, kx, c0, &full[r.slot]);
        if (GATED) tma_load_2d(w + kWBytes / 2, &P.tw, kx, A.n + c0, &full[r.slot]);
        tma_load_2d(xt + static_cast<size_t>(r.slot) * xbytes, &P.tx, kx, 0, &full[r.slot]);
        issued = kt + 1;
      }
      for (int kt = max(0, issued - S); kt < issued; ++kt) {  // every issued copy lands before the CTA leaves
        const uint64_t since = globaltimer();
        while (!mbar_try(&full[kt % S], (kt / S) & 1))
          if (globaltimer() - since > kTimeoutNs) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
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
          mma_i8<1>(tmem, wd + 2 * j, xd + 2 * j, idesc, (kt > 0 || j > 0) ? 1u : 0u, 1u);
        mma_commit(&empty[r.slot]);
      }
      mma_commit(done);
      const uint64_t since = globaltimer();  // every MMA is finished before the tensor memory is freed
      while (!mbar_try(done, 0u))
        if (globaltimer() - since > kTimeoutNs) break;
    }
  } else {
    if (warp == 2)
      for (int kt = lane; kt < ksteps; kt += 32) {  // the weights come nearer while the kernel before ends
        prefetch_2d(&P.tw, (kbeg + kt) * kBK, c0);
        if (GATED) prefetch_2d(&P.tw, (kbeg + kt) * kBK, A.n + c0);
      }
    lmps_pdl_wait();  // before any read of scales and residual, or write of y
    // what the sums meet, on its way before they do
    if (const int i = tid - 64 - 128; i >= 0 && i < P.xrows) xs[i] = i < A.m ? A.xs[i] : 0.0f;
    if (const int i = tid - 64 - 256; i >= 0 && i < outs) {
      const bool in = cbase + i < A.n;
      cs[i] = in ? A.ws[cbase + i] : 0.0f;
      if (GATED) cs[128 + i] = in ? A.ws[A.n + cbase + i] : 0.0f;
      cs[256 + i] = in && A.bias ? __half2float(A.bias[cbase + i]) : 0.0f;
    }
  }
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp >= 2) {
    // (a wait that ran out leaves the sums without meaning; they still go out, so that no CTA waits for them)
    const bool ok = warp_wait(done, 0u, P.error, abort_v) && ksteps > 0;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const int q = warp & 3, row = 32 * q + lane;  // TMEM lane = row of the tile
    const int c = row % kOut, owner = c >> log_outs, local = (GATED ? row / 64 * outs : 0) + (c & (outs - 1));
    if (const int j0 = 32 * ((warp - 2) / 4); j0 < P.xrows) {
      uint32_t v[32];
      if (ok) {
        tmem_ld32(tmem + (static_cast<uint32_t>(32 * q) << 16) + j0, v);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = 0u;
      }
      const uint32_t bar = cluster_addr(sums, static_cast<uint32_t>(owner));
      const uint32_t to = cluster_addr(red + j0 / 4 * 128 + static_cast<int>(rank) * rows + local, static_cast<uint32_t>(owner));
#pragma unroll
      for (int j = 0; j < 32; j += 4)
        if (j0 + j < P.xrows) store_cluster(to + j / 4 * 128 * 16, v + j, bar);
    }
  }
  lmps_pdl_wait();
  const int tok = A.m, tok4 = (tok + 3) / 4;
  const bool here = __syncthreads_and(tid != 0 || mbar_wait_cluster(sums, 0u, P.error, abort_v));
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  for (int i = tid; here && i < outs * tok4; i += kSplitThreads) {
    const int lc = i & (outs - 1), j = 4 * (i >> log_outs), c = cbase + lc;
    if (c >= A.n) continue;
    float res[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      res[e] = !GATED && A.residual && j + e < tok ? __half2float(A.residual[static_cast<size_t>(j + e) * A.ldr + c]) : kNone;
    int g[4] = {0, 0, 0, 0}, u[4] = {0, 0, 0, 0};
    const int4* at = red + j / 4 * 128 + lc;
#pragma unroll 4
    for (int z = 0; z < splits; ++z, at += rows) {
      const int4 v = at[0];
      g[0] += v.x, g[1] += v.y, g[2] += v.z, g[3] += v.w;
      if (GATED) {
        const int4 b = at[outs];
        u[0] += b.x, u[1] += b.y, u[2] += b.z, u[3] += b.w;
      }
    }
    const float ws = cs[lc], bias = GATED ? 0.0f : cs[256 + lc], wu = GATED ? cs[128 + lc] : 0.0f;
    const float4 x4 = *reinterpret_cast<const float4*>(xs + j);
    const float xv[4] = {x4.x, x4.y, x4.z, x4.w};
    __half* y = A.y + static_cast<size_t>(j) * A.ldy + c;
#pragma unroll
    for (int e = 0; e < 4; ++e, y += A.ldy) {
      float v = linear_value(g[e], xv[e], ws, bias);
      if (GATED) v = silu_product(v, linear_value(u[e], xv[e], wu));
      if (j + e < tok) *y = __float2half_rn(v + res[e]);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // no CTA leaves while another waits for sums
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tcols) : "memory");
}

// --- whole_kernel -------------------------------------------------------------
// Up to 128 tokens and tiles enough for the GPU (no residual): a CTA multiplies
// the whole of K for 128 weight rows (gated: 64 gate and their 64 up rows).  The tokens are
// the MMA's 128 rows (those past the last hold what the ring held before, and
// their sums are not read), so a TMEM lane has a token's gates in columns 0 ..
// and their up values 64 further: nothing is exchanged, and a lane writes its
// token's 16 or 32 channels side by side.
//   warp 0: TMA loads; warp 1: MMAs; warps 2-17: epilogue, four for each 32
//   tokens (those without tokens rest).
// Bound by what an SM loads, some 50 B a clock: 64 x 8960 x 1536 gated 6.5 us
// out of L2 (288 KB a CTA: 3.3 us), 9.4 out of DRAM.
constexpr int kWholeThreads = 64 + 512;
constexpr int kWholeStages = 6;  // at most
constexpr int kXSlot = 128 * kBK;

template <bool GATED>
__global__ void __launch_bounds__(kWholeThreads) whole_kernel(const __grid_constant__ Params P) {
  extern __shared__ unsigned char smem_raw[];
  const Args& A = P.a;
  const int S = P.stages;
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* cs = reinterpret_cast<float*>(base + static_cast<size_t>(S) * (kWBytes + kXSlot));  // [128] scales, [128] biases
  uint64_t* full = reinterpret_cast<uint64_t*>(cs + 2 * 128);
  uint64_t* empty = full + kWholeStages;
  uint64_t* done = empty + kWholeStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* abort_v = abort_flag;
  constexpr int kOut = GATED ? 64 : 128, kMine = kOut / 4;  // channels of a tile, of an epilogue warp

  lmps_pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int c0 = blockIdx.x * kOut, ksteps = (A.k + kBK - 1) / kBK;
  if (warp == 0) {  // a lane per barrier
    if (lane < S) {
      mbar_init(&full[lane], 1);
      mbar_init(&empty[lane], 1);
    } else if (lane == 31) {
      mbar_init(done, 1);
      *abort_flag = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 128;" ::"r"(smem_u32(tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      lmps_pdl_wait();  // both operands may be the previous kernel's output
      Ring r;
      int issued = 0;
      for (int kt = 0; kt < ksteps; ++kt, r.next(S)) {
        if (kt >= S && !mbar_wait(&empty[r.slot], r.phase ^ 1u, P.error, abort_v)) break;
        mbar_expect_tx(&full[r.slot], static_cast<uint32_t>(kWBytes + P.xrows * kBK));
        unsigned char* w = base + static_cast<size_t>(r.slot) * (kWBytes + kXSlot);
        tma_load_2d(w, &P.tw, kt * kBK, c0, &full[r.slot]);
        if (GATED) tma_load_2d(w + kWBytes / 2, &P.tw, kt * kBK, A.n + c0, &full[r.slot]);
        tma_load_2d(w + kWBytes, &P.tx, kt * kBK, 0, &full[r.slot]);
        issued = kt + 1;
      }
      for (int kt = max(0, issued - S); kt < issued; ++kt) {  // every issued copy lands before the CTA leaves
        const uint64_t since = globaltimer();
        while (!mbar_try(&full[kt % S], (kt / S) & 1))
          if (globaltimer() - since > kTimeoutNs) break;
      }
    }
  } else if (warp == 1) {
    lmps_pdl_wait();  // (bounded waits begin when the work does)
    const uint32_t lead = lane == 0 ? 1u : 0u;
    const uint64_t wd0 = sw128_desc(smem_u32(base)), xd0 = sw128_desc(smem_u32(base) + kWBytes);
    Ring r;
    for (int kt = 0; kt < ksteps; ++kt, r.next(S)) {
      if (!warp_wait(&full[r.slot], r.phase, P.error, abort_v)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t at = static_cast<uint64_t>(r.slot) * ((kWBytes + kXSlot) >> 4);
#pragma unroll
      for (int j = 0; j < kBK / 32; ++j)
        mma_i8<1>(tmem, xd0 + at + 2 * j, wd0 + at + 2 * j, idesc_i8(128, 128), (kt > 0 || j > 0) ? 1u : 0u, lead);
      if (lane == 0) mma_commit(&empty[r.slot]);
    }
    if (lane == 0) {
      mma_commit(done);
      const uint64_t since = globaltimer();  // every MMA is finished before the tensor memory is freed
      while (!mbar_try(done, 0u))
        if (globaltimer() - since > kTimeoutNs) break;
    }
  } else {
    if (warp == 17)
      for (int kt = lane; kt < ksteps; kt += 32) {  // the weights come nearer while the kernel before ends
        prefetch_2d(&P.tw, kt * kBK, c0);
        if (GATED) prefetch_2d(&P.tw, kt * kBK, A.n + c0);
      }
    lmps_pdl_wait();  // before any read of scales, or write of y
    const int q = warp & 3, first = (warp - 2) / 4 * kMine, token = 32 * q + lane;
    const bool live = token < A.m;
    if (const int i = tid - 64; i < kOut) {
      const bool in = c0 + i < A.n;
      cs[i] = in ? A.ws[c0 + i] : 0.0f;
      cs[128 + i] = !in ? 0.0f : GATED ? A.ws[A.n + c0 + i] : A.bias ? __half2float(A.bias[c0 + i]) : 0.0f;
    }
    const float xs = live ? A.xs[token] : 0.0f;
    asm volatile("bar.sync 1, 512;" ::: "memory");
    if (32 * q < A.m && warp_wait(done, 0u, P.error, abort_v)) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t tl = tmem + (static_cast<uint32_t>(32 * q) << 16) + first;
      uint32_t g[32];  // gated: 16 gates, 16 up values
      if (GATED) {
        tmem_start16(tl, g);
        tmem_start16(tl + kOut, g + 16);
      } else {
        tmem_start32(tl, g);
      }
      tmem_arrived(g);
      const uint64_t xs2 = pair2(xs, xs);
      const uint64_t* w2 = reinterpret_cast<const uint64_t*>(cs + first);
      const uint64_t* b2 = reinterpret_cast<const uint64_t*>(cs + 128 + first);
      __half* y = A.y + static_cast<size_t>(token) * A.ldy + c0 + first;
#pragma unroll
      for (int j = 0; j < kMine; j += 8) {
        float v[8];
#pragma unroll
        for (int l = 0; l < 8; l += 2) {
          uint64_t r = linear2(g[j + l], g[j + l + 1], xs2, w2[(j + l) / 2], GATED ? 0ull : b2[(j + l) / 2]);
          if (GATED) r = silu2(r, linear2(g[16 + j + l], g[16 + j + l + 1], xs2, b2[(j + l) / 2], 0ull));
          const float2 f = both(r);
          v[l] = f.x, v[l + 1] = f.y;
        }
        const int left = live ? A.n - (c0 + first + j) : 0;
        if (left >= 8) {  // (rows of y start at multiples of 16 bytes)
          uint4 packed;
          __half2* h2 = reinterpret_cast<__half2*>(&packed);
#pragma unroll
          for (int l = 0; l < 4; ++l) h2[l] = __floats2half2_rn(v[2 * l], v[2 * l + 1]);
          *reinterpret_cast<uint4*>(y + j) = packed;
        } else {
#pragma unroll
          for (int l = 0; l < 8; ++l)
            if (l < left) y[j + l] = __float2half_rn(v[l]);
        }
      }
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 128;" ::"r"(tmem) : "memory");
}

static size_t whole_smem(int stages) {
  return static_cast<size_t>(stages) * (kWBytes + kXSlot) + 2 * 128 * sizeof(float) + 1024 +
         (2 * kWholeStages + 1) * sizeof(uint64_t) + 16;
}

static size_t split_smem(int stages, int xrows) {
  return static_cast<size_t>(stages) * (kWBytes + xrows * kBK) + static_cast<size_t>(xrows) * 512 +
         (kSplitTokens + 3 * 128) * sizeof(float) + 1024 + (2 * kSplitStages + 2) * sizeof(uint64_t) + 16;
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
//   warps 2 ..: epilogue, four warps (TMEM lanes 32 (w % 4) ..) for each 64 or 32 channels of the tile
// Tiles of 256 x 256 because a pair then loads 64 KB for 512 cycles of products
// of both SMs, near what they can load (10 TB/s over the GPU); of 128 where
// there are few.  Bound by power, so by the codes too: 16384 x 8960 x 1536 gated
// 350 to 358 us of bell-shaped codes up to 127 (2.5 POP/s at some 1.4 GHz; 258
// without the epilogue, 222 of zeros; 300 of even codes up to 34), 16384 x 1536 x
// 8960 with residual 190 (166 of the latter).
// Split K (SPLITS > 1): the pairs of a cluster send their sums of a warp's
// channels to the pair that finishes them.

template <int BN, bool GATED, int SPLITS = 1>
struct PairShape {
  static constexpr int kX = 128 * kBK, kW = BN / 2 * kBK;
  static constexpr int kStage = kX + kW;
  static constexpr int kOut = GATED ? BN / 2 : BN;     // channels of a tile
  static constexpr int kParts = kOut >= 128 ? 4 : 2;   // epilogue warps side by side
  static constexpr int kWarps = 4 * kParts;
  static constexpr int kThreads = 64 + kWarps * kWarp;
  static constexpr int kMine = kOut / kParts;          // channels of an epilogue warp: a store of 32 rows
  static constexpr int kBoxBytes = 32 * kMine * 2;
  static constexpr int kStore = kWarps * kBoxBytes;
  static constexpr int kCols = kWarps * 2 * kMine * 4;  // a warp's scales and biases (gated: gate and up scales)
  // split K: sums from the other pairs, [pair][warp][tokens 32 x channels kMine]
  static constexpr int kSums = (SPLITS - 1) * (kWarps / SPLITS) * 32 * kMine * 4;
  static constexpr int kStages = (208 * 1024 - kStore - kCols - kSums) / kStage;  // 4 (gated 5) of 32 KB, 7 of 24 KB
  static constexpr int kBars = 2 * kStages + 6 + kWarps;
  static constexpr size_t kSmem =
      static_cast<size_t>(kStages) * kStage + kSums + kStore + kCols + 1024 + kBars * sizeof(uint64_t) + 16;
};

template <int BN, bool GATED, int SPLITS>
__global__ void __launch_bounds__(PairShape<BN, GATED, SPLITS>::kThreads, 1)
    pair_kernel(const __grid_constant__ Params P) {
  static_assert(SPLITS == 1 || !GATED, "a gated tile is not split");
  using Sh = PairShape<BN, GATED, SPLITS>;
  constexpr int S = Sh::kStages, kOut = Sh::kOut;
  constexpr uint32_t kTmem = BN > 128 ? 512u : 256u;
  constexpr uint32_t kAcc = kTmem / 2;  // columns from one accumulator to the other
  extern __shared__ unsigned char smem_raw[];
  const Args& A = P.a;
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* stage = base;  // [S] codes tile, weight tile
  int4* sums = reinterpret_cast<int4*>(base + static_cast<size_t>(S) * Sh::kStage);  // (SPLITS > 1)
  unsigned char* store = base + static_cast<size_t>(S) * Sh::kStage + Sh::kSums;
  float* cols = reinterpret_cast<float*>(store + Sh::kStore);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<unsigned char*>(cols) + Sh::kCols);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;   // [2] accumulator complete
  uint64_t* tempty = tfull + 2;  // [2] accumulator read by both CTAs' epilogues (the first CTA's counts)
  uint64_t* done = tempty + 2;
  uint64_t* rfull = done + 1;  // [epilogue warps] residual box arrived
  uint64_t* arrived = rfull + Sh::kWarps;  // the other pairs' sums
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(arrived + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* abort_v = abort_flag;

  lmps_pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // split K: pair `split` of a cluster of SPLITS multiplies its share of the K steps of the cluster's one tile
  const uint32_t crank = cluster_rank(), rank = crank & 1u, first_cta = crank & ~1u;
  const int split = static_cast<int>(crank >> 1), steps = (A.k + kBK - 1) / kBK;
  const int kbeg = steps * split / SPLITS, ksteps = steps * (split + 1) / SPLITS - kbeg;
  const int pair = static_cast<int>(blockIdx.x) / (2 * SPLITS), pairs = static_cast<int>(gridDim.x) / (2 * SPLITS);
  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 2 * Sh::kWarps);
    }
    mbar_init(done, 1);
    for (int i = 0; i < Sh::kWarps; ++i) mbar_init(&rfull[i], 1);
    mbar_init(arrived, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (SPLITS > 1) mbar_expect_tx(arrived, Sh::kSums);
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
    lmps_pdl_wait();  // both operands may be the previous kernel's output
    const uint32_t lead = lane == 0 ? 1u : 0u, x0 = smem_u32(stage), bar0 = cluster_addr(full, first_cta);
    Ring r;
    int issued = 0;
    bool ok = true;
    for (int tile = pair; ok && tile < P.tiles; tile += pairs) {
      const int c0 = (tile % P.tiles_n) * kOut, t0 = (tile / P.tiles_n) * 256 + static_cast<int>(rank) * 128;
      const int w0 = GATED ? static_cast<int>(rank) * A.n + c0 : c0 + static_cast<int>(rank) * (BN / 2);
      for (int kt = 0; kt < ksteps; ++kt, r.next(S)) {
        if (issued >= S && !warp_wait(&empty[r.slot], r.phase ^ 1u, P.error, abort_v)) {
          ok = false;
          break;
        }
        // the first CTA's barrier counts the bytes of both
        if (rank == 0 && lane == 0) mbar_expect_tx(&full[r.slot], 2u * Sh::kStage);
        const uint32_t x = x0 + static_cast<uint32_t>(r.slot) * Sh::kStage, bar = bar0 + 8u * static_cast<uint32_t>(r.slot);
        tma_load_pair(x, &P.tx, (kbeg + kt) * kBK, t0, bar, lead);
        tma_load_pair(x + Sh::kX, &P.tw, (kbeg + kt) * kBK, w0, bar, lead);
        ++issued;
      }
    }
    // every copy has landed and every release of a stage has reached this CTA before it leaves
    for (int g = max(0, issued - S); lane == 0 && g < issued; ++g) {
      const uint64_t since = globaltimer();
      while (!mbar_try(&empty[g % S], (g / S) & 1))
        if (globaltimer() - since > kTimeoutNs) break;
    }
  } else if (warp == 1) {
    if (rank == 0) {
      lmps_pdl_wait();  // (bounded waits begin when the work does)
      constexpr uint32_t idesc = idesc_i8(256, BN);
      const uint32_t lead = lane == 0 ? 1u : 0u;
      const uint64_t xd0 = sw128_desc(smem_u32(stage)), wd0 = sw128_desc(smem_u32(stage) + Sh::kX);
      Ring r;
      uint32_t uses[2] = {0u, 0u};
      int buf = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < P.tiles; tile += pairs, buf ^= 1) {
        if (!__all_sync(0xffffffffu, mbar_wait_cluster(&tempty[buf], (uses[buf] & 1u) ^ 1u, P.error, abort_v))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t acc = tmem + static_cast<uint32_t>(buf) * kAcc;
        for (int kt = 0; kt < ksteps; ++kt, r.next(S)) {
          if (!warp_wait(&full[r.slot], r.phase, P.error, abort_v)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t at = static_cast<uint64_t>(r.slot) * (Sh::kStage >> 4);
#pragma unroll
          for (int j = 0; j < kBK / 32; ++j)
            mma_i8<2>(acc, xd0 + at + 2 * j, wd0 + at + 2 * j, idesc, (kt > 0 || j > 0) ? 1u : 0u, lead);
          commit_pair(&empty[r.slot], first_cta, lead);
        }
        if (!ok) break;
        commit_pair(&tfull[buf], first_cta, lead);
        ++uses[buf];
      }
      commit_pair(done, first_cta, lead);
    }
  } else {
    lmps_pdl_wait();  // before any read of scales and residual, or write of y
    constexpr int kMine = Sh::kMine, kChunks = kMine / 32;
    const int e = warp - 2, q = warp & 3, first = e / 4 * kMine;  // TMEM lanes 32 q .., channels first ..
    unsigned char* box = store + e * Sh::kBoxBytes;  // [32 rows][kMine] fp16, swizzled as the TMA unit does
    float* ws = cols + e * (2 * kMine);
    float* bs = ws + kMine;
    // byte of the box at which the 16-byte piece i of row r lies
    auto piece = [&](int r, int i) { return r * (kMine * 2) + ((kMine == 64 ? i ^ (r & 7) : i ^ ((r >> 1) & 3)) << 4); };
    auto element = [&](int r, int j) { return reinterpret_cast<__half*>(box + piece(r, j / 8) + (j % 8) * 2); };
    // Rows of any alignment, between memory and the box: kBatch rows of elements a lane loads before it stores any.
    constexpr int kLane = kMine / 32, kBatch = 16 / kLane;
    auto rows_batch = [&](auto whole, int r0, int t0, int c0, auto&& load, auto&& put) {
      auto in = [&](int i, int l) { return whole() || (t0 + r0 + i < A.m && c0 + lane + 32 * l < A.n); };
      __half v[kBatch][kLane];
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
#pragma unroll
        for (int l = 0; l < kLane; ++l) v[i][l] = in(i, l) ? load(r0 + i, lane + 32 * l) : __half(0.0f);
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
#pragma unroll
        for (int l = 0; l < kLane; ++l)
          if (in(i, l)) put(r0 + i, lane + 32 * l, v[i][l]);
    };
    auto rows_any = [&](int t0, int c0, auto&& load, auto&& put) {
#pragma unroll 1
      for (int r0 = 0; r0 < 32; r0 += kBatch) {
        if (t0 + 32 <= A.m && c0 + kMine <= A.n) rows_batch(std::true_type{}, r0, t0, c0, load, put);
        else rows_batch(std::false_type{}, r0, t0, c0, load, put);
      }
    };
    // scales (and biases) of this warp's channels and this lane's token, on their way for the next tile
    float nxs = 0.0f, nws[kChunks], nus[kChunks];
    __half nbs[kChunks];
    auto fetch = [&](int tile) {
      const int c0 = (tile % P.tiles_n) * kOut + first;
      const int row = (tile / P.tiles_n) * 256 + static_cast<int>(rank) * 128 + 32 * q + lane;
      nxs = row < A.m ? A.xs[row] : 0.0f;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int c = c0 + 32 * i + lane;
        const bool in = c < A.n;
        nws[i] = in ? A.ws[c] : 0.0f;
        if (GATED) nus[i] = in ? A.ws[A.n + c] : 0.0f;
        else nbs[i] = in && A.bias ? A.bias[c] : __half(0.0f);
      }
    };
    if (pair < P.tiles) fetch(pair);
    // split K: the pair that finishes this warp's channels, and its place among the warps there
    const int owner = e / 4 * SPLITS / Sh::kParts, place = e - owner * (Sh::kWarps / SPLITS);
    const bool extra = GATED || A.bias != nullptr;  // (bs holds something)
    const bool add = !GATED && A.residual != nullptr && (SPLITS == 1 || owner == split);
    uint32_t uses[2] = {0u, 0u}, rphase = 0u;
    bool awaited = false;  // a residual is on its way
    int buf = 0;
    for (int tile = pair; tile < P.tiles; tile += pairs, buf ^= 1) {
      const int c0 = (tile % P.tiles_n) * kOut + first;
      const int t0 = (tile / P.tiles_n) * 256 + static_cast<int>(rank) * 128 + 32 * q;
      const uint64_t xs2 = pair2(nxs, nxs);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        ws[32 * i + lane] = nws[i];
        bs[32 * i + lane] = GATED ? nus[i] : __half2float(nbs[i]);
      }
      if (tile + pairs < P.tiles) fetch(tile + pairs);
      // the box is free once the last tile's store has read it; the residual comes in where the sums go out
      if (lane == 0) {
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        if (add && P.tma_y) {
          mbar_expect_tx(&rfull[e], Sh::kBoxBytes);
          tma_load_2d(box, &P.tr, c0, t0, &rfull[e]);
        }
      }
      __syncwarp();
      if (add && P.tma_y) {
        awaited = true;
      } else if (add) {  // rows of any alignment: a row a time
        const __half* p = A.residual + static_cast<size_t>(t0) * A.ldr + c0;
        rows_any(t0, c0, [&](int r, int j) { return p[static_cast<size_t>(r) * A.ldr + j]; },
                 [&](int r, int j, __half v) { *element(r, j) = v; });
        __syncwarp();
      }
      if (!warp_wait(&tfull[buf], uses[buf] & 1u, P.error, abort_v)) break;
      ++uses[buf];
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t tl = tmem + static_cast<uint32_t>(buf) * kAcc + (static_cast<uint32_t>(32 * q) << 16) + first;
      uint32_t g[kChunks][32], u[kChunks][32];  // (u: gated)
      tmem_start32(tl, g[0]);
      if (GATED) tmem_start32(tl + kOut, u[0]);
      if constexpr (SPLITS > 1) {
        static_assert(kChunks == 1, "a warp's sums are 32 registers");
        // [pair][warp][channel / 4][lane]: a warp's stores and loads are contiguous
        const int at = place * 8 * 32 + lane, block = Sh::kWarps / SPLITS * 8 * 32;
        tmem_arrived(g[0]);
        if (owner != split) {
          const uint32_t cta = 2u * static_cast<uint32_t>(owner) + rank;
          const uint32_t to = cluster_addr(sums + (split < owner ? split : split - 1) * block + at, cta);
          const uint32_t bar = cluster_addr(arrived, cta);
#pragma unroll
          for (int j = 0; j < 8; ++j) store_cluster(to + static_cast<uint32_t>(j * 32 * 16), &g[0][4 * j], bar);
          break;
        }
        if (!__all_sync(0xffffffffu, mbar_wait_cluster(arrived, 0u, P.error, abort_v))) break;
#pragma unroll
        for (int z = 0; z < SPLITS - 1; ++z)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int4 v = sums[z * block + at + j * 32];
            g[0][4 * j] += v.x, g[0][4 * j + 1] += v.y, g[0][4 * j + 2] += v.z, g[0][4 * j + 3] += v.w;
          }
      }
      if (awaited) {
        if (!warp_wait(&rfull[e], rphase, P.error, abort_v)) break;
        rphase ^= 1u;
        awaited = false;
      }
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {  // 32 channels; the next ones are on their way meanwhile
        tmem_arrived(g[i]);
        if (GATED) tmem_arrived(u[i]);
        if (i + 1 < kChunks) {
          tmem_start32(tl + 32 * (i + 1), g[i + 1]);
          if (GATED) tmem_start32(tl + kOut + 32 * (i + 1), u[i + 1]);
        } else {  // the accumulator is read
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) arrive_cluster(cluster_addr(&tempty[buf], first_cta));
        }
        const ulonglong2* w4 = reinterpret_cast<const ulonglong2*>(ws + 32 * i);
        const ulonglong2* b4 = reinterpret_cast<const ulonglong2*>(bs + 32 * i);
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          float v[8];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const ulonglong2 w = w4[j / 4 + h], o = extra ? b4[j / 4 + h] : make_ulonglong2(0ull, 0ull);
#pragma unroll
            for (int l = 0; l < 2; ++l) {
              const int k = j + 4 * h + 2 * l;
              const uint64_t wl = l ? w.y : w.x, ol = l ? o.y : o.x;
              uint64_t r = linear2(g[i][k], g[i][k + 1], xs2, wl, GATED ? 0ull : ol);
              if (GATED) r = silu2(r, linear2(u[i][k], u[i][k + 1], xs2, ol, 0ull));
              const float2 f = both(r);
              v[4 * h + 2 * l] = f.x, v[4 * h + 2 * l + 1] = f.y;
            }
          }
          uint4* to = reinterpret_cast<uint4*>(box + piece(lane, (32 * i + j) / 8));
          if (add) {
            const uint4 rv = *to;
            const __half2* r2 = reinterpret_cast<const __half2*>(&rv);
#pragma unroll
            for (int l = 0; l < 4; ++l) {
              const float2 f = __half22float2(r2[l]);
              v[2 * l] += f.x, v[2 * l + 1] += f.y;
            }
          }
          uint4 packed;
          __half2* h2 = reinterpret_cast<__half2*>(&packed);
#pragma unroll
          for (int l = 0; l < 4; ++l) h2[l] = __floats2half2_rn(v[2 * l], v[2 * l + 1]);
          *to = packed;
        }
      }
      if (P.tma_y) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0 && c0 < A.n && t0 < A.m) {
          tma_store_2d(&P.ty, c0, t0, box);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      } else {
        __syncwarp();
        __half* p = A.y + static_cast<size_t>(t0) * A.ldy + c0;
        rows_any(t0, c0, [&](int r, int j) { return *element(r, j); },
                 [&](int r, int j, __half v) { p[static_cast<size_t>(r) * A.ldy + j] = v; });
      }
    }
    if (lane == 0) {
      // (after a wait that ran out: a residual on its way lands before the CTA leaves)
      const uint64_t since = globaltimer();
      while (awaited && !mbar_try(&rfull[e], rphase))
        if (globaltimer() - since > kTimeoutNs) break;
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
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

// Whether rows of fp16 start at multiples of 16 bytes.
static bool rows16(const __half* p, size_t ld) { return ld % 8 == 0 && lmps_aligned(p, 16); }

// A launch of clusters that may begin while its predecessor ends.
static int launch_clusters(void (*kernel)(Params), dim3 grid, int threads, size_t smem, dim3 cluster, cudaStream_t st,
                           const Params& P) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster.x;
  at[0].val.clusterDim.y = cluster.y;
  at[0].val.clusterDim.z = cluster.z;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P);
  return e == cudaSuccess ? lmps_launch_status() : static_cast<int>(e);
}

static bool encode_codes(CUtensorMap* map, const int8_t* p, int k, size_t rows, size_t ld, int box_rows) {
  return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, p, static_cast<uint64_t>(k), rows, ld, kBK,
                   static_cast<uint32_t>(box_rows), CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int NT, bool GATED, int WARPS>
static int launch_few_warps(const Args& A, int tiles, cudaStream_t st) {
  return lmps_launch_pdl(few_kernel<NT, GATED, WARPS>, dim3(tiles), dim3(WARPS * kWarp), 0, st, A);
}
// The fewer tiles there are for an SM, the more warps share one out (as their sums fit 48 KB of shared memory).
template <int NT, bool GATED>
static int launch_few(const Args& A, int sms, cudaStream_t st) {
  constexpr int kFit = 64 / (NT * (GATED ? 2 : 1));
  const int tiles = (A.n + 15) / 16;
  if constexpr (kFit >= 32)
    if (tiles <= sms) return launch_few_warps<NT, GATED, 32>(A, tiles, st);
  if constexpr (NT != 2) {
    if constexpr (kFit >= 16)
      if (tiles <= 2 * sms) return launch_few_warps<NT, GATED, 16>(A, tiles, st);
    return launch_few_warps<NT, GATED, 8>(A, tiles, st);
  } else {  // (two token tiles: never more tiles than SMs)
    return launch_few_warps<NT, GATED, GATED ? 16 : 32>(A, tiles, st);
  }
}

template <bool GATED>
static int launch_split(const Args& A, int* error, int sms, cudaStream_t st) {
  Params P{};
  P.a = A;
  P.error = error;
  P.xrows = (A.m + 15) / 16 * 16;
  const int out = GATED ? 64 : 128;
  const int tiles = (A.n + out - 1) / out, steps = (A.k + kBK - 1) / kBK;
  // no more CTAs than two an SM, at least three K steps each (64 x 2048 x 1536: 5.6 us with 4 splits, 5.9 with 8, 7.5
  // with 2).  This counts CTAs, not the clusters that fit: with an SM a CTA a device holds some 15 clusters of eight, so
  // 16 to 18 tiles behind a long K take a second wave (64 x 2048 x 8192 16.7 us; 12 tiles, 64 x 1536 x 8960, 6.6).
  int splits = 1;
  while (splits < 8 && 2 * splits * tiles <= 2 * sms && 6 * splits <= steps) splits *= 2;
  P.ksteps = (steps + splits - 1) / splits;
  // half an SM's shared memory where there are more CTAs than SMs, else all of it.  Past 96 tokens two stages and the
  // sums alone are more than half, so such CTAs run one an SM, in two waves (128 x 2560 x 9728 24.9 us).
  const size_t room = tiles * splits > sms ? 113 * 1024 : 226 * 1024;
  int stages = P.ksteps < 2 ? 2 : P.ksteps < kSplitStages ? P.ksteps : kSplitStages;  // (the ring also holds the CTA's sums)
  while (stages > 2 && split_smem(stages, P.xrows) > room) --stages;
  P.stages = stages;
  const size_t w_rows = static_cast<size_t>(A.n) * (GATED ? 2 : 1);
  if (!encode_codes(&P.tx, A.x, A.k, static_cast<size_t>(A.m), A.ldx, P.xrows) ||
      !encode_codes(&P.tw, A.w, A.k, w_rows, A.ldw, out))
    return LMPS_ERR_INVALID_ARGUMENT;
  const size_t smem = split_smem(stages, P.xrows);
  const int attr = lmps_max_dyn_smem<split_kernel<GATED>>(static_cast<int>(smem));
  if (attr != LMPS_OK) return attr;
  return launch_clusters(split_kernel<GATED>, dim3(tiles, 1, splits), kSplitThreads, smem, dim3(1, 1, splits), st, P);
}

template <bool GATED>
static int launch_whole(const Args& A, int* error, int sms, cudaStream_t st) {
  Params P{};
  P.a = A;
  P.error = error;
  P.xrows = (A.m + 15) / 16 * 16;
  constexpr int out = GATED ? 64 : 128;
  const int tiles = (A.n + out - 1) / out, steps = (A.k + kBK - 1) / kBK;
  const int most = tiles > sms ? 3 : kWholeStages;  // (two CTAs an SM, the loads of one under the epilogue of the other)
  P.stages = steps < most ? steps : most;
  if (!encode_codes(&P.tx, A.x, A.k, static_cast<size_t>(A.m), A.ldx, P.xrows) ||
      !encode_codes(&P.tw, A.w, A.k, static_cast<size_t>(A.n) * (GATED ? 2 : 1), A.ldw, out))
    return LMPS_ERR_INVALID_ARGUMENT;
  const size_t smem = whole_smem(P.stages);
  const int attr = lmps_max_dyn_smem<whole_kernel<GATED>>(static_cast<int>(smem));
  if (attr != LMPS_OK) return attr;
  return lmps_launch_pdl(whole_kernel<GATED>, dim3(tiles), dim3(kWholeThreads), smem, st, P);
}

template <int BN, bool GATED, int SPLITS = 1>
static int launch_pair(const Args& A, int* error, int sms, cudaStream_t st) {
  Params P{};
  P.a = A;
  P.error = error;
  constexpr int kOut = PairShape<BN, GATED>::kOut;
  P.tiles_n = (A.n + kOut - 1) / kOut;
  const long long tiles = static_cast<long long>(P.tiles_n) * ((A.m + 255) / 256);
  if (tiles > (1ll << 30)) return LMPS_ERR_UNSUPPORTED;
  P.tiles = static_cast<int>(tiles);
  const size_t w_rows = static_cast<size_t>(A.n) * (GATED ? 2 : 1);
  if (!encode_codes(&P.tx, A.x, A.k, static_cast<size_t>(A.m), A.ldx, 128) ||
      !encode_codes(&P.tw, A.w, A.k, w_rows, A.ldw, BN / 2))
    return LMPS_ERR_INVALID_ARGUMENT;
  using Sh = PairShape<BN, GATED, SPLITS>;
  P.tma_y = rows16(A.y, A.ldy) && (!A.residual || rows16(A.residual, A.ldr));
  const CUtensorMapSwizzle swz = Sh::kMine == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if (P.tma_y && (!encode_2d(&P.ty, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, A.y, static_cast<uint64_t>(A.n),
                             static_cast<uint64_t>(A.m), A.ldy * 2, Sh::kMine, 32, swz) ||
                  (A.residual && !encode_2d(&P.tr, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, A.residual,
                                            static_cast<uint64_t>(A.n), static_cast<uint64_t>(A.m), A.ldr * 2, Sh::kMine,
                                            32, swz))))
    return LMPS_ERR_INVALID_ARGUMENT;
  constexpr int kBytes = static_cast<int>(Sh::kSmem);
  const int attr = lmps_max_dyn_smem<pair_kernel<BN, GATED, SPLITS>>(kBytes);
  if (attr != LMPS_OK) return attr;
  // one tile a cluster where K is split, else a pair walks several
  const int clusters = SPLITS > 1 || P.tiles < sms / 2 ? P.tiles : sms / 2;
  return launch_clusters(pair_kernel<BN, GATED, SPLITS>, dim3(2 * SPLITS * clusters), Sh::kThreads, kBytes,
                         dim3(2 * SPLITS), st, P);
}

static long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// Clusters of SPLITS pairs that the current device holds at once (asked once a device; 0: an error, then K is not split).
template <int SPLITS>
static int resident_clusters() {
  constexpr int kMaxDevices = 64;
  static int known[kMaxDevices] = {};  // the number, plus one
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  if (const int n = __atomic_load_n(&known[dev], __ATOMIC_ACQUIRE)) return n - 1;
  using Sh = PairShape<128, false, SPLITS>;
  if (lmps_max_dyn_smem<pair_kernel<128, false, SPLITS>>(static_cast<int>(Sh::kSmem)) != LMPS_OK) return 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * SPLITS);
  cfg.blockDim = dim3(Sh::kThreads);
  cfg.dynamicSmemBytes = Sh::kSmem;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2 * SPLITS;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, pair_kernel<128, false, SPLITS>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  __atomic_store_n(&known[dev], n + 1, __ATOMIC_RELEASE);
  return n;
}

template <bool GATED>
static int launch(const Args& A, int* error, int sms, cudaStream_t st) {
  const long long codes = static_cast<long long>(A.n) * A.k * (GATED ? 2 : 1);  // weight bytes
  // Weights straight into mma.sync: up to 8 tokens always (8 x 8960 x 1536 gated 7.1 us, split_kernel 9.0), up to 16
  // with at most a tile an SM (16 x 1536 x 8960 6.9, 7.7; not 16 x 8192 x 1536: 6.8, 5.4), up to 32 with small
  // weights (32 x 2048 x 1536 2.9, 4.3; not 32 x 1536 x 8960: 8.7, 8.0).
  if (A.m <= 8) return launch_few<1, GATED>(A, sms, st);
  if (A.m <= 16 && ceil_div(A.n, 16) <= sms) return launch_few<2, GATED>(A, sms, st);
  if (A.m <= 32 && codes <= (4 << 20)) return launch_few<4, GATED>(A, sms, st);
  // CTA pairs with 128 or 256 weight rows a tile, by the waves they take: a tile of 128 takes 0.78 of the time of one
  // of 256 (16384 x 8960 x 1536 gated: 495, 318 us), so it is for equal waves (1024 x 2048 x 1536: 9.5, 11.0 us).
  const int pairs = sms / 2;
  const long long rows = ceil_div(A.m, 256), t128 = rows * ceil_div(A.n, GATED ? 64 : 128),
                  t256 = rows * ceil_div(A.n, GATED ? 128 : 256);
  // Up to 64 tokens, and up to 128 where pairs would leave two thirds of the GPU idle, the weights are the MMA's 128
  // rows (128 x 1536 x 8960 8.3 us, pairs 11.7; not 128 x 8192 x 1536: 10.7, 10.0).
  // Wide outputs for 33 to 64 tokens, or 128 where there is no tile a second time: K whole in a CTA, the tokens as the
  // MMA's rows, nothing exchanged (64 x 8960 x 1536 gated 7.8 -> 6.5 us, 128 x 8960 x 1536 9.0 -> 7.4; 16 x 8960 x 1536
  // would be 6.7 instead of 6.0, 128 x 151936 x 1536 74 instead of 59).  Not for rows of y at odd places (64 x 9500 x
  // 1536: 14.8 us, 7.3 split).
  const long long whole = ceil_div(A.n, GATED ? 64 : 128);
  if (A.m > 32 && A.m <= (whole <= sms ? 128 : 64) && !A.residual && rows16(A.y, A.ldy) && 2 * whole >= sms)
    return launch_whole<GATED>(A, error, sms, st);
  if (A.m <= 64 || (A.m <= kSplitTokens && 3 * t128 < pairs)) return launch_split<GATED>(A, error, sms, st);
  // Few tiles: two or four pairs share K out, six steps or more each, as far as their clusters of four or eight CTAs
  // are all resident at once (512 x 1536 x 8960 24 -> 16 us with two, 700 x 1300 x 8960 25 -> 17; 768 x 1536 x 8960
  // would be 31 instead of 24).
  if constexpr (!GATED) {
    const long long steps = ceil_div(A.k, kBK);
    if (4 * t128 <= pairs && steps >= 24 && t128 <= resident_clusters<4>())
      return launch_pair<128, false, 4>(A, error, sms, st);
    if (2 * t128 <= pairs && steps >= 12 && t128 <= resident_clusters<2>())
      return launch_pair<128, false, 2>(A, error, sms, st);
  }
  if (100 * ceil_div(t256, pairs) > 78 * ceil_div(t128, pairs)) return launch_pair<128, GATED>(A, error, sms, st);
  return launch_pair<256, GATED>(A, error, sms, st);
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
  if (k > w8::kMaxK || m > (1 << 29) || n > (1 << 29)) return LMPS_ERR_UNSUPPORTED;  // (tile numbers and rows fit 32 bits)
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
  cudaStream_t st = lmps_stream(stream);
  int sms = 0;
  if (const int e = w8::device_sms(&sms)) return e;
  return swiglu ? w8::launch<true>(A, error, sms, st) : w8::launch<false>(A, error, sms, st);
}

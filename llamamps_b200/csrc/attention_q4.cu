// Decode attention over the paged 4-bit KV cache (kv_q4.cuh: format).
//
// For the query heads h of one KV head and one sequence of n positions:
//   s_i = 0.088388 q_h . k_i,  p = softmax(s),  o_h = sum_i p_i v_i,
// with k_i = c s (codes times the scale of their 32-element group).  K's codes
// go to the tensor cores as exact fp16 integers and their scales are applied in
// fp32 around them; V's go there times their scales, which is exact in fp16
// (kv_q4.cuh).  So neither K nor V is rounded:
//   S = sum_g ks[i, g] (sum_{d in g} c_k[i, d] q[d])   4 accumulators a block
//   O = sum_i p_i (c_v[i, d] vs[i, g])
// P is rounded to fp16 once, held times 2^15: under a running maximum p is at
// most 1, so it keeps 11 bits down to 2^-29 of the maximum whatever V's size.
// (P times V's scale instead, over codes, lost the weights behind a strong
// position where V is small: 2500 positions of size 0.01, 7e-3 of the result.)
//
// mma.sync m16n8k16: M = 16 positions (S) or 16 dims (O), N = 8 heads.
// tcgen05 has M = 128 rows: with at most 8 query heads a KV head it would
// spend 15 of 16 rows on nothing, and its operands would have to be written
// to shared memory as fp16 first; the work here is unpacking nibbles.
// Fragments come straight from the nibbles:
//   K (A operand, rows = positions): ldmatrix gives lane (g8, t) word 4g + t
//     of row g8, the dims 32g + 8t + 0..7; masking gives pairs (n, n + 4), and
//     the sum over dims does not care about their order, so q is loaded in the
//     same order.
//   V (A operand, rows = dims): a transposing ldmatrix over halfwords (4 dims)
//     gives halfword g8 of positions 2t and 2t + 1 in one register, and masking
//     then gives (position 2t, position 2t + 1) pairs of one dim.
//     m-tile 2g + m: rows r < 8 are dims 32g + 4r + 2m, rows r >= 8 the dims
//     32g + 4(r - 8) + 2m + 1; a lane ends with 4 consecutive dims per group.
//
// A CTA has one KV head of a row, of a share of a row that it merges with the
// other CTAs of its cluster, or (long or many rows) of an equal share of all
// rows laid end to end, merged by a second kernel; the lengths are on the
// device, so the shares are found there.  A warp walks its own 32-position
// steps through its own ring of cp.async stages; no CTA-wide barrier until the
// warps' states meet.  16-byte chunk c of a staged row r is stored at
// c ^ ((r >> 1) & 3): both fragment reads are then free of bank conflicts.
//
// What bounds it.  A step of 32 positions is 4.6 KB and some 740 instructions a
// warp (unpacking, scales, the softmax): with 12 warps an SM goes through its
// steps at 4.4 TB/s over the GPU, 0.7 of the measured copy rate, issue slots
// (55 % used) and memory latency about even.  What is left is around them: 4 us of an empty
// call (launch, page table, first loads, meeting of the warps) and 3 us of the
// second kernel.  Measured (12 query, 2 KV heads, a stream of calls on a few
// caches): 1 x 131 4.2 us; 64 x 1..1000 9.8; 4 x 32768 19.1 (2.0 TB/s);
// 64 x 4100..8200 35.4 (3.1 TB/s; on caches that are never in L2 36.2); with
// RoPE and append 1 x 2049 8.0, 64 x 500..2100 on 6 heads 11.5.  Tried without gain: a third stage, 16 warps of 128 registers, codes
// left as fp16 subnormals (a third fewer unpacking instructions, but the offset
// then goes into the sums in fp32).
#include <algorithm>
#include <cmath>

#include "attention_q4.cuh"
#include "flash_decode.cuh"

namespace lmps {
namespace q4 {

// Warps per CTA.  A step takes a lone warp 1.4 us, so short rows want many warps at once: 8, one CTA to an SM
// (1 x 131: with 4 warps 0.6 us longer).  Pieces, and rows of which there are more than SMs, have 4, three CTAs to
// an SM.  The 12 warps may have 168 registers each; 16 of 128 take longer (64 x 1..1000 in one CTA a row: 12.6 us
// against 9.3).
constexpr int kShortWarps = 8, kPieceWarps = 4;
constexpr int kSms = 148, kPieceCtas = 3;
constexpr int kStep = 32;  // positions per warp step: two runs of 16
constexpr int kStages = 2;
constexpr int kHead = 8, kManyShares = 8;
constexpr int kMaxCluster = 8;
constexpr float kPBias = 15.0f;  // P is held times 2^15
constexpr int kClusterShare = 1280;  // positions of a CTA up to which a row is shared by a cluster
constexpr int kOffV = kStep * kCodeBytes;
constexpr int kOffKs = 2 * kOffV;
constexpr int kOffVs = kOffKs + kStep * 8;
constexpr int kStageBytes = kOffVs + kStep * 8;  // 4608

struct AttnParams {
  const __half* q;  // [rows, n_q * 128]
  Cache c;
  const int32_t* seq_lens;  // [rows]
  __half* out;              // [rows, n_q * 128]
  float* part_o;            // with more than one split: Partials
  float2* part_ml;
  int2* pieces;             // with more than one split: first piece and their number, per row
  int n_q, n_splits, rows, max_seq_len;
  int cluster;  // CTAs of a cluster that share a row (0: pieces and a merge kernel where n_splits > 1)
  // fused RoPE + append (qkv != nullptr)
  const __half* qkv;
  const int32_t* pos;
  const float* inv_freq;
  int style;
  uint8_t* k_new;
  uint8_t* v_new;

  // Positions of a row that are in the cache.
  __device__ __forceinline__ int length(int row) const { return max(0, min(seq_lens[row], max_seq_len)); }
};

// mma.sync m16n8k16 without `volatile`: the scheduler may move it among the unpacking.
__device__ __forceinline__ void mma_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// Four 8 x 8 matrices of 16-bit elements, 16-byte rows at the lanes' addresses (lanes 8i .. 8i+7: matrix i).
__device__ __forceinline__ void ldmatrix4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void load_scales(const unsigned char* p, float (&s)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
  const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  s[0] = lo.x;
  s[1] = lo.y;
  s[2] = hi.x;
  s[3] = hi.y;
}
// The scales of the two rows at p (16-byte aligned) as pairs, one per group, with `keep` cleared bits zero.
__device__ __forceinline__ void load_scale_pairs(const unsigned char* p, uint32_t keep, uint32_t (&s)[4]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  s[0] = __byte_perm(v.x, v.z, 0x5410) & keep;
  s[1] = __byte_perm(v.x, v.z, 0x7632) & keep;
  s[2] = __byte_perm(v.y, v.w, 0x5410) & keep;
  s[3] = __byte_perm(v.y, v.w, 0x7632) & keep;
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Of the units of all rows, heads included: first one of the current row, the CTA's share from .. last - 1; their
// number and that of the shares.
struct Share {
  unsigned long long before, from, last, total, ctas;
  int row, head;
};

template <int kWarps>
struct __align__(16) Smem {
  union {
    unsigned char stage[kWarps][kStages][kStageBytes];
    float wo[kWarps][kMaxHeads][kDim];  // after the steps: the warps' O
  };
  __half q[kMaxHeads][kDim];
  uint32_t knew[kRowBytes / 4], vnew[kRowBytes / 4];  // the appended row (fused form)
  double2 csd[kDim / 2];  // (cos, sin) of the new position: K's and q's
  float2 csf[kDim / 2];
  float wm[kWarps][kMaxHeads], wl[kWarps][kMaxHeads], wf[kWarps][kMaxHeads];
  float cm[kMaxHeads], cl[kMaxHeads];
  Share share;
  __align__(16) float co[kMaxHeads][kDim];  // the CTA's, for the other CTAs of a cluster
};

// This word, or these four, of shared memory in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(const float* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(const float* p, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr(p, rank))
               : "memory");
  return v;
}
__device__ __forceinline__ void fma4(float4& a, const float4& x, float f) {
  a.x = fmaf(x.x, f, a.x);
  a.y = fmaf(x.y, f, a.y);
  a.z = fmaf(x.z, f, a.z);
  a.w = fmaf(x.w, f, a.w);
}
// o / l as fp16 (zeros where there was no position).
__device__ __forceinline__ void store_row4(__half* dst, const float4& o, float l) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const __half2 lo = __floats2half2_rn(o.x * inv, o.y * inv), hi = __floats2half2_rn(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A warp's running state: per lane heads 2t, 2t + 1; m is the largest score q . k, l the lane's own part of the
// sum; l and O times 2^kPBias.
struct State {
  float o[8][4];
  float m0, m1, l0, l1;
};

// Folds the staged step (first position p0, `end` exclusive; `ok` bit x: run x
// is loaded) into the state.  kFull: every position counts.
template <bool kFull>
__device__ __forceinline__ void fold_step(const unsigned char* st, int p0, int end, uint32_t ok,
                                          const uint32_t (&qf)[16], State& S) {
  const int lane = threadIdx.x & 31, g8 = lane >> 2;
  // this lane's row address for ldmatrix: row lane & 7, chunk lane >> 3, stored at chunk ^ ((row >> 1) & 3)
  const uint32_t lm = smem_u32(st) + (lane & 7) * kCodeBytes + (((lane >> 3) ^ ((lane >> 1) & 3)) << 4);
  float s[2][4];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    uint32_t w0[4], w1[4];  // word 4g + t of rows g8 and g8 + 8
    ldmatrix4(lm + 16 * x * kCodeBytes, w0);
    ldmatrix4(lm + (16 * x + 8) * kCodeBytes, w1);
    float ks0[4], ks1[4];
    load_scales(st + kOffKs + (16 * x + g8) * 8, ks0);
    load_scales(st + kOffKs + (16 * x + g8 + 8) * 8, ks1);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const uint32_t a0 = w0[g], a1 = w1[g];
      float a[4];
      mma_zero(a, codes_lo(a0), codes_lo(a1), codes_hi(a0), codes_hi(a1), qf[4 * g], qf[4 * g + 1]);
      mma(a, codes_lo(a0 >> 8), codes_lo(a1 >> 8), codes_hi(a0 >> 8), codes_hi(a1 >> 8), qf[4 * g + 2], qf[4 * g + 3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ks = i < 2 ? ks0[g] : ks1[g];
        s[x][i] = g == 0 ? ks * a[i] : fmaf(ks, a[i], s[x][i]);
      }
    }
    if (!kFull) {  // rows g8, g8 + 8 of the run that do not count
      const int left = ((ok >> x) & 1u) ? end - p0 - 16 * x - g8 : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) s[x][i] = (i < 2 ? left > 0 : left > 8) ? s[x][i] : -INFINITY;
    }
  }
  float mx0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2]));
  float mx1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
  }
  if (__any_sync(0xffffffffu, mx0 > S.m0 || mx1 > S.m1)) {  // some head's max grew
    const float n0 = fmaxf(S.m0, mx0), n1 = fmaxf(S.m1, mx1);
    // a head without a position yet keeps max -inf; its sums are zero
    const float a0 = n0 == -INFINITY ? 1.0f : ex2((S.m0 - n0) * kScaleLog2);
    const float a1 = n1 == -INFINITY ? 1.0f : ex2((S.m1 - n1) * kScaleLog2);
    S.l0 *= a0;
    S.l1 *= a1;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      S.o[mt][0] *= a0;
      S.o[mt][2] *= a0;
      S.o[mt][1] *= a1;
      S.o[mt][3] *= a1;
    }
    S.m0 = n0;
    S.m1 = n1;
  }
  // differences to the maximum before the scale: exactly 0 at the maximum, so that P stays below 2^15 for scores of
  // any size
  const float m0 = S.m0 == -INFINITY ? 0.0f : S.m0, m1 = S.m1 == -INFINITY ? 0.0f : S.m1;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const float e0 = ex2(fmaf(s[x][0] - m0, kScaleLog2, kPBias)), e1 = ex2(fmaf(s[x][1] - m1, kScaleLog2, kPBias));
    const float e2 = ex2(fmaf(s[x][2] - m0, kScaleLog2, kPBias)), e3 = ex2(fmaf(s[x][3] - m1, kScaleLog2, kPBias));
    S.l0 += e0 + e2;
    S.l1 += e1 + e3;
    uint32_t u0[4], u1[4];  // halfword g8 of chunk g: positions 2t, 2t + 1 and 2t + 8, 2t + 9
    ldmatrix4_trans(lm + kOffV + 16 * x * kCodeBytes, u0);
    ldmatrix4_trans(lm + kOffV + (16 * x + 8) * kCodeBytes, u1);
    uint32_t vs0[4], vs1[4];  // their scales; of positions that do not count zero, whatever lies there
    uint32_t keep0 = 0xFFFFFFFFu, keep1 = 0xFFFFFFFFu;
    if (!kFull) {
      const int left = ((ok >> x) & 1u) ? end - p0 - 16 * x - 2 * (lane & 3) : 0;
      keep0 = left > 1 ? 0xFFFFFFFFu : left == 1 ? 0x0000FFFFu : 0u;
      keep1 = left > 9 ? 0xFFFFFFFFu : left == 9 ? 0x0000FFFFu : 0u;
    }
    load_scale_pairs(st + kOffVs + (16 * x + 2 * (lane & 3)) * 8, keep0, vs0);
    load_scale_pairs(st + kOffVs + (16 * x + 2 * (lane & 3) + 8) * 8, keep1, vs1);
    const uint32_t b0 = transpose(fd::pack_half2(e0, e1)), b1 = transpose(fd::pack_half2(e2, e3));
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const uint32_t u = u0[g], w = u1[g];
      mma(S.o[2 * g], mul2(codes_lo(u), vs0[g]), mul2(codes_hi(u), vs0[g]), mul2(codes_lo(w), vs1[g]),
          mul2(codes_hi(w), vs1[g]), b0, b1);
      mma(S.o[2 * g + 1], mul2(codes_lo(u >> 8), vs0[g]), mul2(codes_hi(u >> 8), vs0[g]),
          mul2(codes_lo(w >> 8), vs1[g]), mul2(codes_hi(w >> 8), vs1[g]), b0, b1);
    }
  }
}

// Attends to positions start .. end - 1 of a row of T.  `slot`: where its partials go (pieces).
template <int kWarps>
__device__ __forceinline__ void attend(const AttnParams& P, Smem<kWarps>& S, int row, int T, int start, int end,
                                       size_t slot) {
  constexpr int kThreads = kWarps * kWarp;
  const int kvh = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
  const int G = P.n_q / P.c.n_kv;
  if (tid == 0 && kvh == 0 && start == 0) {
    const int given = P.seq_lens[row];
    if (given < 0 || given > P.max_seq_len) raise_error(P.c.error, kErrPosition);
  }
  const int32_t* bt = P.c.bt + static_cast<size_t>(row) * P.c.max_pages;
  int pnew = -1;

  const uint32_t ring = smem_u32(&S.stage[warp][0][0]);
  const uint32_t scale_off = static_cast<uint32_t>(P.c.page_size) * kCodeBytes;
  const uint32_t block_bytes = static_cast<uint32_t>(P.c.page_size) * kRowBytes;
  const bool one_page = P.c.page_size % kStep == 0;  // a step's two runs lie in one page
  // Page of the run at position p (or -1: past the end or a bad page).
  auto page_of = [&](int p) {
    if (p >= end) return -1;
    const int page = __ldg(bt + P.c.page_index(p));
    if (static_cast<uint32_t>(page) < static_cast<uint32_t>(P.c.n_pages)) return page;
    if (lane == 0) raise_error(P.c.error, kErrPage);
    return -1;
  };
  // Pages of the two runs of the step at p.
  auto pages_of = [&](int p) {
    const int a = page_of(p);
    return make_int2(a, one_page ? a : page_of(p + 16));
  };
  // Copies the step at p0 into stage sb; returns the bits of the loaded runs.  Code chunk i of a run
  // (row i / 4) goes to chunk (i & 3) ^ ((row >> 1) & 3) of its row; 8 rows on that is the same place.
  // In one page the step is 2048 and 256 contiguous bytes of K, and of V (rows past the end are in the
  // page too, and masked).
  const uint32_t code_dst = (lane >> 2) * kCodeBytes + (((lane & 3) ^ ((lane >> 3) & 3)) << 4);
  const uint8_t* const scale_pool = lane < 16 ? P.c.k : P.c.v;
  const uint32_t scale_dst = (lane < 16 ? kOffKs : kOffVs) + 16 * (lane & 15);
  auto load = [&](int p0, int sb, int2 pages) {
    const uint32_t st = ring + sb * kStageBytes;
    if (one_page) {
      if (pages.x < 0) return 0u;
      const uint32_t off = p0 - P.c.page_index(p0) * P.c.page_size;
      const size_t blk = static_cast<size_t>(static_cast<uint32_t>(pages.x) * P.c.n_kv + kvh) * block_bytes;
      const uint8_t* k = P.c.k + (blk + off * kCodeBytes + 16 * lane);
      const uint8_t* v = P.c.v + (blk + off * kCodeBytes + 16 * lane);
      const uint32_t d = st + code_dst;
#pragma unroll
      for (int x = 0; x < kStep / 8; ++x) {
        cp16(d + 8 * kCodeBytes * x, k + 8 * kCodeBytes * x);
        cp16(d + kOffV + 8 * kCodeBytes * x, v + 8 * kCodeBytes * x);
      }
      cp16(st + scale_dst, scale_pool + (blk + scale_off + off * 8 + 16 * (lane & 15)));
      return 3u;
    }
    uint32_t ok = 0u;
#pragma unroll 1
    for (int x = 0; x < 2; ++x) {
      const int page = x ? pages.y : pages.x;
      if (page < 0) continue;
      ok |= 1u << x;
      const int p = p0 + 16 * x, off = p - P.c.page_index(p) * P.c.page_size;
      const size_t at = P.c.block(page, kvh), code = at + off * kCodeBytes + 16 * lane;
      const uint32_t d = st + 16 * x * kCodeBytes + code_dst;
      cp16(d, P.c.k + code);
      cp16(d + 8 * kCodeBytes, P.c.k + code + 8 * kCodeBytes);
      cp16(d + kOffV, P.c.v + code);
      cp16(d + kOffV + 8 * kCodeBytes, P.c.v + code + 8 * kCodeBytes);
      if ((lane & 15) < 8)  // scales: 8 chunks of K, 8 of V
        cp16(st + scale_dst + 128 * x, scale_pool + at + scale_off + off * 8 + 16 * (lane & 7));
    }
    return ok;
  };

  // the first step's copies are on their way while the queries are prepared
  const int first = start + warp * kStep, stride = kWarps * kStep;
  uint32_t ok = first < end ? load(first, 0, pages_of(first)) : 0u;
  asm volatile("cp.async.commit_group;" ::: "memory");
  int sb = 0;
  int2 next = pages_of(first + stride);

  if (P.qkv) {
    const int p = P.pos[row];
    const bool mine = p >= 0 && p == T - 1 && p >= start && p < end;
    if (p != T - 1 && tid == 0) raise_error(P.c.error, kErrPosition);
    const int heads = P.n_q + 2 * P.c.n_kv;
    const __half* src = P.qkv + static_cast<size_t>(row) * heads * kDim;
    if (tid < kDim / 2) {
      double2 d;
      rope_cos_sin(p, P.inv_freq[tid], d.x, d.y);
      S.csd[tid] = d;
      S.csf[tid] = make_float2(static_cast<float>(d.x), static_cast<float>(d.y));
    }
    __syncthreads();
    for (int h = warp; h < G + 2; h += kWarps) {  // the query heads, then K and V of the new position
      if (h >= G && !mine) continue;
      union {
        uint2 u;
        __half x[4];
      } e;
      const int from = h < G ? kvh * G + h : P.n_q + (h - G) * P.c.n_kv + kvh;
      e.u = *reinterpret_cast<const uint2*>(src + from * kDim + 4 * lane);
      if (h < G) {
        rotate_head(e.x, S.csf, P.style, lane);
        *reinterpret_cast<uint2*>(&S.q[h][4 * lane]) = e.u;
        continue;
      }
      if (h == G) rotate_head(e.x, S.csd, P.style, lane);
      const int pi = P.c.page_index(p), off = p - pi * P.c.page_size;
      const int page = bt[pi];
      if (page < 0 || page >= P.c.n_pages) continue;  // raised where the steps are loaded
      const float x[4] = {__half2float(e.x[0]), __half2float(e.x[1]), __half2float(e.x[2]), __half2float(e.x[3])};
      float scale;
      const uint32_t w = quantise_row(x, scale);
      uint8_t* block = (h == G ? P.k_new : P.v_new) + P.c.block(page, kvh);
      uint32_t* copy = h == G ? S.knew : S.vnew;
      *reinterpret_cast<uint16_t*>(block + off * kCodeBytes + 2 * lane) = static_cast<uint16_t>(w);
      reinterpret_cast<uint16_t*>(copy)[lane] = static_cast<uint16_t>(w);
      if ((lane & 7) == 0) {
        const __half hs = __float2half_rn(scale);
        *reinterpret_cast<__half*>(block + P.c.page_size * kCodeBytes + off * 8 + (lane >> 3) * 2) = hs;
        reinterpret_cast<__half*>(copy)[kDim / 4 + (lane >> 3)] = hs;
      }
    }
    if (mine) pnew = p;
    __syncthreads();
  }

  // B operand Q^T of this lane: head g8 (zero past the group), the word order of K's nibbles
  uint32_t qf[16];
  {
    const __half* qrow = P.qkv ? &S.q[0][0] + (g8 < G ? g8 : 0) * kDim
                               : P.q + (static_cast<size_t>(row) * P.n_q + kvh * G + (g8 < G ? g8 : 0)) * kDim;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      uint4 v = *reinterpret_cast<const uint4*>(qrow + 32 * g + 8 * t4);
      if (g8 >= G) v = make_uint4(0u, 0u, 0u, 0u);
      qf[4 * g] = __byte_perm(v.x, v.z, 0x5410);      // dims 0, 4
      qf[4 * g + 1] = __byte_perm(v.x, v.z, 0x7632);  // 1, 5
      qf[4 * g + 2] = __byte_perm(v.y, v.w, 0x5410);  // 2, 6
      qf[4 * g + 3] = __byte_perm(v.y, v.w, 0x7632);  // 3, 7
    }
  }

  State A;
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) A.o[mt][0] = A.o[mt][1] = A.o[mt][2] = A.o[mt][3] = 0.0f;
  A.m0 = A.m1 = -INFINITY;
  A.l0 = A.l1 = 0.0f;
  for (int p0 = first; p0 < end; p0 += stride) {
    uint32_t next_ok = 0u;
    if (p0 + stride < end) next_ok = load(p0 + stride, sb ^ 1, next);
    asm volatile("cp.async.commit_group;" ::: "memory");
    next = pages_of(p0 + 2 * stride);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    const uint32_t st = ring + sb * kStageBytes;
    if (pnew >= p0 && pnew < p0 + kStep) {  // the appended row over its (older) staged one
      const int r = pnew - p0, i = lane & 15;
      const uint32_t d = st + r * kCodeBytes + (((i >> 2) ^ ((r >> 1) & 3)) << 4) + 4 * (i & 3);
      if (lane < 16) asm volatile("st.shared.u32 [%0], %1;" ::"r"(d), "r"(S.knew[i]) : "memory");
      else asm volatile("st.shared.u32 [%0], %1;" ::"r"(d + kOffV), "r"(S.vnew[i]) : "memory");
      if (lane < 2) asm volatile("st.shared.u32 [%0], %1;" ::"r"(st + kOffKs + r * 8 + 4 * lane), "r"(S.knew[16 + lane]) : "memory");
      else if (lane < 4)
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(st + kOffVs + r * 8 + 4 * (lane - 2)), "r"(S.vnew[14 + lane]) : "memory");
      __syncwarp();
    }
    const unsigned char* sp = &S.stage[warp][sb][0];
    if (ok == 3u && p0 + kStep <= end) fold_step<true>(sp, p0, end, ok, qf, A);
    else if (ok) fold_step<false>(sp, p0, end, ok, qf, A);
    __syncwarp();  // the stage is free
    ok = next_ok;
    sb ^= 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  // the lanes' parts of the sums
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    A.l0 += __shfl_xor_sync(0xffffffffu, A.l0, o);
    A.l1 += __shfl_xor_sync(0xffffffffu, A.l1, o);
  }
  __syncthreads();  // every warp is done with its stages: S.wo takes their place
  if (g8 == 0) {
    S.wm[warp][2 * t4] = A.m0;
    S.wm[warp][2 * t4 + 1] = A.m1;
    S.wl[warp][2 * t4] = A.l0;
    S.wl[warp][2 * t4 + 1] = A.l1;
  }
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int d = 32 * g + 4 * g8;
    *reinterpret_cast<float4*>(&S.wo[warp][2 * t4][d]) =
        make_float4(A.o[2 * g][0], A.o[2 * g][2], A.o[2 * g + 1][0], A.o[2 * g + 1][2]);
    *reinterpret_cast<float4*>(&S.wo[warp][2 * t4 + 1][d]) =
        make_float4(A.o[2 * g][1], A.o[2 * g][3], A.o[2 * g + 1][1], A.o[2 * g + 1][3]);
  }
  __syncthreads();
  // the warps' states meet: weights once per (warp, head), then four dims a thread
  if (tid < kMaxHeads) {
    float M = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) M = fmaxf(M, S.wm[i][tid]);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      // a warp without positions has max -inf and sums 0; a NaN score leaves NaN in its sums
      const float f = S.wm[i][tid] == -INFINITY ? 1.0f : ex2((S.wm[i][tid] - M) * kScaleLog2);
      l = fmaf(S.wl[i][tid], f, l);
      S.wf[i][tid] = f;
    }
    S.cm[tid] = M;
    S.cl[tid] = l;
  }
  __syncthreads();
  __half* const out = P.out + (static_cast<size_t>(row) * P.n_q + kvh * G) * kDim;
  for (int w = tid; w < G * (kDim / 4); w += kThreads) {
    const int h = w >> 5, d = 4 * (w & 31);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) fma4(o, *reinterpret_cast<const float4*>(&S.wo[i][h][d]), S.wf[i][h]);
    if (P.n_splits == 1) {
      store_row4(out + h * kDim + d, o, S.cl[h]);
    } else if (P.cluster) {
      *reinterpret_cast<float4*>(&S.co[h][d]) = o;
    } else {
      const size_t at = slot * P.n_q + kvh * G + h;
      *reinterpret_cast<float4*>(P.part_o + at * kDim + d) = o;
      if (d == 0) P.part_ml[at] = make_float2(S.cm[h] * kScaleLog2, S.cl[h]);
    }
  }
  if (P.cluster) {  // the CTAs' states meet: each writes its part of the row
    cluster_sync();
    const int rank = blockIdx.x - row * P.cluster, units = G * (kDim / 4), share = (units + P.cluster - 1) / P.cluster;
    for (int x = tid; x < share; x += kThreads) {
      const int w = rank * share + x;
      if (w >= units) break;
      const int h = w >> 5, d = 4 * (w & 31);
      float m[kMaxCluster], l[kMaxCluster], M = -INFINITY, den = 0.0f;
      float4 o[kMaxCluster], num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < kMaxCluster; ++i)
        if (i < P.cluster) {
          m[i] = ld_cluster(&S.cm[h], i);
          l[i] = ld_cluster(&S.cl[h], i);
          o[i] = ld_cluster4(&S.co[h][d], i);
        }
#pragma unroll
      for (int i = 0; i < kMaxCluster; ++i)
        if (i < P.cluster) M = fmaxf(M, m[i]);
#pragma unroll
      for (int i = 0; i < kMaxCluster; ++i)
        if (i < P.cluster) {
          const float f = m[i] == -INFINITY ? 1.0f : ex2((m[i] - M) * kScaleLog2);
          fma4(num, o[i], f);
          den = fmaf(l[i], f, den);
        }
      store_row4(out + h * kDim + d, num, den);
    }
    cluster_sync();  // nobody's shared memory goes while it is read
  }
}

// A row a CTA, or a share of one a CTA of a cluster.
template <int kWarps>
__global__ void __launch_bounds__(kWarps * kWarp, kWarps == kShortWarps ? 1 : kPieceCtas) attn_q4_kernel(const AttnParams P) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const int parts = P.cluster ? P.cluster : 1, row = blockIdx.x / parts, T = P.length(row);
  const int share = ((T + parts - 1) / parts + kStep - 1) / kStep * kStep;
  const int start = min(T, static_cast<int>(blockIdx.x - row * parts) * share);
  attend(P, *reinterpret_cast<Smem<kWarps>*>(smem_raw), row, T, start, min(T, start + share), 0);
}

// a * b / c; in 32 bits where the product fits (a 64-bit division is some 100 instructions in a row).
__device__ __forceinline__ unsigned long long mul_div(unsigned long long a, unsigned long long b, unsigned long long c) {
  const unsigned long long ab = a * b;
  if (ab <= 0xFFFFFFFFull && c <= 0xFFFFFFFFull) return static_cast<uint32_t>(ab) / static_cast<uint32_t>(c);
  return ab / c;
}

// Equal shares of the rows laid end to end, in units of a warp's step (a row without positions has one): a share
// may take in the end of a row and the start of the next, a segment each.  `head` units in front of each row
// stand for what starting another segment costs: under load a chain of three memory accesses, which other shares
// hide only where every SM has many of them to do.  So with kManyShares shares or more to a row a head is one
// unit longer than a share of the rows without heads.  The heads make a share longer by `head` times the rows to a
// share, an eighth at most, so few shares take in two rows: of 54 x 8000..16000 on one KV head 1 of 444 (fresh
// caches: 8 x 20000..30000 24.5 us, 29 with short heads; 32 x 1..16000 25.6 and 24.2).  Segment (CTA i, row r) has slot i + r.
__global__ void __launch_bounds__(kPieceWarps * kWarp, kPieceCtas) attn_q4_pieces_kernel(const AttnParams P) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Smem<kPieceWarps>& S = *reinterpret_cast<Smem<kPieceWarps>*>(smem_raw);
  constexpr int kUnit = kStep;
  const int lane = threadIdx.x & 31;
  auto units = [](int len) { return max(1, (len + kUnit - 1) / kUnit); };
  {
    unsigned long long total = 0ull, before = 0ull;  // before: units of the rows in front
    for (int r = lane; r < P.rows; r += kWarp) total += units(P.length(r));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const int head = gridDim.x >= static_cast<unsigned>(kManyShares) * P.rows ? static_cast<int>(total / gridDim.x) + 1 : kHead;
    total += static_cast<unsigned long long>(head) * P.rows;
    const unsigned long long ctas = min(static_cast<unsigned long long>(gridDim.x), total);
    if (blockIdx.x >= ctas) return;
    const unsigned long long from = mul_div(blockIdx.x, total, ctas);
    int row = 0, r0 = 0;
    for (;; r0 += kWarp) {  // ends: `from` is below the total
      const int r = r0 + lane, mine = r < P.rows ? head + units(P.length(r)) : 0;
      int sum = mine;  // inclusive prefix
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, from < before + sum);
      if (hit) {
        const int l = __ffs(hit) - 1;
        row = r0 + l;
        before += __shfl_sync(0xffffffffu, sum - mine, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (threadIdx.x == 0) S.share = Share{before, from, mul_div(blockIdx.x + 1, total, ctas), total, ctas, row, head};
  }
  for (;;) {
    __syncthreads();
    const Share sh = S.share;
    const int T = P.length(sh.row), n = sh.head + units(T);
    const unsigned long long next = sh.before + n;
    const int first = max(0, static_cast<int>(max(sh.from, sh.before) - sh.before) - sh.head);
    const int stop = static_cast<int>(min(next, sh.last) - sh.before) - sh.head;
    if (stop > first) {  // (uniform) else only the head of the row
      // The owner of the row's first positions tells the merge from where to where: unit u is in share
      // ((u + 1) * ctas - 1) / total.
      if (first == 0 && blockIdx.y == 0 && threadIdx.x == 0)
        P.pieces[sh.row] = make_int2(static_cast<int>(blockIdx.x) + sh.row,
                                     static_cast<int>((next * sh.ctas - 1) / sh.total) - static_cast<int>(blockIdx.x) + 1);
      attend(P, S, sh.row, T, first * kUnit, min(T, stop * kUnit), static_cast<size_t>(blockIdx.x) + sh.row);
    }
    __syncthreads();  // the segment's states and the share are read
    if (S.share.before + n >= S.share.last) return;
    __syncthreads();
    if (threadIdx.x == 0) {
      S.share.before += n;
      ++S.share.row;
    }
  }
}

constexpr int kMergeWarps = 8, kMergeLoads = 8;
// Log-sum-exp merge of the n pieces first + s * step of a (row, query head) by a warp, 4 dims a lane.  Lane j
// holds the weight of piece j of a chunk of 32; eight partials are on their way at a time.
__device__ __forceinline__ void merge_row(const Partials& P, size_t first, size_t step, int pieces, __half* out) {
  const int lane = threadIdx.x & 31;
  const float2* ml = P.ml + first;
  const float4* o = reinterpret_cast<const float4*>(P.o + first * kDim) + lane;
  const size_t stride = step * (kDim / 4);
  float M = -INFINITY, den = 0.0f;  // den: of this lane's pieces
  float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s0 = 0; s0 < pieces; s0 += kWarp) {
    const float2 m = s0 + lane < pieces ? ml[(s0 + lane) * step] : make_float2(-INFINITY, 0.0f);
    const int n = min(kWarp, pieces - s0);
    float f = 0.0f;
    for (int j0 = 0; j0 < n; j0 += kMergeLoads) {
      float4 v[kMergeLoads];
#pragma unroll
      for (int j = 0; j < kMergeLoads; ++j)
        v[j] = j0 + j < n ? o[(s0 + j0 + j) * stride] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (j0 == 0) {  // the weights, while the first partials travel
        const float top = fmaxf(M, warp_max(m.x));
        const float keep = M == -INFINITY ? 1.0f : ex2(M - top);
        // a piece without positions has max -inf and sums 0; a NaN score leaves NaN in its sums
        f = m.x == -INFINITY ? 1.0f : ex2(m.x - top);
        M = top;
        den = fmaf(den, keep, m.y * f);
        num.x *= keep, num.y *= keep, num.z *= keep, num.w *= keep;
      }
#pragma unroll
      for (int j = 0; j < kMergeLoads; ++j) {
        const float w = __shfl_sync(0xffffffffu, f, (j0 + j) & 31);
        num.x = fmaf(v[j].x, w, num.x);
        num.y = fmaf(v[j].y, w, num.y);
        num.z = fmaf(v[j].z, w, num.z);
        num.w = fmaf(v[j].w, w, num.w);
      }
    }
  }
  den = warp_sum(den);
  store_row4(out + 4 * lane, num, den);
}

// The merge of one (row, query head) of a decode call.  A warp takes every 8th
// piece, 4 dims a lane; the partials of the first 64 pieces are on their way
// before the weights are known.  Of a row of eight pieces or fewer every eighth
// CTA merges eight heads, a warp each, and the others are done (64 rows of
// 4100..8200: 37.3 -> 35.6 us; 4 of 32768, 37 pieces each, with a warp per head: 17.8 -> 20.8).
__global__ void __launch_bounds__(kMergeWarps * kWarp) attn_q4_combine_kernel(const Partials P) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  __shared__ float red[2][kMergeWarps];
  __shared__ float4 acc[kMergeWarps][kWarp];
  const int h = blockIdx.y, row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int2 pc = P.pieces[row];
  const size_t step = P.n_q, first = pc.x * step + h;  // piece s at first + s * step
  if (pc.y <= kMergeLoads) {
    if (h % kMergeWarps == 0 && h + warp < P.n_q)
      merge_row(P, first + warp, step, pc.y, P.out + (static_cast<size_t>(row) * P.n_q + h + warp) * kDim);
    return;
  }
  const float2* ml = P.ml + first;
  const float4* o = reinterpret_cast<const float4*>(P.o + first * kDim) + lane;
  const size_t stride = step * (kDim / 4);
  float4 v[kMergeLoads];
#pragma unroll
  for (int i = 0; i < kMergeLoads; ++i) {
    const int s = warp + kMergeWarps * i;
    v[i] = s < pc.y ? o[s * stride] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  float M = -INFINITY;
  for (int s = tid; s < pc.y; s += kMergeWarps * kWarp) M = fmaxf(M, ml[s * step].x);
  M = warp_max(M);
  if (lane == 0) red[0][warp] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMergeWarps; ++i) M = fmaxf(M, red[0][i]);
  float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float den = 0.0f;
  auto add = [&](int s, const float4& x) {
    const float2 m = ml[s * step];
    // a piece without positions has max -inf and sums 0; a NaN score leaves NaN in its sums
    const float f = m.x == -INFINITY ? 1.0f : ex2(m.x - M);
    den = fmaf(m.y, f, den);
    num.x = fmaf(x.x, f, num.x);
    num.y = fmaf(x.y, f, num.y);
    num.z = fmaf(x.z, f, num.z);
    num.w = fmaf(x.w, f, num.w);
  };
#pragma unroll
  for (int i = 0; i < kMergeLoads; ++i)
    if (warp + kMergeWarps * i < pc.y) add(warp + kMergeWarps * i, v[i]);
  for (int s = warp + kMergeWarps * kMergeLoads; s < pc.y; s += kMergeWarps) add(s, o[s * stride]);
  acc[warp][lane] = num;
  if (lane == 0) red[1][warp] = den;
  __syncthreads();
  if (tid >= kDim) return;
  const float* a = reinterpret_cast<const float*>(&acc[0][0]) + tid;
  float n = 0.0f, d = 0.0f;
#pragma unroll
  for (int i = 0; i < kMergeWarps; ++i) {
    n += a[i * kDim];
    d += red[1][i];
  }
  P.out[(static_cast<size_t>(row) * P.n_q + h) * kDim + tid] = __float2half_rn(d == 0.0f ? 0.0f : n / d);
}

// The same for many queries a sequence: thousands of rows, a warp each.
// (4 x 256 queries behind 1..30000 positions, 18 MB of partials: a CTA per row 104 us the call, this one 80.)
__global__ void __launch_bounds__(kMergeWarps * kWarp) attn_q4_combine_rows_kernel(const Partials P, int n_rows) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  const int item = blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
  const int row = item / P.n_q, h = item - row * P.n_q;
  if (row >= n_rows) return;
  const int b = row / P.seq, i = row - b * P.seq;
  if (P.q_lens && i >= P.q_lens[b]) return;
  const int G = P.n_q / P.n_kv, kvh = h / G, r = i * G + (h - kvh * G), blk = r / P.rows_item;
  const int2 pc = P.pieces[(P.n_blocks - 1 - blk) * P.batch + b];
  const size_t step = static_cast<size_t>(P.n_kv) * P.rows_item;
  const size_t first = pc.x * step + static_cast<size_t>(kvh) * P.rows_item + (r - blk * P.rows_item);
  merge_row(P, first, step, pc.y, P.out + (static_cast<size_t>(row) * P.n_q + h) * kDim);
}

int combine_launch(const Partials& p, int rows, cudaStream_t stream) {
  if (p.rows_item) {
    const unsigned ctas = static_cast<unsigned>((static_cast<long long>(rows) * p.n_q + kMergeWarps - 1) / kMergeWarps);
    return lmps_launch_pdl(attn_q4_combine_rows_kernel, dim3(ctas), dim3(kMergeWarps * kWarp), 0, stream, p, rows);
  }
  return lmps_launch_pdl(attn_q4_combine_kernel, dim3(rows, p.n_q), dim3(kMergeWarps * kWarp), 0, stream, p);
}

int check_attention(int n_pages, int max_pages, int page_size, int n_q_heads, int n_kv_heads, int head_dim,
                    int max_seq_len, int n_splits) {
  LMPS_CHECK_ARG(n_pages >= 1 && max_pages >= 1 && page_size >= 1 && max_seq_len >= 1);
  LMPS_CHECK_ARG(static_cast<long long>(max_pages) * page_size <= 1LL << 29);
  LMPS_CHECK_ARG(max_seq_len <= static_cast<long long>(max_pages) * page_size);
  LMPS_CHECK_ARG(n_kv_heads >= 1 && n_q_heads >= 1 && n_q_heads % n_kv_heads == 0 && n_q_heads <= 65535);
  LMPS_CHECK_ARG(n_splits >= 1 && n_splits <= 1024);
  if (head_dim != kDim || page_size % kRun != 0 || page_size > kMaxPage || n_q_heads / n_kv_heads > kMaxHeads)
    return LMPS_ERR_UNSUPPORTED;
  return LMPS_OK;
}

template <void (*kKernel)(const AttnParams), int kWarps>
static int attn_launch(dim3 grid, cudaStream_t stream, const AttnParams& P) {
  const int st = lmps_max_dyn_smem<kKernel>(static_cast<int>(sizeof(Smem<kWarps>)));
  if (st != LMPS_OK) return st;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kWarps * kWarp);
  cfg.dynamicSmemBytes = sizeof(Smem<kWarps>);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = P.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = P.cluster ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kKernel, P);
  return e == cudaSuccess ? lmps_launch_status() : static_cast<int>(e);
}

static int attention_launch(AttnParams P, const uint8_t* k_pool, const uint8_t* v_pool, int n_pages,
                            const int32_t* block_table, uint16_t* out, void* workspace, size_t workspace_bytes,
                            int max_pages, int page_size, int n_q_heads, int n_kv_heads, int head_dim, int rows,
                            int max_seq_len, int n_splits, int32_t* error, void* stream) {
  LMPS_CHECK_ARG(k_pool && v_pool && block_table && out);
  LMPS_CHECK_ARG(rows >= 1 && rows <= 65535);
  const int st = check_attention(n_pages, max_pages, page_size, n_q_heads, n_kv_heads, head_dim, max_seq_len, n_splits);
  if (st != LMPS_OK) return st;
  LMPS_CHECK_ARG(lmps_aligned(k_pool, 16) && lmps_aligned(v_pool, 16) && lmps_aligned(out, 16));
  const size_t need = lmps_attention_q4_workspace_size(rows, n_q_heads, head_dim, n_splits);
  if (need > 0 && (!workspace || workspace_bytes < need)) return LMPS_ERR_WORKSPACE;
  LMPS_CHECK_ARG(lmps_aligned(workspace, 16));
  P.c = Cache{k_pool, v_pool, block_table, n_pages, max_pages, page_size, n_kv_heads, page_shift_of(page_size), error};
  P.out = reinterpret_cast<__half*>(out);
  P.n_q = n_q_heads;
  P.n_splits = n_splits;
  P.max_seq_len = max_seq_len;
  P.rows = rows;
  const size_t n_part = static_cast<size_t>(rows) * n_q_heads * n_splits;
  P.part_o = reinterpret_cast<float*>(workspace);
  P.part_ml = reinterpret_cast<float2*>(P.part_o + n_part * kDim);
  P.pieces = reinterpret_cast<int2*>(P.part_ml + n_part);
  Partials parts{};
  parts.o = P.part_o;
  parts.ml = P.part_ml;
  parts.pieces = P.pieces;
  parts.out = P.out;
  parts.n_q = n_q_heads;
  cudaStream_t s = lmps_stream(stream);
  // Rows of medium length go to a cluster each, whose CTAs merge through distributed shared memory: one launch
  // (with RoPE and append: 1 x 2049 7.4 us against 8.6 in pieces, 64 x 500..2100 on 6 heads 10.7 against 12.6).
  // Longer ones are cut into pieces, merged by a second kernel.
  P.cluster = n_splits > 1 && lmps_attention_q4_launches(n_splits, max_seq_len) == 1 ? n_splits : 0;
  if (n_splits == 1 || P.cluster) {  // with one CTA to an SM at most it has 8 warps, else 4
    const dim3 grid(static_cast<unsigned>(rows) * n_splits, n_kv_heads);
    const bool alone = static_cast<long long>(rows) * n_splits * n_kv_heads <= kSms;
    return alone ? attn_launch<attn_q4_kernel<kShortWarps>, kShortWarps>(grid, s, P)
                 : attn_launch<attn_q4_kernel<kPieceWarps>, kPieceWarps>(grid, s, P);
  }
  // No more shares than run at once; with the rows' borders they make at most rows * n_splits segments.
  const unsigned slots = n_kv_heads >= kSms * kPieceCtas ? 1u : kSms * kPieceCtas / n_kv_heads;
  const dim3 grid(std::min(slots, (n_splits - 1u) * rows), n_kv_heads);
  const int status = attn_launch<attn_q4_pieces_kernel, kPieceWarps>(grid, s, P);
  if (status) return status;
  return combine_launch(parts, rows, s);
}

}  // namespace q4
}  // namespace lmps

using namespace lmps;

extern "C" int lmps_attention_q4_splits(int batch, int n_kv_heads, int max_seq_len) {
  if (batch <= 0 || n_kv_heads <= 0 || max_seq_len <= 0) return 1;
  const long long items = static_cast<long long>(batch) * n_kv_heads;
  constexpr int kShort = q4::kShortWarps * q4::kStep, kPiece = q4::kPieceWarps * q4::kStep;
  if (max_seq_len <= 2 * kShort || items >= q4::kSms * q4::kPieceCtas) return 1;
  // Clusters of CTAs of 8 warps (one to an SM) or of 4, whichever gives a row more warps.  `room`: CTAs that
  // still run at once as clusters; an SM group takes few large ones, and pairs fit everywhere (us per call,
  // 12 query heads: 8 x 3000..6000 in clusters of 5 / 6 / 7 / 8 11.1 / 9.7 / 16.3 / 15.5, 6 x 3000..6000 in 8 8.8;
  // 12 x 3000..6000 in 5 / 6 11.2 / 17.0; 27 x 500..2000 of 4 warps in 7 / 8 9.8 / 14.0).
  auto fit = [max_seq_len, items](int room, int slots, int unit) {
    long long n = room / items;
    if (n > 6 && items > 12) n = unit == kShort ? 6 : n;
    if (n < 2 && slots >= 2 * items) n = 2;
    return std::min(std::min(n, static_cast<long long>(q4::kMaxCluster)), static_cast<long long>((max_seq_len + unit - 1) / unit));
  };
  const long long wide = fit(120, q4::kSms, kShort), many = fit(384, q4::kSms * q4::kPieceCtas, kPiece);
  const long long warps = std::max(wide * q4::kShortWarps, many * q4::kPieceWarps);
  // (64 x 1..1000: one CTA a row 9.4, a cluster of 3 10.1; 32 x 1..1000: 9.5 and, of 6, 8.0)
  if (items <= q4::kSms && warps < 2 * q4::kShortWarps && max_seq_len <= 4 * kShort) return 1;
  const long long cluster = wide * q4::kShortWarps >= warps ? wide : many;
  if (cluster >= 2 && max_seq_len <= cluster * q4::kClusterShare) return static_cast<int>(cluster);
  if (cluster < 2 && max_seq_len <= 8 * kShort) return 1;  // the rows alone fill the GPU, and a merge would not pay
  long long n = (q4::kSms * q4::kPieceCtas + items - 1) / items;
  const long long most = (max_seq_len + kPiece - 1) / kPiece;
  n = n < 1 ? 1 : n > most ? most : n;
  return static_cast<int>(n > 1023 ? 1024 : n + 1);
}

extern "C" int lmps_attention_q4_launches(int n_splits, int max_seq_len) {
  return n_splits <= 1 || (n_splits <= q4::kMaxCluster && max_seq_len <= n_splits * q4::kClusterShare) ? 1 : 2;
}

extern "C" size_t lmps_attention_q4_workspace_size(int batch, int n_q_heads, int head_dim, int n_splits) {
  if (n_splits <= 1 || batch <= 0 || n_q_heads <= 0 || head_dim <= 0) return 0;
  return static_cast<size_t>(batch) * n_splits * n_q_heads * (head_dim * sizeof(float) + sizeof(float2)) +
         static_cast<size_t>(batch) * sizeof(int2);
}

extern "C" int lmps_gqa_decode_attention_q4(const uint16_t* q, const uint8_t* k_pool, const uint8_t* v_pool,
                                            int n_pages, const int32_t* block_table, const int32_t* seq_lens,
                                            uint16_t* out, void* workspace, size_t workspace_bytes, int max_pages,
                                            int page_size, int n_q_heads, int n_kv_heads, int head_dim, int batch,
                                            int max_seq_len, int n_splits, int32_t* error, void* stream) {
  LMPS_CHECK_ARG(q && seq_lens && lmps_aligned(q, 16));
  q4::AttnParams P{};
  P.q = reinterpret_cast<const __half*>(q);
  P.seq_lens = seq_lens;
  return q4::attention_launch(P, k_pool, v_pool, n_pages, block_table, out, workspace, workspace_bytes, max_pages,
                              page_size, n_q_heads, n_kv_heads, head_dim, batch, max_seq_len, n_splits, error, stream);
}

extern "C" int lmps_gqa_decode_attention_rope_q4(const uint16_t* qkv, const int32_t* pos, const float* inv_freq,
                                                 int style, uint8_t* k_pool, uint8_t* v_pool, int n_pages,
                                                 const int32_t* block_table, const int32_t* seq_lens, uint16_t* out,
                                                 void* workspace, size_t workspace_bytes, int max_pages,
                                                 int page_size, int n_q_heads, int n_kv_heads, int head_dim,
                                                 int batch, int max_seq_len, int n_splits, int32_t* error,
                                                 void* stream) {
  LMPS_CHECK_ARG(qkv && pos && inv_freq && seq_lens && lmps_aligned(qkv, 16));
  LMPS_CHECK_ARG(style == LMPS_ROPE_INTERLEAVED || style == LMPS_ROPE_NEOX);
  q4::AttnParams P{};
  P.qkv = reinterpret_cast<const __half*>(qkv);
  P.pos = pos;
  P.inv_freq = inv_freq;
  P.style = style;
  P.seq_lens = seq_lens;
  P.k_new = k_pool;
  P.v_new = v_pool;
  return q4::attention_launch(P, k_pool, v_pool, n_pages, block_table, out, workspace, workspace_bytes, max_pages,
                              page_size, n_q_heads, n_kv_heads, head_dim, batch, max_seq_len, n_splits, error, stream);
}

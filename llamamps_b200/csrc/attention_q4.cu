// Decode attention over the paged 4-bit KV cache (kv_q4.cuh: format).
//
// For the query heads h of one KV head and one sequence of n positions:
//   s_i = 0.088388 q_h . k_i,  p = softmax(s),  o_h = sum_i p_i v_i,
// with k_i = c s (codes times the scale of their 32-element group).  The
// codes go to the tensor cores as exact fp16 integers and the scales are
// applied in fp32 around them, so neither K nor V is rounded:
//   S   = sum_g ks[i, g] (sum_{d in g} c_k[i, d] q[d])   4 accumulators a block
//   O_g = sum_i (p_i vs[i, g]) c_v[i, d],  d in g        P scaled per group
// (P times a V scale is rounded to fp16 once, as P alone would be.)
//
// mma.sync m16n8k16: M = 16 positions (S) or 16 dims (O), N = 8 heads.
// tcgen05 has M = 128 rows: with at most 8 query heads a KV head it would
// spend 15 of 16 rows on nothing, and its operands would have to be written
// to shared memory as fp16 first; the work here is unpacking nibbles.
// Fragments come straight from the nibbles:
//   K (A operand, rows = positions): word 4g + t of a row holds the dims
//     32g + 8t + 0..7; masking gives pairs (n, n + 4), and the sum over dims
//     does not care about their order, so q is loaded in the same order.
//   V (A operand, rows = dims): the halfwords 4(g8) .. of two positions are
//     joined by one byte permute, and masking then gives (position 2t,
//     position 2t + 1) pairs of one dim: no transpose.
//     m-tile 2g + m: rows r < 8 are dims 32g + 4r + 2m, rows r >= 8 the dims
//     32g + 4(r - 8) + 2m + 1; a lane ends with 4 consecutive dims per group.
//
// One item (split, KV head, sequence) per CTA of 4 warps.  A warp walks its
// own 32-position steps (every 4th of the split) through its own ring of
// cp.async stages; no CTA-wide barrier until the warps' states meet.  16-byte
// chunk c of a staged row r is stored at c ^ ((r >> 1) & 3): both fragment
// reads are then free of bank conflicts.
#include <cmath>

#include "attention_q4.cuh"
#include "flash_decode.cuh"

namespace lmps {
namespace q4 {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * kWarp;
constexpr int kStep = 32;  // positions per warp step: two runs of 16
constexpr int kStages = 2;
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
  int n_q, n_splits, chunk, max_seq_len;
  // fused RoPE + append (qkv != nullptr)
  const __half* qkv;
  const int32_t* pos;
  const float* inv_freq;
  int style;
  uint8_t* k_new;
  uint8_t* v_new;
};

__device__ __forceinline__ void mma_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void lds_scales(uint32_t a, float (&s)[4]) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
  const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  s[0] = lo.x;
  s[1] = lo.y;
  s[2] = hi.x;
  s[3] = hi.y;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

struct __align__(16) Smem {
  union {
    unsigned char stage[kWarps][kStages][kStageBytes];
    float wo[kWarps][kMaxHeads][kDim];  // after the steps: the warps' O
  };
  __half q[kMaxHeads][kDim];
  uint32_t knew[kRowBytes / 4], vnew[kRowBytes / 4];  // the appended row (fused form)
  double2 cs[kDim / 2];
  float wm[kWarps][kMaxHeads], wl[kWarps][kMaxHeads];
};

// A warp's running state: per lane heads 2t, 2t + 1; l is the lane's own part of the sum.
struct State {
  float o[8][4];
  float m0, m1, l0, l1;
};

// Folds the staged step (first position p0, `end` exclusive; `ok` bit x: run x
// is loaded) into the state.
__device__ __forceinline__ void fold_step(uint32_t st, int p0, int end, uint32_t ok, const uint32_t (&qf)[16],
                                          State& S) {
  const int lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
  const bool full = ok == 3u && p0 + kStep <= end;
  float s[2][4];
  bool v0[2], v1[2];  // rows g8 / g8 + 8 of each run count
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const bool run = (ok >> x) & 1u;
    v0[x] = full || (run && p0 + 16 * x + g8 < end);
    v1[x] = full || (run && p0 + 16 * x + g8 + 8 < end);
    const uint32_t kr = st + (16 * x + g8) * kCodeBytes + 4 * t4;
    float ks0[4], ks1[4];
    lds_scales(st + kOffKs + (16 * x + g8) * 8, ks0);
    lds_scales(st + kOffKs + (16 * x + g8 + 8) * 8, ks1);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const uint32_t off = static_cast<uint32_t>(g ^ ((g8 >> 1) & 3)) << 4;
      const uint32_t w0 = lds32(kr + off), w1 = lds32(kr + 8 * kCodeBytes + off);
      float a[4];
      mma_zero(a, codes_lo(w0), codes_lo(w1), codes_hi(w0), codes_hi(w1), qf[4 * g], qf[4 * g + 1]);
      fd::mma_16816(a, codes_lo(w0 >> 8), codes_lo(w1 >> 8), codes_hi(w0 >> 8), codes_hi(w1 >> 8), qf[4 * g + 2],
                    qf[4 * g + 3]);
      if (g == 0) {
        s[x][0] = ks0[0] * a[0];
        s[x][1] = ks0[0] * a[1];
        s[x][2] = ks1[0] * a[2];
        s[x][3] = ks1[0] * a[3];
      } else {
        s[x][0] = fmaf(ks0[g], a[0], s[x][0]);
        s[x][1] = fmaf(ks0[g], a[1], s[x][1]);
        s[x][2] = fmaf(ks1[g], a[2], s[x][2]);
        s[x][3] = fmaf(ks1[g], a[3], s[x][3]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s[x][i] = (i < 2 ? v0[x] : v1[x]) ? s[x][i] * kScaleLog2 : -INFINITY;
  }
  float mx0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2]));
  float mx1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
  }
  const float n0 = fmaxf(S.m0, mx0), n1 = fmaxf(S.m1, mx1);
  if (__any_sync(0xffffffffu, n0 != S.m0 || n1 != S.m1)) {  // some head's max grew
    // a head without a position yet keeps max -inf; its sums are zero
    const float a0 = n0 == -INFINITY ? 1.0f : ex2(S.m0 - n0), a1 = n1 == -INFINITY ? 1.0f : ex2(S.m1 - n1);
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
  const float r0 = n0 == -INFINITY ? 0.0f : n0, r1 = n1 == -INFINITY ? 0.0f : n1;
  const uint32_t sel = (g8 & 1) ? 0x7632u : 0x5410u;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const float e0 = ex2(s[x][0] - r0), e1 = ex2(s[x][1] - r1), e2 = ex2(s[x][2] - r0), e3 = ex2(s[x][3] - r1);
    S.l0 += e0 + e2;
    S.l1 += e1 + e3;
    float vs0[4], vs1[4];
    lds_scales(st + kOffVs + (16 * x + g8) * 8, vs0);
    lds_scales(st + kOffVs + (16 * x + g8 + 8) * 8, vs1);
    // rows that do not count: whatever lies there as a scale, zero
    if (!full) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        vs0[g] = v0[x] ? vs0[g] : 0.0f;
        vs1[g] = v1[x] ? vs1[g] : 0.0f;
      }
    }
    const uint32_t vr = st + kOffV + (16 * x + 2 * t4) * kCodeBytes + 4 * (g8 >> 1);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const uint32_t off = static_cast<uint32_t>(g ^ t4) << 4;
      const uint32_t u = __byte_perm(lds32(vr + off), lds32(vr + kCodeBytes + off), sel);
      const uint32_t w = __byte_perm(lds32(vr + 8 * kCodeBytes + off), lds32(vr + 9 * kCodeBytes + off), sel);
      const uint32_t b0 = fd::movmatrix_t(fd::pack_half2(e0 * vs0[g], e1 * vs0[g]));
      const uint32_t b1 = fd::movmatrix_t(fd::pack_half2(e2 * vs1[g], e3 * vs1[g]));
      fd::mma_16816(S.o[2 * g], codes_lo(u), codes_hi(u), codes_lo(w), codes_hi(w), b0, b1);
      fd::mma_16816(S.o[2 * g + 1], codes_lo(u >> 8), codes_hi(u >> 8), codes_lo(w >> 8), codes_hi(w >> 8), b0, b1);
    }
  }
}

__global__ void __launch_bounds__(kThreads) attn_q4_kernel(const AttnParams P) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  __shared__ Smem S;
  const int split = blockIdx.x, kvh = blockIdx.y, row = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
  const int G = P.n_q / P.c.n_kv;
  int T = P.seq_lens[row];
  if (T > P.max_seq_len || T < 0) {
    if (tid == 0) raise_error(P.c.error, kErrPosition);
    T = T < 0 ? 0 : P.max_seq_len;
  }
  const int start = split * P.chunk, end = min(T, start + P.chunk);
  const int32_t* bt = P.c.bt + static_cast<size_t>(row) * P.c.max_pages;
  int pnew = -1;

  if (P.qkv) {
    const int p = P.pos[row];
    const bool mine = p >= 0 && p == T - 1 && p >= start && p < end;
    if (p != T - 1 && tid == 0) raise_error(P.c.error, kErrPosition);
    const int heads = P.n_q + 2 * P.c.n_kv;
    const __half* src = P.qkv + static_cast<size_t>(row) * heads * kDim;
    if (tid < kDim / 2) rope_cos_sin(p, P.inv_freq[tid], S.cs[tid].x, S.cs[tid].y);
    __syncthreads();
    for (int h = warp; h < G + 2; h += kWarps) {  // the query heads, then K and V of the new position
      if (h >= G && !mine) continue;
      union {
        uint2 u;
        __half x[4];
      } e;
      const int from = h < G ? kvh * G + h : P.n_q + (h - G) * P.c.n_kv + kvh;
      e.u = *reinterpret_cast<const uint2*>(src + from * kDim + 4 * lane);
      if (h <= G) rotate_head(e.x, S.cs, P.style, lane);
      if (h < G) {
        *reinterpret_cast<uint2*>(&S.q[h][4 * lane]) = e.u;
        continue;
      }
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

  const uint32_t ring = smem_u32(&S.stage[warp][0][0]);
  const size_t scale_off = static_cast<size_t>(P.c.page_size) * kCodeBytes;
  // Page of the run at position p (or -1: past the end or a bad page).
  auto page_of = [&](int p) {
    if (p >= end) return -1;
    const int page = __ldg(bt + P.c.page_index(p));
    if (page >= 0 && page < P.c.n_pages) return page;
    if (lane == 0) raise_error(P.c.error, kErrPage);
    return -1;
  };
  // Copies the step at p0 into stage sb; returns the bits of the loaded runs.
  auto load = [&](int p0, int sb, int page0, int page1) {
    const uint32_t st = ring + sb * kStageBytes;
    uint32_t ok = 0u;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int page = x ? page1 : page0;
      if (page < 0) continue;
      ok |= 1u << x;
      const int p = p0 + 16 * x, off = p - P.c.page_index(p) * P.c.page_size;
      const size_t blk = P.c.block(page, kvh);
      const uint8_t* kc = P.c.k + blk + off * kCodeBytes;
      const uint8_t* vc = P.c.v + blk + off * kCodeBytes;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = lane + 32 * j, r = i >> 2;
        const uint32_t d = st + (16 * x + r) * kCodeBytes + (((i & 3) ^ ((r >> 1) & 3)) << 4);
        cp16(d, kc + 16 * i);
        cp16(d + kOffV, vc + 16 * i);
      }
      if (lane < 8) cp16(st + kOffKs + 128 * x + 16 * lane, P.c.k + blk + scale_off + off * 8 + 16 * lane);
      else if (lane < 16)
        cp16(st + kOffVs + 128 * x + 16 * (lane - 8), P.c.v + blk + scale_off + off * 8 + 16 * (lane - 8));
    }
    return ok;
  };

  State A;
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) A.o[mt][0] = A.o[mt][1] = A.o[mt][2] = A.o[mt][3] = 0.0f;
  A.m0 = A.m1 = -INFINITY;
  A.l0 = A.l1 = 0.0f;
  const int first = start + warp * kStep, stride = kWarps * kStep;
  uint32_t ok = first < end ? load(first, 0, page_of(first), page_of(first + 16)) : 0u;
  asm volatile("cp.async.commit_group;" ::: "memory");
  int sb = 0;
  int np0 = page_of(first + stride), np1 = page_of(first + stride + 16);
  for (int p0 = first; p0 < end; p0 += stride) {
    uint32_t next_ok = 0u;
    if (p0 + stride < end) next_ok = load(p0 + stride, sb ^ 1, np0, np1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    np0 = page_of(p0 + 2 * stride);
    np1 = page_of(p0 + 2 * stride + 16);
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
    if (ok) fold_step(st, p0, end, ok, qf, A);
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
  for (int w = tid; w < G * kDim; w += kThreads) {
    const int h = w / kDim, d = w - h * kDim;
    float M = -INFINITY;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) M = fmaxf(M, S.wm[i][h]);
    float num = 0.0f, den = 0.0f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      // a warp without positions has max -inf and sums 0; a NaN score leaves NaN in its sums
      const float f = S.wm[i][h] == -INFINITY ? 1.0f : ex2(S.wm[i][h] - M);
      num = fmaf(S.wo[i][h][d], f, num);
      den = fmaf(S.wl[i][h], f, den);
    }
    const size_t head = static_cast<size_t>(row) * P.n_q + kvh * G + h;
    if (P.n_splits == 1) {
      P.out[head * kDim + d] = __float2half_rn(den == 0.0f ? 0.0f : num / den);
    } else {
      P.part_o[(head * P.n_splits + split) * kDim + d] = num;
      if (d == 0) P.part_ml[head * P.n_splits + split] = make_float2(M, den);
    }
  }
}

// Log-sum-exp merge of the splits of one (row, query head).
__global__ void __launch_bounds__(kDim) attn_q4_combine_kernel(const Partials P) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  const int h = blockIdx.y, row = blockIdx.x, d = threadIdx.x;
  if (P.q_lens && row % P.seq >= P.q_lens[row / P.seq]) return;
  const size_t head = static_cast<size_t>(row) * P.n_q + h, r0 = head * P.n_splits;
  float M = -INFINITY;
  for (int s = 0; s < P.n_splits; ++s) M = fmaxf(M, P.ml[r0 + s].x);
  float num = 0.0f, den = 0.0f;
  for (int s = 0; s < P.n_splits; ++s) {
    const float2 ml = P.ml[r0 + s];
    const float f = ml.x == -INFINITY ? 1.0f : ex2(ml.x - M);
    num = fmaf(P.o[(r0 + s) * kDim + d], f, num);
    den = fmaf(ml.y, f, den);
  }
  P.out[head * kDim + d] = __float2half_rn(den == 0.0f ? 0.0f : num / den);
}

int combine_launch(const Partials& p, int rows, cudaStream_t stream) {
  return lmps_launch_pdl(attn_q4_combine_kernel, dim3(rows, p.n_q), dim3(kDim), 0, stream, p);
}

int check_attention(int n_pages, int max_pages, int page_size, int n_q_heads, int n_kv_heads, int head_dim,
                    int max_seq_len, int n_splits) {
  LMPS_CHECK_ARG(n_pages >= 1 && max_pages >= 1 && page_size >= 1 && max_seq_len >= 1);
  LMPS_CHECK_ARG(static_cast<long long>(max_pages) * page_size <= 1LL << 29);
  LMPS_CHECK_ARG(max_seq_len <= static_cast<long long>(max_pages) * page_size);
  LMPS_CHECK_ARG(n_kv_heads >= 1 && n_q_heads >= 1 && n_q_heads % n_kv_heads == 0 && n_q_heads <= 65535);
  LMPS_CHECK_ARG(n_splits >= 1 && n_splits <= 1024);
  if (head_dim != kDim || page_size % kRun != 0 || n_q_heads / n_kv_heads > kMaxHeads) return LMPS_ERR_UNSUPPORTED;
  return LMPS_OK;
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
  P.chunk = ((max_seq_len + n_splits - 1) / n_splits + kStep - 1) / kStep * kStep;
  const Partials parts = make_partials(workspace, rows, n_q_heads, n_splits, out);
  P.part_o = parts.o;
  P.part_ml = parts.ml;
  cudaStream_t s = lmps_stream(stream);
  const int status = lmps_launch_pdl(attn_q4_kernel, dim3(n_splits, n_kv_heads, rows), dim3(kThreads), 0, s, P);
  if (status || n_splits == 1) return status;
  return combine_launch(parts, rows, s);
}

}  // namespace q4
}  // namespace lmps

using namespace lmps;

extern "C" int lmps_attention_q4_splits(int batch, int n_kv_heads, int max_seq_len) {
  if (batch <= 0 || n_kv_heads <= 0 || max_seq_len <= 0) return 1;
  const long long items = static_cast<long long>(batch) * n_kv_heads;
  const int tiles = (max_seq_len + q4::kWarps * q4::kStep - 1) / (q4::kWarps * q4::kStep);
  long long cap = (4 * 148) / items;
  cap = cap < 1 ? 1 : cap > tiles ? tiles : cap;
  if (cap > 256) cap = 256;
  const int per = static_cast<int>((tiles + cap - 1) / cap);
  return (tiles + per - 1) / per;
}

extern "C" size_t lmps_attention_q4_workspace_size(int batch, int n_q_heads, int head_dim, int n_splits) {
  if (n_splits <= 1 || batch <= 0 || n_q_heads <= 0 || head_dim <= 0) return 0;
  return static_cast<size_t>(batch) * n_q_heads * n_splits * (head_dim * sizeof(float) + sizeof(float2));
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

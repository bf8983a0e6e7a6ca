// Causal attention of many queries a sequence over the paged 4-bit KV cache
// on the 5th-generation tensor cores (tcgen05.mma, S, P and O in tensor
// memory): query i of sequence b, at position starts[b] + i, attends to the
// cached positions 0 .. starts[b] + i.
//
// Rows.  The G query heads of a KV head share its K and V, so a row of the
// score matrix is a (query, head) pair, r = i G + h: any G fills the 128-row
// tiles, and one dequantised K/V tile serves all heads.  A CTA takes 256 rows
// (two M = 128 tiles, t = 0, 1) of one KV head and sequence and walks its
// 128-key tiles:
//   * warps 8-11 (thread = key) read the key's K and V codes, write them as
//     fp16 code * scale -- exact, see kv_q4.cuh -- into two 128-byte-swizzled
//     stages each (K read K-major, V MN-major), loads one tile ahead;
//   * warps 12, 13 (row tile 0, 1) issue S_t = Q_t K^T and O_t += P_t V in half tiles of 64 keys:
//     S has two halves per row tile, so the softmax finds the next one ready
//     while the products behind the last run;
//   * warps 0-3 / 4-7 (thread = row, its TMEM lane) take the softmax of row
//     tile 0 / 1: row max, P = 2^(s - m) as fp16 packed over S's own columns
//     (A operand from tensor memory), sums in fp32, and O rescaled in place
//     only when the max grew by more than 2^8.
// The dims inside a group of 8 stay in the order in which masking the nibbles
// yields them (0 4 1 5 2 6 3 7): Q is staged in that order, and the epilogue
// undoes it for O by naming registers.
// Few rows over a long context are split over the context (grid.y): fp32
// partials, merged by the decode attention's combine kernel.
// Every mbarrier wait is bounded (error bit, no hang).
#include <cmath>

#include "attention_q4.cuh"
#include "tcgen05.cuh"

namespace lmps {
namespace q4 {
namespace pf {

using namespace tc;

constexpr int kRows = 128;  // rows per tile (TMEM lanes)
constexpr int kTiles = 2;   // row tiles per CTA
constexpr int kKeys = 128;  // keys per tile
constexpr int kThreads = 14 * 32;
constexpr int kStages = 2;
constexpr int kSub = 128 * 128;  // 64 dims of 128 rows or keys: 128-byte rows
constexpr int kOffK = kTiles * 2 * kSub;
constexpr int kOffV = kOffK + kStages * 2 * kSub;
constexpr int kOffBar = kOffV + kStages * 2 * kSub;
constexpr int kSmemBytes = kOffBar + 256 + 1024;  // barriers, flags; 1024-byte alignment slack
constexpr uint32_t kTmemCols = 512;
constexpr int kHalf = 64;        // keys per softmax step: half a key tile
constexpr uint32_t kColS = 0;    // S of row tile t, half u at columns 64 (2 t + u); P over its first 32
constexpr uint32_t kColO = 256;  // O of row tile t at columns 256 + 128 t
constexpr float kRescaleLog2 = 8.0f;

struct Params {
  const __half* q;  // [batch * seq, n_q * 128]
  Cache c;
  const int32_t* starts;
  const int32_t* q_lens;
  __half* out;
  float* part_o;
  float2* part_ml;
  int n_q, G, seq, n_blocks, n_splits, max_seq_len;
};

// One MMA with its descriptors' low words computed by the caller: within a
// 128-byte-swizzled tile only the address field moves (it never carries out
// of its 14 bits), so a step costs an add, not a descriptor.
__device__ __forceinline__ uint64_t desc(uint32_t lo, uint32_t hi) {
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
// D += A B with A (fp16) in tensor memory.
__device__ __forceinline__ void mma_f16_ta(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}

// Bounded wait that raises the timeout bit and the CTA's abort flag.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int32_t* err, volatile int* abort_flag) {
  if (mbar_try(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  while (!mbar_try(bar, parity)) {
    if (*abort_flag) return false;
    if (globaltimer() - t0 > kTimeoutNs) {
      raise_error(err, kErrTimeout);
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, int32_t* err, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, wait(bar, parity, err, abort_flag));
}

// One word of codes (8 dims) times its scale: 16 bytes in mask order.
__device__ __forceinline__ uint4 dequant_word(uint32_t w, __half2 s) {
  uint4 r;
  uint32_t c[4] = {codes_lo(w), codes_hi(w), codes_lo(w >> 8), codes_hi(w >> 8)};
  uint32_t* d = &r.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&c[i]), s);
    d[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return r;
}
__device__ __forceinline__ __half scale_of(uint2 s, int g) {
  const uint32_t w = g < 2 ? s.x : s.y;
  return __ushort_as_half(static_cast<unsigned short>(g & 1 ? w >> 16 : w & 0xFFFFu));
}
// Whether any of four fp16 numbers is not finite (exponent bits all ones).
__device__ __forceinline__ bool any_not_finite(uint2 s) {
  return ((((s.x & 0x7C007C00u) + 0x04000400u) | ((s.y & 0x7C007C00u) + 0x04000400u)) & 0x80008000u) != 0u;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two fp32 numbers in a register pair: one instruction for both.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
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

template <int N>
struct Int {
  static constexpr int value = N;
};
struct Raw {  // a key's cached rows
  uint4 k[4], v[4];
  uint2 ks, vs;
};

__global__ void __launch_bounds__(kThreads, 1) prefill_q4_kernel(const __grid_constant__ Params P) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* sq = base;
  unsigned char* sk = base + kOffK;
  unsigned char* sv = base + kOffV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + kOffBar);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;   // [kStages]
  uint64_t* k_empty = bars + 3;
  uint64_t* v_full = bars + 5;
  uint64_t* v_empty = bars + 7;
  uint64_t* s_full = bars + 9;   // [kTiles][2]: S of the row tile and half ready
  uint64_t* p_full = bars + 13;  // P written (and S read)
  uint64_t* o_done = bars + 17;  // O += P V done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 21);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* abort_v = abort_flag;
  uint32_t* absent = tmem_slot + 4;  // [4][4]: keys of a tile whose page is not in the pool, ring of 4 tiles

  lmps_pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  lmps_pdl_wait();
  // this CTA's rows: the last (longest) row blocks first
  const int per_block = static_cast<int>(gridDim.x) / P.n_blocks;
  const int blk = P.n_blocks - 1 - static_cast<int>(blockIdx.x) / per_block;
  const int rest = static_cast<int>(blockIdx.x) % per_block;
  const int kvh = rest % P.c.n_kv, b = rest / P.c.n_kv, split = blockIdx.y;
  const int n_queries = min(P.seq, P.q_lens ? P.q_lens[b] : P.seq);
  const int n_rows = n_queries * P.G, r0 = blk * kTiles * kRows;
  if (r0 >= n_rows) return;  // (uniform)
  const int n_t = n_rows - r0 > kRows ? 2 : 1;  // row tiles in use
  const long long first = P.starts ? P.starts[b] : 0;
  const int i_last = (min(n_rows, r0 + n_t * kRows) - 1) / P.G;
  // positions that row i may see, inside the cache
  auto limit = [&](int i) {
    const long long n = first + i + 1;
    return static_cast<int>(n < 0 ? 0 : n > P.max_seq_len ? P.max_seq_len : n);
  };
  if (tid == 0 && split == 0 && (first < 0 || first + i_last + 1 > P.max_seq_len)) raise_error(P.c.error, kErrPosition);
  const int kv_end = limit(i_last);
  const int all_tiles = (kv_end + kKeys - 1) / kKeys;
  const int per_split = (all_tiles + P.n_splits - 1) / P.n_splits;
  const int tile0 = min(all_tiles, split * per_split), nt = min(all_tiles, tile0 + per_split) - tile0;
  const int nh = min(2 * nt, (kv_end - tile0 * kKeys + kHalf - 1) / kHalf);  // softmax steps: half tiles with keys

  if (tid == 0) {
    mbar_init(q_full, 8);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&v_full[s], 4);
      mbar_init(&k_empty[s], n_t);
      mbar_init(&v_empty[s], n_t);
    }
    for (int t = 0; t < 2 * kTiles; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot, tmem_u = __shfl_sync(0xffffffffu, tmem, 0);

  if (warp >= 8 && warp < 12) {
    // ---- dequantisation: thread = key
    const int key = tid - 256;
    const int32_t* bt = P.c.bt + static_cast<size_t>(b) * P.c.max_pages;
    const size_t scale_off = static_cast<size_t>(P.c.page_size) * kCodeBytes;
    auto page_of = [&](int i) {  // page of this thread's key in local tile i; -1 past the end, -2 outside the pool
      const int p = (tile0 + i) * kKeys + key;
      if (i >= nt || p >= kv_end) return -1;
      const int page = __ldg(bt + P.c.page_index(p));
      return page >= 0 && page < P.c.n_pages ? page : -2;
    };
    auto fetch = [&](int i, int page, Raw& r) {
      if (page < 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r.k[j] = r.v[j] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
        r.ks = r.vs = make_uint2(0u, 0u);
        return;
      }
      const int p = (tile0 + i) * kKeys + key, off = p - P.c.page_index(p) * P.c.page_size;
      const size_t o = P.c.block(page, kvh);
      const uint4* kc = reinterpret_cast<const uint4*>(P.c.k + o + off * kCodeBytes);
      const uint4* vc = reinterpret_cast<const uint4*>(P.c.v + o + off * kCodeBytes);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        r.k[j] = __ldg(kc + j);
        r.v[j] = __ldg(vc + j);
      }
      r.ks = __ldg(reinterpret_cast<const uint2*>(P.c.k + o + scale_off + off * 8));
      r.vs = __ldg(reinterpret_cast<const uint2*>(P.c.v + o + scale_off + off * 8));
    };
    auto write = [&](unsigned char* dst, const uint4 (&c)[4], uint2 s, float fix) {
      // row `key`, 16-byte chunk x of a 64-dim half at x ^ (key & 7)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const __half2 hs = __half2half2(__float2half_rn(__half2float(scale_of(s, g)) * fix));
        const uint32_t* w = &c[g].x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int ch = 4 * (g & 1) + j;
          *reinterpret_cast<uint4*>(dst + (g >> 1) * kSub + key * 128 + ((ch ^ (key & 7)) << 4)) = dequant_word(w[j], hs);
        }
      }
    };
    Raw cur;
    int page = page_of(0), next_page = page_of(1);
    fetch(0, page, cur);
    bool ok = true;
    for (int i = 0; ok && i < nt; ++i) {
      const int s = i & 1;
      const uint32_t gone = __ballot_sync(0xffffffffu, page == -2);
      if (gone && lane == 0) raise_error(P.c.error, kErrPage);
      // the next tile's loads go out before this one's arithmetic
      const Raw r = cur;
      page = next_page;
      fetch(i + 1, page, cur);
      next_page = page_of(i + 2);
      // a row with a scale that is not finite: NaN scores for whoever attends to it, and zeros
      // as V, which P = 0 of the others meets
      const bool poison = any_not_finite(r.vs);
      if (i >= kStages) ok = wait_warp(&k_empty[s], ((i >> 1) - 1) & 1, P.c.error, abort_v);
      if (!ok) break;
      // ring of 4: slot i & 3 is free, since K's stage is (S of tile i - 2 done, so the softmax of
      // tile i - 3, and with it tile i - 4, is)
      if (lane == 0) absent[4 * (i & 3) + warp - 8] = gone;
      write(sk + s * 2 * kSub, r.k, r.ks, poison ? __int_as_float(0x7FC00000) : 1.0f);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[s]);
      if (i >= kStages) ok = wait_warp(&v_empty[s], ((i >> 1) - 1) & 1, P.c.error, abort_v);
      if (!ok) break;
      write(sv + s * 2 * kSub, r.v, poison ? make_uint2(0u, 0u) : r.vs, 1.0f);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[s]);
    }
  } else if (warp >= 12) {
    // ---- MMA issuers, a warp per row tile: while one waits for its softmax (some 200 cycles from
    // the barrier to the next MMA) the other's products run.  The whole warp runs the code and one
    // elected lane issues: uniform, with tiles and stages unrolled, it keeps the descriptors in
    // uniform registers.  (Issued from a divergent branch an MMA costs some ten instructions, and on
    // a scheduler shared with three busy warps they came 110 .. 130 cycles apart, not 64.)
    uint32_t elected;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(elected));
    const bool leader = elected != 0u;
    const uint32_t id_s = idesc_f16(kRows, kHalf), id_o = idesc_f16(kRows, kDim) | kBMajorMN;
    const uint64_t dk = sw128_desc(smem_u32(sk)), dv = sw128_mn_desc(smem_u32(sv), kSub);
    const uint32_t hi_k = static_cast<uint32_t>(dk >> 32), hi_v = static_cast<uint32_t>(dv >> 32);
    const uint32_t lo_q = static_cast<uint32_t>(sw128_desc(smem_u32(sq))), lo_k = static_cast<uint32_t>(dk),
                   lo_v = static_cast<uint32_t>(dv);
    constexpr uint32_t kNext = kSub >> 4;  // the next 64 dims
    auto after = [] { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); };
    auto run = [&](auto tile) {
      constexpr int t = decltype(tile)::value;
      auto issue_s = [&](int s, int u) {  // S_t,u = Q_t K_u^T over 8 steps of 16 dims
        if (leader) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t o = (j >> 2) * kNext + 2 * (j & 3);
            mma_f16(tmem_u + kColS + kHalf * (2 * t + u), desc(lo_q + 2 * t * kNext + o, hi_k),
                    desc(lo_k + 2 * s * kNext + u * (kHalf * 128 >> 4) + o, hi_k), id_s, j > 0 ? 1u : 0u);
          }
          mma_commit(&s_full[2 * t + u]);
        }
      };
      auto issue_o = [&](int s, int u, bool acc) {  // O_t += P_t,u V_u over 4 steps of 16 keys
        if (leader) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_f16_ta(tmem_u + kColO + kDim * t, tmem_u + kColS + kHalf * (2 * t + u) + 8 * j,
                       desc(lo_v + 2 * s * kNext + 128 * (4 * u + j), hi_v), id_o, (acc || j > 0) ? 1u : 0u);
          mma_commit(&o_done[2 * t + u]);
        }
      };
      bool ok = wait_warp(q_full, 0, P.c.error, abort_v) && wait_warp(&k_full[0], 0, P.c.error, abort_v);
      if (ok) {
        after();
        issue_s(0, 0);
        if (nh > 1) issue_s(0, 1);
        if (leader) mma_commit(&k_empty[0]);
      }
      // step i, half u of key tile j in stage s: O, then S of the same half of the next tile
      auto step = [&](int i, auto stage, auto half) {
        constexpr int s = decltype(stage)::value, s1 = s ^ 1, u = decltype(half)::value;
        const int j = i >> 1;
        const bool more = i + 2 < nh;
        if (u == 0) ok = wait_warp(&v_full[s], (j >> 1) & 1, P.c.error, abort_v);
        if (u == 0 && more) ok = ok && wait_warp(&k_full[s1], ((j + 1) >> 1) & 1, P.c.error, abort_v);
        ok = ok && wait_warp(&p_full[2 * t + u], j & 1, P.c.error, abort_v);
        if (!ok) return;
        after();
        issue_o(s, u, i > 0);
        if (more) issue_s(s1, u);  // (P, under S's columns, is read by the P V before it in the issue order)
        if (u == 1 && leader) {
          mma_commit(&v_empty[s]);
          if (more) mma_commit(&k_empty[s1]);
        }
      };
      for (int i = 0; ok && i < nh; i += 4) {
        step(i, Int<0>{}, Int<0>{});
        if (ok && i + 1 < nh) step(i + 1, Int<0>{}, Int<1>{});
        if (ok && i + 2 < nh) step(i + 2, Int<1>{}, Int<0>{});
        if (ok && i + 3 < nh) step(i + 3, Int<1>{}, Int<1>{});
      }
    };
    if (nh > 0) {
      if (warp == 12) run(Int<0>{});
      else if (n_t > 1) run(Int<1>{});
    }
  } else {
    // ---- softmax of row tile t: thread = row (TMEM lane)
    const int t = warp >> 2, quad = warp & 3, rl = 32 * quad + lane, r = r0 + kRows * t + rl;
    {  // stage Q: 16 lanes a row, dims of each 8 in mask order
      const int c = lane & 15;
#pragma unroll 1
      for (int x0 = 0; x0 < 32; x0 += 16) {
        uint4 v[8];  // loads of 16 rows in flight
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int rr = r0 + kRows * t + 32 * quad + x0 + 2 * x + (lane >> 4);
          v[x] = make_uint4(0u, 0u, 0u, 0u);
          if (rr < n_rows) {
            const int i = rr / P.G, h = rr - i * P.G;
            v[x] = __ldg(reinterpret_cast<const uint4*>(P.q + (static_cast<size_t>(b) * P.seq + i) * P.n_q * kDim +
                                                        (kvh * P.G + h) * kDim) + c);
          }
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int row = 32 * quad + x0 + 2 * x + (lane >> 4);
          const uint4 m = make_uint4(__byte_perm(v[x].x, v[x].z, 0x5410), __byte_perm(v[x].x, v[x].z, 0x7632),
                                     __byte_perm(v[x].y, v[x].w, 0x5410), __byte_perm(v[x].y, v[x].w, 0x7632));
          *reinterpret_cast<uint4*>(sq + (2 * t + (c >> 3)) * kSub + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = m;
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    if (t < n_t) {
      const uint32_t tl = tmem + (static_cast<uint32_t>(32 * quad) << 16);
      const uint32_t to = tl + kColO + kDim * t;
      const int qi = r / P.G;
      const int lim = r < n_rows ? limit(qi) : kv_end;
      const int lim_min = limit((r0 + kRows * t) / P.G);
      float m_used = -INFINITY, l = 0.0f;  // running max (scaled, base 2) and sum
      bool ok = true;
      for (int i = 0; ok && i < nh; ++i) {
        const int u = i & 1, j = i >> 1, k0 = tile0 * kKeys + i * kHalf;
        const uint32_t ts = tl + kColS + kHalf * (2 * t + u);
        ok = wait_warp(&s_full[2 * t + u], j & 1, P.c.error, abort_v);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t sc[64];
        tmem_ld64(ts, sc);
        const volatile uint32_t* av = absent + 4 * (j & 3) + 2 * u;
        const uint32_t gone[2] = {av[0], av[1]};
        if (k0 + kHalf > lim_min || (gone[0] | gone[1]) != 0u) {  // (uniform)
          const int nv = lim - k0;  // columns below it count
#pragma unroll
          for (int c = 0; c < kHalf; ++c)
            if (c >= nv || ((gone[c >> 5] >> (c & 31)) & 1u)) sc[c] = 0xFF800000u;  // -inf
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kHalf; c += 2)
          mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], __uint_as_float(sc[c]), __uint_as_float(sc[c + 1]));
        const float mt = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * kScaleLog2;
        const float mnew = fmaxf(m_used, mt);
        const bool grow = mnew > m_used + kRescaleLog2;  // (always on a row's first positions)
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? ex2(m_used - mnew) : 1.0f;
          if (i > 0) {  // warp-wide read-modify-write of O_t, once the P V of the step before is done
            ok = wait_warp(&o_done[2 * t + (u ^ 1)], ((i - 1) >> 1) & 1, P.c.error, abort_v);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int cc = 0; cc < kDim; cc += 32) {
              uint32_t o[32];
              tmem_ld32(to + cc, o);
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
              tmem_st32(to + cc, o);
            }
          }
          l *= alpha;
          if (grow) m_used = mnew;
        }
        const float nm = m_used == -INFINITY ? 0.0f : -m_used;
        const uint64_t nm2 = pair(nm, nm), scale2 = pair(kScaleLog2, kScaleLog2);
        uint64_t sm[4] = {0ull, 0ull, 0ull, 0ull};
        uint32_t pk[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          float a0, a1;
          const uint64_t x = fma2(pair(__uint_as_float(sc[2 * e]), __uint_as_float(sc[2 * e + 1])), scale2, nm2);
          unpair(x, a0, a1);
          a0 = ex2(a0);
          a1 = ex2(a1);
          sm[e & 3] = add2(sm[e & 3], pair(a0, a1));
          const __half2 hh = __floats2half2_rn(a0, a1);
          pk[e] = *reinterpret_cast<const uint32_t*>(&hh);
        }
        tmem_st32(ts, pk);
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + u]);
        float s0, s1;
        unpair(add2(add2(sm[0], sm[1]), add2(sm[2], sm[3])), s0, s1);
        l += s0 + s1;
      }
      // ---- epilogue: this row of O (dims of each 8 back in order), normalised or as a partial
      if (ok && nh > 0) ok = wait_warp(&o_done[2 * t + ((nh - 1) & 1)], ((nh - 1) >> 1) & 1, P.c.error, abort_v);
      if (ok) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int h = r - qi * P.G;
        const size_t head = (static_cast<size_t>(b) * P.seq + qi) * P.n_q + kvh * P.G + h;
        const size_t part = ((static_cast<size_t>(b) * P.seq + qi) * P.n_splits + split) * P.n_q + kvh * P.G + h;
        if (P.n_splits > 1 && r < n_rows) P.part_ml[part] = make_float2(m_used, l);
#pragma unroll 1
        for (int cc = 0; cc < kDim; cc += 32) {
          uint32_t o[32];
          if (nh > 0) {
            tmem_ld32(to + cc, o);
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = 0u;
          }
          if (r < n_rows) {
            constexpr int at[8] = {0, 2, 4, 6, 1, 3, 5, 7};  // where dim e of a group of 8 is
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              float v[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(o[8 * g + at[e]]);
              if (P.n_splits == 1) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const __half2 hh = __floats2half2_rn(v[2 * e] * inv, v[2 * e + 1] * inv);
                  w[e] = *reinterpret_cast<const uint32_t*>(&hh);
                }
                *reinterpret_cast<uint4*>(P.out + head * kDim + cc + 8 * g) = make_uint4(w[0], w[1], w[2], w[3]);
              } else {
                float4* dst = reinterpret_cast<float4*>(P.part_o + part * kDim + cc + 8 * g);
                dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                dst[1] = make_float4(v[4], v[5], v[6], v[7]);
              }
            }
          }
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 12)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

}  // namespace pf
}  // namespace q4
}  // namespace lmps

using namespace lmps;

extern "C" int lmps_prefill_q4_splits(int batch, int seq_len, int n_q_heads, int n_kv_heads, int max_seq_len) {
  if (batch <= 0 || seq_len <= 0 || n_kv_heads <= 0 || n_q_heads < n_kv_heads || max_seq_len <= 0) return 1;
  const long long rows = static_cast<long long>(seq_len) * (n_q_heads / n_kv_heads);
  const long long items = (rows + 255) / 256 * n_kv_heads * batch;
  const int tiles = (max_seq_len + 127) / 128;
  long long cap = 2 * 148 / items;
  cap = cap < 1 ? 1 : cap > tiles ? tiles : cap;
  if (cap > 64) cap = 64;
  const int per = static_cast<int>((tiles + cap - 1) / cap);
  return (tiles + per - 1) / per;
}

extern "C" size_t lmps_prefill_q4_workspace_size(int batch, int seq_len, int n_q_heads, int head_dim, int n_splits) {
  if (seq_len <= 0) return 0;
  return seq_len * lmps_attention_q4_workspace_size(batch, n_q_heads, head_dim, n_splits);
}

extern "C" int lmps_prefill_attention_q4(const uint16_t* q, const uint8_t* k_pool, const uint8_t* v_pool,
                                         int n_pages, const int32_t* block_table, const int32_t* starts,
                                         const int32_t* q_lens, uint16_t* out, void* workspace,
                                         size_t workspace_bytes, int max_pages, int page_size, int n_q_heads,
                                         int n_kv_heads, int head_dim, int batch, int seq_len, int max_seq_len,
                                         int n_splits, int32_t* error, void* stream) {
  namespace pf = q4::pf;
  LMPS_CHECK_ARG(q && k_pool && v_pool && block_table && out && error && batch >= 1 && seq_len >= 1);
  const int st = q4::check_attention(n_pages, max_pages, page_size, n_q_heads, n_kv_heads, head_dim, max_seq_len,
                                     n_splits);
  if (st != LMPS_OK) return st;
  LMPS_CHECK_ARG(lmps_aligned(q, 16) && lmps_aligned(k_pool, 16) && lmps_aligned(v_pool, 16) &&
                 lmps_aligned(out, 16) && lmps_aligned(workspace, 16));
  const long long rows = static_cast<long long>(batch) * seq_len;
  const long long G = n_q_heads / n_kv_heads;
  const long long blocks = (seq_len * G + pf::kTiles * pf::kRows - 1) / (pf::kTiles * pf::kRows);
  const long long items = blocks * n_kv_heads * batch;
  if (rows > 0x7FFFFFFFLL || seq_len * G > 0x7FFFFF00LL || items > 0x7FFFFFFFLL) return LMPS_ERR_UNSUPPORTED;
  const size_t need = lmps_prefill_q4_workspace_size(batch, seq_len, n_q_heads, head_dim, n_splits);
  if (need > 0 && (!workspace || workspace_bytes < need)) return LMPS_ERR_WORKSPACE;
  q4::Partials parts = q4::make_partials(workspace, static_cast<int>(rows), n_q_heads, n_splits, out);
  parts.q_lens = q_lens;
  parts.seq = seq_len;
  pf::Params P{};
  P.q = reinterpret_cast<const __half*>(q);
  P.c = q4::Cache{k_pool, v_pool, block_table, n_pages, max_pages, page_size, n_kv_heads,
                  q4::page_shift_of(page_size), error};
  P.starts = starts;
  P.q_lens = q_lens;
  P.out = reinterpret_cast<__half*>(out);
  P.part_o = parts.o;
  P.part_ml = parts.ml;
  P.n_q = n_q_heads;
  P.G = static_cast<int>(G);
  P.seq = seq_len;
  P.n_blocks = static_cast<int>(blocks);
  P.n_splits = n_splits;
  P.max_seq_len = max_seq_len;
  const int st_attr = lmps_max_dyn_smem<pf::prefill_q4_kernel>(pf::kSmemBytes);
  if (st_attr != LMPS_OK) return st_attr;
  cudaStream_t s = lmps_stream(stream);
  const int status = lmps_launch_pdl(pf::prefill_q4_kernel, dim3(static_cast<unsigned>(items), n_splits),
                                     dim3(pf::kThreads), static_cast<size_t>(pf::kSmemBytes), s, P);
  if (status || n_splits == 1) return status;
  return q4::combine_launch(parts, static_cast<int>(rows), s);
}

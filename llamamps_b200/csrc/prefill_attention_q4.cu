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
//   * warp 14 brings a tile's cached rows to shared memory (bulk copies);
//   * warps 8-11 write its K and V as fp16 code * scale -- exact, see kv_q4.cuh
//     -- into two 128-byte-swizzled stages each (K read K-major, V MN-major);
//   * warps 12, 13 (row tile 0, 1) issue S_t = Q_t K^T and O_t += P_t V in half
//     tiles of 64 keys: S has two halves per row tile, so the softmax finds the
//     next one ready while the products behind the last run;
//   * warps 0-3 / 4-7 (thread = row, its TMEM lane) take the softmax of row
//     tile 0 / 1: row max, P = 2^(s - m) as fp16 packed over S's own columns
//     (A operand from tensor memory), sums in fp32, and O rescaled in place
//     only when the max grew by more than 2^8.
// The dims inside a group of 8 stay in the order in which masking the nibbles
// yields them (0 4 1 5 2 6 3 7): Q is staged in that order, and the epilogue
// undoes it for O by naming registers.
// Few rows over a long context are cut into pieces of equal length along it:
// fp32 partials, merged by a second kernel.  Units of work go to 148 persistent
// CTAs, from the longest rows to the shortest, forwards and backwards in turn.
// Every mbarrier wait is bounded (error bit, no hang).
//
// What bounds it: not the tensor core.  A 256 x 128 tile has 2048 cycles of
// products and takes about 4200: the softmax of 64 keys is a chain of one TMEM
// load, 64 exponentials a thread, conversions and a TMEM store, and the four
// dequantising warps share its schedulers.  Measured (12 query, 2 KV heads):
// 8 x 2048 causal 155 us = 665 TFLOP/s, 0.40 of the bf16 peak measured by a
// library product; 4 x 256 queries behind 1..30000 positions 81 us; one
// prompt of 37 tokens 8 us.  Tried without gain: exponentials by polynomial on
// the FMA units for a part of a row, the two softmax groups held half a step
// apart, the next unit's queries fetched during the epilogue (64 registers, spilled).
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
constexpr int kThreads = 15 * 32;
constexpr int kStages = 2;
constexpr int kSub = 128 * 128;  // 64 dims of 128 rows or keys: 128-byte rows
constexpr int kOffK = kTiles * 2 * kSub;
constexpr int kOffV = kOffK + kStages * 2 * kSub;
constexpr int kOffRaw = kOffV + kStages * 2 * kSub;  // a tile as cached: K codes, V codes, K scales, V scales
constexpr int kRawV = kKeys * kCodeBytes, kRawKs = 2 * kRawV, kRawVs = kRawKs + kKeys * 8;
constexpr int kOffBar = kOffRaw + kRawVs + kKeys * 8;
constexpr int kSmemBytes = kOffBar + 512 + 1024;  // barriers, flags; 1024-byte alignment slack
constexpr uint32_t kTmemCols = 512;
constexpr int kHalf = 64;        // keys per softmax step: half a key tile
constexpr uint32_t kColS = 0;    // S of row tile t, half u at columns 64 (2 t + u); P over its first 32
constexpr uint32_t kColO = 256;  // O of row tile t at columns 256 + 128 t
constexpr float kRescaleLog2 = 8.0f;
// P is held times 2^7 (below 2^15 with the above): in a long flat softmax most weights lie 2^-13 and
// less under the largest, where fp16 would lose bits to its subnormals.
constexpr float kPBias = 7.0f;
constexpr int kSms = 148;  // one CTA per SM

struct Params {
  const __half* q;  // [batch * seq, n_q * 128]
  Cache c;
  const int32_t* starts;
  const int32_t* q_lens;
  __half* out;
  float* part_o;   // with n_splits > 1: Partials of BlockPieces
  float2* part_ml;
  int2* pieces;    // first piece and their number, per (row block, sequence)
  int n_q, G, seq, batch, n_blocks, n_splits, max_seq_len, rows_item;
  uint32_t by_G, by_kv, by_batch;  // reciprocals for quotient()
};

// n / d by the reciprocal floor(2^32 / d) + 1 (0 stands for d = 1): exact for n < 2^29 and d <= 8, and
// for n d < 2^32, since the reciprocal is too large by less than 1 and n times that stays below 2^32 / d.
__device__ __forceinline__ int quotient(int n, uint32_t by) {
  return by ? static_cast<int>(__umulhi(static_cast<uint32_t>(n), by)) : n;
}

// One unit of work: a row block of a KV head and sequence, and the key tiles of it that are taken.
struct Work {
  int b, kvh, r0, n_rows, n_t;  // first row, rows of the sequence, row tiles in use
  int first;                    // position of query 0 (clamped)
  int kv_end, tile0, nt, nh;    // keys that count; first key tile, tiles, half tiles with keys
  int piece;
  bool found;
};

// Positions that query i may see, inside the cache.
__device__ __forceinline__ int limit(const Params& P, int first, int i) {
  return max(0, min(first + i + 1, P.max_seq_len));
}
// Rows of sequence b, and its first position.
__device__ __forceinline__ void sequence(const Params& P, int b, int& n_rows, int& first) {
  n_rows = max(0, min(P.seq, P.q_lens ? __ldg(P.q_lens + b) : P.seq)) * P.G;
  // (a start outside the cache is reported; clamped, so that sums of positions stay in range)
  first = P.starts ? max(-(1 << 30), min(__ldg(P.starts + b), 1 << 30)) : 0;
}
__device__ __forceinline__ int last_query(const Params& P, int n_rows, int r0) {
  return quotient(min(n_rows, r0 + kTiles * kRows) - 1, P.by_G);
}
// Key tiles of entry e = (row block from the last, sequence); -1: no rows.
__device__ __forceinline__ int entry_tiles(const Params& P, int e) {
  const int from_last = quotient(e, P.by_batch), r0 = (P.n_blocks - 1 - from_last) * kTiles * kRows;
  int n_rows, first;
  sequence(P, e - from_last * P.batch, n_rows, first);
  if (r0 >= n_rows) return -1;
  return (limit(P, first, last_query(P, n_rows, r0)) + kKeys - 1) / kKeys;
}
// Pieces of `cut` tiles that an entry is cut into.
__device__ __forceinline__ int entry_pieces(int tiles, int cut) { return tiles < 0 ? 0 : max(1, (tiles + cut - 1) / cut); }

// Tiles per piece: the fewest (in steps of a sixteenth) with which the pieces of all entries fit
// n_splits per entry.  A warp computes it; the tiles of the first 32 entries stay in its registers.
__device__ __forceinline__ int piece_tiles(const Params& P) {
  const int entries = P.n_blocks * P.batch, lane = threadIdx.x & 31;
  const int room = P.n_splits * entries;
  const int own = lane < entries ? entry_tiles(P, lane) : -1;
  int total = max(0, own);
  for (int e = lane + kWarp; e < entries; e += kWarp) total += max(0, entry_tiles(P, e));
  total = __reduce_add_sync(0xffffffffu, total);
  int cut = max(1, (total + room - 1) / room);
  for (;;) {  // ends: with `cut` at the longest entry every entry is one piece
    int n = entry_pieces(own, cut);
    for (int e = lane + kWarp; e < entries; e += kWarp) n += entry_pieces(entry_tiles(P, e), cut);
    n = __reduce_add_sync(0xffffffffu, n);
    if (n <= room || cut > total) return cut;
    cut += max(1, cut >> 4);
  }
}

// Work unit `item` (a warp looks it up; uniform).  Without splits the row blocks go from the last (longest)
// to the first; with splits the pieces are numbered over the entries in order.
__device__ __forceinline__ Work locate(const Params& P, int item, int cut) {
  Work w{};
  w.found = true;
  int e;
  int j = 0;
  const int unit = quotient(item, P.by_kv);
  w.kvh = item - unit * P.c.n_kv;
  if (P.n_splits == 1) {
    e = unit;
  } else {
    const int lane = threadIdx.x & 31, entries = P.n_blocks * P.batch;
    w.piece = unit;
    int before = 0;
    w.found = false;
    e = 0;
    for (int e0 = 0; e0 < entries && !w.found; e0 += kWarp) {
      const int mine = e0 + lane < entries ? entry_pieces(entry_tiles(P, e0 + lane), cut) : 0;
      int sum = mine;  // inclusive prefix
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, w.piece < before + sum);
      if (hit) {
        const int l = __ffs(hit) - 1;
        e = e0 + l;
        before += __shfl_sync(0xffffffffu, sum - mine, l);
        j = w.piece - before;
        w.found = true;
        const int n = __shfl_sync(0xffffffffu, mine, l);
        if (threadIdx.x == 0 && w.kvh == 0 && j == 0) P.pieces[e] = make_int2(before, n);
      } else {
        before += __shfl_sync(0xffffffffu, sum, 31);
      }
    }
    if (!w.found) return w;
  }
  const int from_last = quotient(e, P.by_batch);
  w.b = e - from_last * P.batch;
  w.r0 = (P.n_blocks - 1 - from_last) * kTiles * kRows;
  sequence(P, w.b, w.n_rows, w.first);
  if (w.r0 >= w.n_rows) return w;  // nothing to do: n_t = 0
  w.n_t = w.n_rows - w.r0 > kRows ? 2 : 1;
  w.kv_end = limit(P, w.first, last_query(P, w.n_rows, w.r0));
  const int all = (w.kv_end + kKeys - 1) / kKeys;
  if (P.n_splits == 1) {
    w.nt = all;
  } else {
    w.tile0 = j * cut;
    w.nt = min(cut, all - w.tile0);
  }
  w.nh = min(2 * w.nt, (w.kv_end - w.tile0 * kKeys + kHalf - 1) / kHalf);
  return w;
}

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
// Untiled bulk copy of `bytes` (a multiple of 16, both addresses 16-byte aligned) to shared memory.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
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
__global__ void __launch_bounds__(kThreads, 1) prefill_q4_kernel(const __grid_constant__ Params P) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* sq = base;
  unsigned char* sk = base + kOffK;
  unsigned char* sv = base + kOffV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + kOffBar);
  uint64_t* q_full = bars;          // [kTiles]
  uint64_t* k_full = bars + 2;      // [kStages]
  uint64_t* k_empty = bars + 4;
  uint64_t* v_full = bars + 6;
  uint64_t* v_empty = bars + 8;
  uint64_t* s_full = bars + 10;     // [kTiles][2]: S of the row tile and half ready
  uint64_t* p_full = bars + 14;     // P written (and S read)
  uint64_t* o_done = bars + 18;     // O += P V done
  uint64_t* raw_full = bars + 22;   // cached rows of a tile landed
  uint64_t* raw_empty = bars + 23;  // and read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* abort_v = abort_flag;
  uint32_t* absent = tmem_slot + 2;    // [4][4]: keys of a tile whose page is not in the pool, ring of 4 tiles
  uint32_t* absent_raw = absent + 16;  // [4]: of the tile in the raw stage
  volatile int* cut_slot = reinterpret_cast<int*>(absent_raw + 4);

  lmps_pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int t = 0; t < kTiles; ++t) mbar_init(&q_full[t], 4);
    mbar_init(raw_full, 1);
    mbar_init(raw_empty, 4);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&v_full[s], 4);
      mbar_init(&k_empty[s], kTiles);
      mbar_init(&v_empty[s], kTiles);
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
  lmps_pdl_wait();
  if (P.n_splits > 1) {  // (uniform) one warp looks the lengths over
    if (warp == 14) {
      const int c = piece_tiles(P);
      if (lane == 0) *cut_slot = c;
    }
    __syncthreads();
  }

  // Every role walks the same work units; stages, S halves and their barriers' phases run on over them.
  const int n_items = P.n_blocks * P.batch * P.n_splits * P.c.n_kv;
  const int cut = P.n_splits > 1 ? *cut_slot : 0;
  // the CTA's units: every gridDim.x-th, odd rounds in reverse (units are ordered by size)
  auto nth = [&](int turn) {
    return turn * static_cast<int>(gridDim.x) +
           ((turn & 1) ? static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x));
  };
  int32_t* const err = P.c.error;
  bool ok = true;
  if (warp >= 8 && warp < 12) {
    // ---- dequantisation.  A warp takes 32 keys of a tile as 4 units of 8 consecutive keys; a lane
    // holds one group of 32 dims of one key.  So a unit is 512 contiguous bytes of codes, and the
    // lanes of each quarter warp (4 keys, two adjacent groups) write to 8 different 16-byte columns.
    const int w = warp - 8, kk = ((lane >> 1) & 3) + ((lane >> 4) << 2), g = 2 * ((lane >> 3) & 1) + (lane & 1);
    const unsigned char* raw = base + kOffRaw;
    // codes * scale to row `key` of a tile, 16-byte chunk x of a 64-dim half at x ^ (key & 7)
    auto write = [&](unsigned char* tile, const uint4 (&c)[4], const uint32_t (&s)[4]) {
      unsigned char* dst = tile + (g >> 1) * kSub + (32 * w + kk) * 128;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const __half2 hs = __half2half2(__ushort_as_half(static_cast<unsigned short>(s[m])));
        const uint32_t* x = &c[m].x;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint4*>(dst + m * 1024 + (((4 * (g & 1) + j) ^ kk) << 4)) = dequant_word(x[j], hs);
      }
    };
    int T = 0;  // tiles so far
    for (int turn = 0, item = nth(0); ok && item < n_items; item = nth(++turn)) {
      const Work W = locate(P, item, cut);
      if (!W.found) break;
      for (int i = 0; ok && i < W.nt; ++i, ++T) {
        const int s = T & 1;
        ok = wait_warp(raw_full, T & 1, err, abort_v);
        if (!ok) break;
        uint4 ck[4], cv[4];
        uint32_t ks[4], vs[4];
        const unsigned char* code = raw + (32 * w + kk) * kCodeBytes + 16 * g;
        const unsigned char* scale = raw + kRawKs + (32 * w + kk) * 8 + 2 * g;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          ck[m] = *reinterpret_cast<const uint4*>(code + 8 * kCodeBytes * m);
          cv[m] = *reinterpret_cast<const uint4*>(code + kRawV + 8 * kCodeBytes * m);
          ks[m] = *reinterpret_cast<const unsigned short*>(scale + 64 * m);
          vs[m] = *reinterpret_cast<const unsigned short*>(scale + kRawVs - kRawKs + 64 * m);
        }
        const uint32_t gone = absent_raw[w];
        __syncwarp();
        if (lane == 0) mbar_arrive(raw_empty);  // the next tile may land
        const int left = W.kv_end - (W.tile0 + i) * kKeys - 32 * w;  // keys of this warp that are there
        if (left < 32 || gone) {  // what lies in the others' places counts as zeros
#pragma unroll
          for (int m = 0; m < 4; ++m)
            if (8 * m + kk >= left || ((gone >> (8 * m + kk)) & 1u)) {
              ck[m] = cv[m] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
              ks[m] = vs[m] = 0u;
            }
        }
        // a key whose scales are not all finite: NaN scores for whoever attends to it, and zeros as V,
        // which P = 0 of the others meets
        const bool some = (vs[0] & 0x7C00u) == 0x7C00u || (vs[1] & 0x7C00u) == 0x7C00u ||
                          (vs[2] & 0x7C00u) == 0x7C00u || (vs[3] & 0x7C00u) == 0x7C00u;
        if (__any_sync(0xffffffffu, some)) {
          const uint32_t mine = 0x00000303u << (lane & 0x16);  // the key's four lanes
#pragma unroll
          for (int m = 0; m < 4; ++m)
            if (__ballot_sync(0xffffffffu, (vs[m] & 0x7C00u) == 0x7C00u) & mine) {
              ks[m] = 0x7E00u;  // NaN
              vs[m] = 0u;
            }
        }
        if (T >= kStages) ok = wait_warp(&k_empty[s], ((T >> 1) - 1) & 1, err, abort_v);
        if (!ok) break;
        // ring of 4: slot T & 3 is free, since K's stage is (S of tile T - 2 done, so the softmax of
        // tile T - 3, and with it tile T - 4, is)
        if (lane == 0) absent[4 * (T & 3) + w] = gone;
        write(sk + s * 2 * kSub, ck, ks);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_full[s]);
        if (T >= kStages) ok = wait_warp(&v_empty[s], ((T >> 1) - 1) & 1, err, abort_v);
        if (!ok) break;
        write(sv + s * 2 * kSub, cv, vs);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[s]);
      }
    }
  } else if (warp == 14) {
    // ---- loads: the cached rows of a tile by bulk copies, one run per page: a lane per run of 16 keys
    // (the first of each page's issues it), while the tile before is converted
    const uint32_t scale_off = static_cast<uint32_t>(P.c.page_size) * kCodeBytes;
    unsigned char* raw = base + kOffRaw;
    int T = 0;
    for (int turn = 0, item = nth(0); ok && item < n_items; item = nth(++turn)) {
      const Work W = locate(P, item, cut);
      if (!W.found) break;
      if (W.n_t && W.tile0 == 0 && lane == 0) {
        const int start = P.starts ? P.starts[W.b] : 0;
        if (start < 0 || static_cast<long long>(start) + last_query(P, W.n_rows, W.r0) + 1 > P.max_seq_len)
          raise_error(err, kErrPosition);
      }
      const int32_t* bt = P.c.bt + static_cast<size_t>(W.b) * P.c.max_pages;
      auto page_of = [&](int i) {  // page of this lane's run (lanes 0..7); -1 past the end, -2 outside the pool
        const int p = (W.tile0 + i) * kKeys + kRun * lane;
        if (lane >= kKeys / kRun || i >= W.nt || p >= W.kv_end) return -1;
        const int page = __ldg(bt + P.c.page_index(p));
        return page >= 0 && page < P.c.n_pages ? page : -2;
      };
      int next = page_of(0);
      for (int i = 0; ok && i < W.nt; ++i, ++T) {
        const int page = next;
        next = page_of(i + 1);
        const int p = (W.tile0 + i) * kKeys + kRun * lane, row = p - P.c.page_index(p) * P.c.page_size;
        // a lane whose run continues the one before in the same page leaves it to that lane
        const uint32_t heads = __ballot_sync(0xffffffffu, page >= 0 && (row == 0 || lane == 0));
        const uint32_t live = __ballot_sync(0xffffffffu, page >= 0), out = __ballot_sync(0xffffffffu, page == -2);
        if (T > 0) ok = wait_warp(raw_empty, (T - 1) & 1, err, abort_v);
        if (!ok) break;
        if (out && lane == 0) raise_error(err, kErrPage);
        if (lane < 4)
          absent_raw[lane] = ((out >> (2 * lane)) & 1u) * 0x0000FFFFu | ((out >> (2 * lane + 1)) & 1u) * 0xFFFF0000u;
        __syncwarp();
        if (lane == 0) mbar_expect_tx(raw_full, __popc(live) * kRun * 2 * kRowBytes);
        __syncwarp();
        if ((heads >> lane) & 1u) {
          // runs from this lane to the next head or gap
          const uint32_t stop = (heads | ~live) & ~((2u << lane) - 1u);
          const uint32_t n = (stop ? __ffs(stop) - 1 : 32) - lane;
          const size_t blk = P.c.block(page, W.kvh);
          bulk_load(raw + kRun * lane * kCodeBytes, P.c.k + blk + row * kCodeBytes, n * kRun * kCodeBytes, raw_full);
          bulk_load(raw + kRawV + kRun * lane * kCodeBytes, P.c.v + blk + row * kCodeBytes, n * kRun * kCodeBytes,
                    raw_full);
          bulk_load(raw + kRawKs + kRun * lane * 8, P.c.k + blk + scale_off + row * 8, n * kRun * 8, raw_full);
          bulk_load(raw + kRawVs + kRun * lane * 8, P.c.v + blk + scale_off + row * 8, n * kRun * 8, raw_full);
        }
        __syncwarp();
      }
    }
    if (T > 0) {  // the last copies land before the CTA may exit (after a break: T names the last tile issued)
      const uint64_t t0 = globaltimer();
      while (!mbar_try(raw_full, (T - 1) & 1))
        if (globaltimer() - t0 > kTimeoutNs) break;
    }
  } else if (warp >= 12) {
    // ---- MMA issuers, a warp per row tile: while one waits for its softmax (some 200 cycles from
    // the barrier to the next MMA) the other's products run.  The whole warp runs the code and one
    // elected lane issues: uniform code keeps the descriptors in uniform registers.  (Issued from a
    // divergent branch an MMA costs some ten instructions, and on a scheduler shared with three busy
    // warps they came 110 .. 130 cycles apart, not 64.)
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
      auto issue_s = [&](int s, auto half) {  // S_t,u = Q_t K_u^T over 8 steps of 16 dims
        constexpr int u = decltype(half)::value;
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
      auto issue_o = [&](int s, auto half, bool acc) {  // O_t += P_t,u V_u over 4 steps of 16 keys
        constexpr int u = decltype(half)::value;
        if (leader) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_f16_ta(tmem_u + kColO + kDim * t, tmem_u + kColS + kHalf * (2 * t + u) + 8 * j,
                       desc(lo_v + 2 * s * kNext + 128 * (4 * u + j), hi_v), id_o, (acc || j > 0) ? 1u : 0u);
          mma_commit(&o_done[2 * t + u]);
        }
      };
      int T = 0, n_work = 0;  // tiles and units so far
      uint32_t used = 0u;     // bit u: parity of the uses of S half u so far
      for (int turn = 0, item = nth(0); ok && item < n_items; item = nth(++turn)) {
        const Work W = locate(P, item, cut);
        if (!W.found) break;
        if (W.nh == 0) continue;
        if (t >= W.n_t) {  // no rows here: only the stages' releases, tile by tile
          for (int i = 0; ok && i < W.nt; ++i, ++T) {
            const int s = T & 1;
            ok = wait_warp(&k_full[s], (T >> 1) & 1, err, abort_v) && wait_warp(&v_full[s], (T >> 1) & 1, err, abort_v);
            if (ok && leader) {
              mbar_arrive(&k_empty[s]);
              mbar_arrive(&v_empty[s]);
            }
          }
          continue;
        }
        ok = wait_warp(&q_full[t], n_work & 1, err, abort_v) && wait_warp(&k_full[T & 1], (T >> 1) & 1, err, abort_v);
        if (!ok) break;
        ++n_work;
        after();
        issue_s(T & 1, Int<0>{});
        if (W.nh > 1) issue_s(T & 1, Int<1>{});
        if (leader) mma_commit(&k_empty[T & 1]);
        // step i, half u of key tile T: O, then S of the same half of the next tile
        auto step = [&](int i, auto half) {
          constexpr int u = decltype(half)::value;
          const int s = T & 1, s1 = s ^ 1;
          const bool more = i + 2 < W.nh;
          if (u == 0) {
            ok = wait_warp(&v_full[s], (T >> 1) & 1, err, abort_v);
            if (more) ok = ok && wait_warp(&k_full[s1], ((T + 1) >> 1) & 1, err, abort_v);
          }
          ok = ok && wait_warp(&p_full[2 * t + u], (used >> u) & 1u, err, abort_v);
          if (!ok) return;
          used ^= 1u << u;
          after();
          issue_o(s, half, i > 0);
          if (more) issue_s(s1, half);  // (P, under S's columns, is read by the P V before it in the issue order)
          if (leader) {  // the stages' releases, at the last use of each
            if (u == 1 || i + 1 == W.nh) mma_commit(&v_empty[s]);
            if (more && (u == 1 || i + 3 == W.nh)) mma_commit(&k_empty[s1]);
          }
        };
        for (int i = 0; ok && i < W.nh; i += 2, ++T) {
          step(i, Int<0>{});
          if (ok && i + 1 < W.nh) step(i + 1, Int<1>{});
        }
      }
    };
    if (warp == 12) run(Int<0>{});
    else run(Int<1>{});
  } else {
    // ---- softmax of row tile t: thread = row (TMEM lane)
    const int t = warp >> 2, quad = warp & 3, rl = kRows * t + 32 * quad + lane;
    const uint32_t tl = tmem + (static_cast<uint32_t>(32 * quad) << 16), to = tl + kColO + kDim * t;
    // the queries of a unit: 16 lanes a row, dims of each 8 in mask order, all loads in flight.  Row rr of
    // the sequence is at rr * 128 + (rr / G) * (n_q - G) * 128 from its first query's heads.
    auto stage_q = [&](const Work& W) {
      const int c = lane & 15, row0 = 32 * quad + (lane >> 4);
      const __half* src = P.q + static_cast<size_t>(W.b) * P.seq * P.n_q * kDim + W.kvh * P.G * kDim + 8 * c;
      const int skip = (P.n_q - P.G) * kDim;
      uint4 v[16];
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int rr = W.r0 + kRows * t + row0 + 2 * x;
        v[x] = make_uint4(0u, 0u, 0u, 0u);
        if (rr < W.n_rows)
          v[x] = __ldg(reinterpret_cast<const uint4*>(src + static_cast<long long>(quotient(rr, P.by_G)) * skip +
                                                      static_cast<long long>(rr) * kDim));
      }
      unsigned char* dst = sq + (2 * t + (c >> 3)) * kSub + row0 * 128;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const uint4 m = make_uint4(__byte_perm(v[x].x, v[x].z, 0x5410), __byte_perm(v[x].x, v[x].z, 0x7632),
                                   __byte_perm(v[x].y, v[x].w, 0x5410), __byte_perm(v[x].y, v[x].w, 0x7632));
        *reinterpret_cast<uint4*>(dst + 256 * x + (((c & 7) ^ ((row0 + 2 * x) & 7)) << 4)) = m;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[t]);
    };
    // the next unit from `item` on that has rows for this tile; the key tiles of those passed over are counted
    int T = 0;
    uint32_t used = 0u;  // bit u: parity of the uses of S half u so far
    auto next_work = [&](int& turn, int& skipped) {
      Work W{};
      for (int item = nth(turn); item < n_items; item = nth(++turn)) {
        W = locate(P, item, cut);
        if (!W.found) break;
        if (t < W.n_t) return W;
        skipped += W.nt;
      }
      W.found = false;
      return W;
    };
    int turn = 0, skipped = 0;
    Work W = next_work(turn, skipped);
    if (W.found && W.nh > 0) stage_q(W);
    while (ok && W.found) {
      T += skipped;
      const int r = W.r0 + rl, qi = quotient(r, P.by_G);
      const int lim = r < W.n_rows ? limit(P, W.first, qi) : W.kv_end;
      const int lim_min = limit(P, W.first, quotient(W.r0 + kRows * t, P.by_G));
      float m_used = -INFINITY, l = 0.0f;  // running max (of q . k) and sum
      for (int i = 0; ok && i < W.nh; ++i) {
        const int u = i & 1, k0 = W.tile0 * kKeys + i * kHalf;
        const uint32_t ts = tl + kColS + kHalf * (2 * t + u);
        ok = wait_warp(&s_full[2 * t + u], (used >> u) & 1u, err, abort_v);
        if (!ok) break;
        used ^= 1u << u;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t sc[64];
        tmem_ld64(ts, sc);
        const volatile uint32_t* av = absent + 4 * ((T + (i >> 1)) & 3) + 2 * u;
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
        const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
        const float more = (top - m_used) * kScaleLog2;
        const bool grow = more > kRescaleLog2;  // (always on a row's first positions)
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? ex2(-more) : 1.0f;
          if (i > 0) {  // warp-wide read-modify-write of O_t, once the P V of the step before is done
            ok = wait_warp(&o_done[2 * t + (u ^ 1)], (~used >> (u ^ 1)) & 1u, err, abort_v);
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
          if (grow) m_used = top;
        }
        // differences to the maximum before the scale: exactly 0 at the maximum, so that P stays below 2^15 for scores
        // of any size (score times scale less a rounded product, one operation in place of two, is off by up to 2^3 at
        // scores of 10^9; 8 x 2048 155.0 us, with it 151.4)
        const float nm = m_used == -INFINITY ? 0.0f : -m_used;
        const uint64_t nm2 = pair(nm, nm), bias2 = pair(kPBias, kPBias), scale2 = pair(kScaleLog2, kScaleLog2);
        uint64_t sm[4] = {0ull, 0ull, 0ull, 0ull};
        uint32_t pk[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          float a0, a1;
          unpair(fma2(add2(pair(__uint_as_float(sc[2 * e]), __uint_as_float(sc[2 * e + 1])), nm2), scale2, bias2), a0, a1);
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
      T += W.nt;
      // the next unit's queries (every S of this one is read, so its Q is free): its first S is made
      // while this one's result is written
      const Work D = W;
      ++turn;
      skipped = 0;
      W = next_work(turn, skipped);
      if (ok && W.found && W.nh > 0) stage_q(W);
      // ---- this row of O (dims of each 8 back in order), normalised or as a partial
      if (ok && D.nh > 0) {
        const int u = (D.nh - 1) & 1;
        ok = wait_warp(&o_done[2 * t + u], (~used >> u) & 1u, err, abort_v);
      }
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const size_t head = (static_cast<size_t>(D.b) * P.seq + qi) * P.n_q + D.kvh * P.G + (r - qi * P.G);
      const size_t part = (static_cast<size_t>(D.piece) * P.c.n_kv + D.kvh) * P.rows_item + rl;
      const bool there = r < D.n_rows;
      if (P.n_splits > 1 && there) P.part_ml[part] = make_float2(m_used * kScaleLog2, l);
#pragma unroll 1
      for (int cc = 0; cc < kDim; cc += 32) {
        uint32_t o[32];
        if (D.nh > 0) {
          tmem_ld32(to + cc, o);
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = 0u;
        }
        if (there) {
          constexpr int at[8] = {0, 2, 4, 6, 1, 3, 5, 7};  // where dim e of a group of 8 is
          uint32_t out8[8];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(o[8 * g + at[e]]);
            if (P.n_splits == 1) {
              uint32_t* x = out8 + 4 * (g & 1);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const __half2 hh = __floats2half2_rn(v[2 * e] * inv, v[2 * e + 1] * inv);
                x[e] = *reinterpret_cast<const uint32_t*>(&hh);
              }
              if (g & 1) {  // a sector of this lane's row
                asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(P.out + head * kDim + cc + 8 * (g - 1)),
                             "r"(out8[0]), "r"(out8[1]), "r"(out8[2]), "r"(out8[3]), "r"(out8[4]), "r"(out8[5]),
                             "r"(out8[6]), "r"(out8[7])
                             : "memory");
              }
            } else {
              asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(P.part_o + part * kDim + cc + 8 * g),
                           "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                           : "memory");
            }
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
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

// Rows of a work unit's partials, and row blocks of a sequence.
static int rows_of_item(long long seq_len, int G) {
  return static_cast<int>(seq_len * G < q4::pf::kTiles * q4::pf::kRows ? seq_len * G : q4::pf::kTiles * q4::pf::kRows);
}
static long long blocks_of(long long seq_len, int G) {
  return (seq_len * G + q4::pf::kTiles * q4::pf::kRows - 1) / (q4::pf::kTiles * q4::pf::kRows);
}

extern "C" int lmps_prefill_q4_splits(int batch, int seq_len, int n_q_heads, int n_kv_heads, int max_seq_len) {
  if (batch <= 0 || seq_len <= 0 || n_kv_heads <= 0 || n_q_heads < n_kv_heads || max_seq_len <= 0) return 1;
  // One CTA per SM: as many pieces of the context as there are SMs for a unit of work, none below 8 tiles
  // (the merge is another launch of some 3 us); two where the units fill half the SMs.
  const long long items = blocks_of(seq_len, n_q_heads / n_kv_heads) * n_kv_heads * batch;
  if (items >= q4::pf::kSms) return 1;
  const long long most = max_seq_len / (8 * q4::pf::kKeys), n = items > q4::pf::kSms / 2 ? 2 : q4::pf::kSms / items;
  return static_cast<int>(n < most ? n : most < 1 ? 1 : most);
}

extern "C" size_t lmps_prefill_q4_workspace_size(int batch, int seq_len, int n_q_heads, int head_dim, int n_splits) {
  if (n_splits <= 1 || batch <= 0 || seq_len <= 0 || n_q_heads <= 0 || head_dim <= 0) return 0;
  // partials in whole row blocks where a sequence may have more than one (at most 8 rows a query)
  const size_t blocks = static_cast<size_t>(blocks_of(seq_len, q4::kMaxHeads));
  const size_t rows = (static_cast<size_t>(seq_len) + (blocks > 1 ? q4::pf::kTiles * q4::pf::kRows - 1 : 0)) * n_q_heads;
  return static_cast<size_t>(batch) * n_splits * rows * (head_dim * sizeof(float) + sizeof(float2)) +
         static_cast<size_t>(batch) * blocks * sizeof(int2);
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
                 lmps_aligned(out, 32) && lmps_aligned(workspace, 32));
  const int G = n_q_heads / n_kv_heads;
  const long long rows = static_cast<long long>(batch) * seq_len, blocks = blocks_of(seq_len, G);
  const long long items = blocks * n_kv_heads * batch;
  // (positions and rows are ints; tile counts of all units are summed in one)
  if (rows > 0x7FFFFFFFLL || static_cast<long long>(seq_len) * G >= 1LL << 29 ||
      items * n_splits * n_kv_heads >= 1LL << 31 || blocks * batch * batch >= 1LL << 31 ||
      blocks * batch > (1LL << 30) / ((max_seq_len + pf::kKeys - 1) / pf::kKeys))
    return LMPS_ERR_UNSUPPORTED;
  const size_t need = lmps_prefill_q4_workspace_size(batch, seq_len, n_q_heads, head_dim, n_splits);
  if (need > 0 && (!workspace || workspace_bytes < need)) return LMPS_ERR_WORKSPACE;
  pf::Params P{};
  P.q = reinterpret_cast<const __half*>(q);
  P.c = q4::Cache{k_pool, v_pool, block_table, n_pages, max_pages, page_size, n_kv_heads,
                  q4::page_shift_of(page_size), error};
  P.starts = starts;
  P.q_lens = q_lens;
  P.out = reinterpret_cast<__half*>(out);
  P.n_q = n_q_heads;
  P.G = G;
  P.seq = seq_len;
  P.batch = batch;
  P.n_blocks = static_cast<int>(blocks);
  P.n_splits = n_splits;
  P.max_seq_len = max_seq_len;
  P.rows_item = rows_of_item(seq_len, G);
  auto reciprocal = [](int d) { return d == 1 ? 0u : static_cast<uint32_t>((1ull << 32) / d + 1); };
  P.by_G = reciprocal(G);
  P.by_kv = reciprocal(n_kv_heads);
  P.by_batch = reciprocal(batch);
  q4::Partials parts{};
  const size_t n_part = static_cast<size_t>(items) * n_splits * P.rows_item;
  parts.o = P.part_o = reinterpret_cast<float*>(workspace);
  parts.ml = P.part_ml = reinterpret_cast<float2*>(P.part_o + n_part * q4::kDim);
  parts.pieces = P.pieces = reinterpret_cast<int2*>(P.part_ml + n_part);
  parts.out = P.out;
  parts.n_q = n_q_heads;
  parts.n_kv = n_kv_heads;
  parts.rows_item = P.rows_item;
  parts.q_lens = q_lens;
  parts.seq = seq_len;
  parts.batch = batch;
  parts.n_blocks = P.n_blocks;
  const int st_attr = lmps_max_dyn_smem<pf::prefill_q4_kernel>(pf::kSmemBytes);
  if (st_attr != LMPS_OK) return st_attr;
  cudaStream_t s = lmps_stream(stream);
  const long long ctas = items * n_splits < pf::kSms ? items * n_splits : pf::kSms;
  const int status = lmps_launch_pdl(pf::prefill_q4_kernel, dim3(static_cast<unsigned>(ctas)), dim3(pf::kThreads),
                                     static_cast<size_t>(pf::kSmemBytes), s, P);
  if (status || n_splits == 1) return status;
  return q4::combine_launch(parts, static_cast<int>(rows), s);
}

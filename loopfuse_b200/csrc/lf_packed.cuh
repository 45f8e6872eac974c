// Attention tiles of batches whose requests have different lengths: the kernel behind packed prefill
// (lf_packed_prefill.cu) and behind the shared part of shared-prefix decode (lf_shared_prefix.cu).
//
// A tile is up to 128 score rows of one kv head: `tq` consecutive query tokens (or requests, for the
// shared prefix), each with the G query heads that share the kv head, token-major. The rows of a tile
// see the same keys but for the mask, so K and V are fetched once for all G heads, and a prompt of a few
// tokens still fills 128 / G rows' worth of the tensor pipe. Mathematics: online softmax in the log2
// domain, o = sum_j 2^(f(s_j) - m) v_j, l = sum_j 2^(f(s_j) - m), with a reference m that moves when
// the row maximum passes it by more than 2^8 (the rescale is rare) and out = o / l.
//
// Two CTAs per SM, each of which takes tiles (or slices of the keys of long ones) from a list until it is
// empty. 256 threads:
//   warps 0-3   softmax (one thread per score row)
//   warp  4     takes the items from the list and hands them to the other warps; Q, and the K blocks
//   warp  5     issues S[g & 1] = Q K^T, as soon as PV of block g - 2 is done with the buffer
//   warp  6     the V blocks
//   warp  7     issues O += P V
// (One warp for both products takes longer over a block than the softmax warps: beside them it gets few
// issue slots. 8 prompts up to 8192 tokens 718 us, and 806 with every other wait in front of that for P.)
// Blocks are numbered through over all items of a CTA (g): the producers and the issuer run on into the
// next item while the softmax warps finish the last one, so the look-ups, copies and first scores of a
// tile lie under the blocks of the tile before it. (Short prompts are mostly starts and ends: one CTA per
// tile, 28 prompts of 512 tokens, 32 heads on 8, took 144 us.)
// Tensor memory (256 columns): S of buffer b at column b * 64, P (bf16) over its first 32 columns, O at 128.
//
// What bounds it: with a head dim of 128 the products of a block are 512 clocks of the tensor pipe, and two
// CTAs of 128 rows keep it busy half of the time; the rest is the chain score -> exp2 -> P of each CTA
// and the load of a row's scores and store of its weights (the load of S 160 clocks, the arithmetic some
// 1200, the hand-over of P and the wait for the next S 700). 8 prompts up to 8192 tokens, 32 heads on 8: 662 us
// for 664 GFLOP (1.0 PFLOP/s); 24 up to 2048 with a window of 256 and a softcap: 131 us, of which the tensor pipe is
// active 26 %.
//
// What a packed batch adds to the tiles of the prefill kernels: the last key block of a request holds
// rows of the next one (or, in a page, of whoever had it before). Their scores are masked; their V rows
// are zeroed in shared memory by the softmax warps before P V, since 0 * infinity or 0 * NaN of a
// stranger would reach every row. (Rows that a window leaves out of a paged tile's first block come as zeros.)
#pragma once

#include "lf_common.cuh"
#include "lf_tensor_map.h"

#include <float.h>

namespace lf {

constexpr int kPackedRows = 128;  // of a tile
constexpr int kPackedKeys = 64;   // of a block
constexpr int kPackedThreads = 256;
constexpr int kMostKeys = 1 << 30;  // of a request: no sum of a key and a block passes 32 bits
constexpr float kPackedLog2e = 1.4426950408889634f;

// Where a tile's rows and keys come from.
enum PackedKind {
  kPackedDense = 0,   // packed queries, packed keys
  kPackedPaged = 1,   // packed queries, keys through a block table
  kPackedPrefix = 2,  // one query token per request against a slice of the shared prefix; partial results
};

// A tile, or a slice of its keys, as the list has it (the kv head comes with the place in the order).
struct __align__(16) PackedItem {
  int32_t q_row;    // first query row (token of the packed batch; request, for the prefix)
  int32_t count;    // tokens; 0: none, the end of a CTA's items
  int32_t k_from;   // dense: row of the request's first key; paged: row of the block table
  int32_t m;        // the request's keys
  int32_t pos;      // last key that the first token sees
  int32_t lo, hi;   // key blocks
  int32_t hkv;      // (in shared memory)
  int32_t part;     // slices of one tile: the first one's place in the workspace, else -1
  int32_t n_parts, index;
  int32_t counter;  // ... and the count of those that are done
};

struct PackedParams {
  __nv_bfloat16* out;
  int64_t o_stride[2];        // (token, head)
  int32_t out_sectors;        // output rows are 32-byte aligned
  const int32_t* cu_q;        // [B + 1] first query token of each request
  const int32_t* cu_k;        // dense: [B + 1] first key
  const int32_t* kv_lens;     // paged, prefix: [B] keys of each request
  const int32_t* table;       // block table
  int64_t bt_stride;
  const PackedItem* items;    // the list, or null: a CTA has one tile, which it looks up
  uint32_t* list;             // [0] items of a kv head, [1] ticket, [2 ..] slices done, by counter
  int32_t B, T, Tk, Hkv, G;
  int32_t tq;                 // tokens (requests) per tile: 128 / G
  int32_t mask_kind, window;
  float a;                    // softcap: score = tanh(raw * a) * c2
  float c2;                   // logit in the log2 domain = score * c2; > 0
  float m_first;              // a row's first reference: -inf, or 0 where no logit is far from it
  int32_t bt_blocks, page_size, page_shift, n_pages;
  int32_t box, box_shift;     // keys per copy of a paged operand, a power of two: they lie in one page
  int32_t page_groups;        // groups of 8 slots per page, where a copy can move several (see packed_pool_map)
  int32_t n_tiles;            // tiles of a kv head (no list: an upper bound)
  FastDiv div_chunk;          // heads of a chunk of kv heads (see the launch); prefix: kv heads
  FastDiv div_tiles;          // tiles (no list)
  FastDiv div_g;              // query heads per kv head
  int32_t prefix_len, chunk;  // prefix: keys [split * chunk, ...) below prefix_len
  float* part_o;              // [slice][row][D] un-normalised
  float2* part_ml;            // [slice][row] (reference, sum)
  int32_t* status;
};

template <int D>
struct PackedShape {
  static constexpr int kStages = D == 64 ? 4 : 2;  // of K, and of V: blocks in flight
  // Behind the rings, unused: see packed_keeps_tensor_memory.
  static constexpr uint32_t kRest = 13 * 1024;
  static constexpr uint32_t kTmemColumns = 256;
  static constexpr uint32_t kQBlockBytes = kPackedRows * 128;  // [128][64] bf16
  static constexpr uint32_t kKVBlockBytes = kPackedKeys * 128;
  static constexpr uint32_t kTileBytes = kKVBlockBytes * (D / 64);
  static constexpr size_t kSmem = 1024 /*barriers*/ + kRest +
                                  kQBlockBytes * (D / 64) + kStages * 2 * kTileBytes;
};

// An SM's 512 columns, by shared memory (of 228 KB): two of these CTAs, never three, and never one beside a CTA of
// prefill_kernel that takes all the columns, whose smallest leaves less than 96256 bytes. (A CTA may wait for the
// kernel before its own with its columns taken.)
template <int D>
constexpr bool packed_keeps_tensor_memory() {
  constexpr size_t smem = PackedShape<D>::kSmem;
  return smem >= 96256 && 2 * (smem + 1024) <= 233472 && 3 * (smem + 1024) > 233472;
}
static_assert(packed_keeps_tensor_memory<64>() && packed_keeps_tensor_memory<128>(), "tensor memory runs out on an SM");

constexpr int kItemSlots = 4;

struct __align__(16) PackedBarriers {
  PackedItem item[kItemSlots];
  uint64_t item_full[kItemSlots], item_empty[kItemSlots];
  uint64_t q_full, q_empty;
  uint64_t k_full[4], k_empty[4];
  uint64_t v_full[4], v_empty[4];
  uint64_t s_full[2];   // MMA -> softmax
  uint64_t p_full[2];   // softmax -> MMA
  uint64_t s_free[2];   // PV done: the buffer may take other scores
  uint64_t pv_done;     // second-to-last PV of an item done
  uint64_t o_final;     // last PV of an item done
  uint64_t o_empty;     // softmax -> MMA: O has been read
  uint32_t tmem_base;
  uint32_t last_part;
};
static_assert(sizeof(PackedBarriers) <= 1024, "the block in front of the staging");

// A value that is the same in all lanes, as one that the compiler knows to be: loops and branches on it
// need no registers to bring the lanes together again.
__device__ __forceinline__ int warp_uniform(int x) { return __reduce_max_sync(0xffffffffu, x); }

__device__ __forceinline__ void packed_timeout(int32_t* status, int where) {
  if (status) atomicCAS(status, LF_DEV_OK, LF_DEV_TIMEOUT | (where << 8));
}

// A request of a packed batch. Offsets that are not in order or leave the tensors are cut to them.
struct PackedRequest {
  int q0, n;  // first query token, tokens
  int k0, m;  // first key (dense), keys
};
__device__ __forceinline__ int clamp_to(int x, int most) { return min(max(x, 0), most); }

template <int KIND>
__device__ __forceinline__ PackedRequest packed_request(const PackedParams& p, int b) {
  PackedRequest r;
  r.q0 = clamp_to(p.cu_q[b], p.T);
  r.n = max(clamp_to(p.cu_q[b + 1], p.T) - r.q0, 0);
  if constexpr (KIND == kPackedDense) {
    r.k0 = clamp_to(p.cu_k[b], p.Tk);
    r.m = max(clamp_to(p.cu_k[b + 1], p.Tk) - r.k0, 0);
  } else {
    r.k0 = b;
    const int64_t held = static_cast<int64_t>(p.bt_blocks) * p.page_size;
    r.m = clamp_to(p.kv_lens[b], held > kMostKeys ? kMostKeys : static_cast<int>(held));
  }
  return r;
}

// First key that any row of an item sees.
__device__ __forceinline__ int first_key(const PackedParams& p, const PackedItem& it) {
  return p.mask_kind == LF_MASK_CAUSAL_WINDOW ? max(0, it.pos - (p.window - 1)) : 0;
}

// Tile `tile` of request r as one item.
__device__ __forceinline__ PackedItem packed_item(const PackedParams& p, const PackedRequest& r, int tile) {
  PackedItem it;
  const int t0 = tile * p.tq;
  it.q_row = r.q0 + t0;
  it.count = min(p.tq, r.n - t0);
  it.k_from = r.k0;
  it.m = r.m;
  it.pos = t0 + r.m - r.n;
  const int first = first_key(p, it);
  int end = r.m;
  if (p.mask_kind != LF_MASK_NONE) end = min(end, it.pos + it.count);
  it.lo = first / kPackedKeys;
  it.hi = end > first ? (end + kPackedKeys - 1) / kPackedKeys : it.lo;
  it.hkv = 0;
  it.part = -1;
  it.n_parts = 1;
  it.index = it.counter = 0;
  return it;
}

// Request and tile of place `rank`, requests in order and a request's heaviest tile first; the whole
// warp. Request -1: there is no such tile.
__device__ __forceinline__ int2 find_tile(const PackedParams& p, int rank) {
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    int tiles = 0;
    if (b0 + lane < p.B) {
      const int q0 = clamp_to(p.cu_q[b0 + lane], p.T);
      const int n = max(clamp_to(p.cu_q[b0 + lane + 1], p.T) - q0, 0);
      tiles = (n + p.tq - 1) / p.tq;
    }
    int incl = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, base + incl > rank);
    if (past) {
      const int at = __ffs(past) - 1;
      return make_int2(b0 + at, base + __shfl_sync(0xffffffffu, incl, at) - 1 - rank);
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  return make_int2(-1, 0);
}

// Item at place `at` of the order: chunks of kv heads, in each the list, longest first, for every head of
// the chunk. `n`: items of the list.
__device__ __forceinline__ PackedItem listed_item(const PackedParams& p, uint32_t at, uint32_t n) {
  PackedItem it;
  it.count = 0;
  const uint32_t r = p.div_chunk.div(at);
  const uint32_t chunk = r / n;
  const uint32_t hkv = chunk * p.div_chunk.d + (at - r * p.div_chunk.d);
  if (chunk * p.div_chunk.d >= static_cast<uint32_t>(p.Hkv)) return it;  // past the last one
  const int4* src = reinterpret_cast<const int4*>(p.items + (r - chunk * n));
  const int4 x = src[0], y = src[1], z = src[2];
  it.q_row = x.x, it.count = x.y, it.k_from = x.z, it.m = x.w;
  it.pos = y.x, it.lo = y.y, it.hi = y.z;
  it.part = z.x, it.n_parts = z.y, it.index = z.z, it.counter = z.w;
  it.hkv = static_cast<int>(hkv);
  if (it.hkv >= p.Hkv) it.lo = it.hi = it.hkv = -1;  // a place of the last chunk that has no head
  return it;
}

// The only item of a CTA without a list.
template <int KIND>
__device__ __forceinline__ PackedItem own_item(const PackedParams& p, int cta) {
  PackedItem it;
  it.count = 0;
  if constexpr (KIND == kPackedPrefix) {
    const int unit = static_cast<int>(p.div_tiles.div(cta));  // (split, kv head); tiles of it together
    it.q_row = (cta - unit * static_cast<int>(p.div_tiles.d)) * p.tq;
    it.index = static_cast<int>(p.div_chunk.div(unit));       // split
    it.hkv = unit - it.index * static_cast<int>(p.div_chunk.d);
    it.count = min(p.tq, p.B - it.q_row);
    it.k_from = 0;
    it.pos = 0;
    it.m = min(p.prefix_len, (it.index + 1) * p.chunk);
    it.lo = it.index * (p.chunk / kPackedKeys);
    it.hi = (it.m + kPackedKeys - 1) / kPackedKeys;
    it.part = it.n_parts = it.counter = 0;
  } else {
    const int r = static_cast<int>(p.div_chunk.div(cta));
    const int chunk = static_cast<int>(p.div_tiles.div(r));
    const int hkv = chunk * static_cast<int>(p.div_chunk.d) + cta - r * static_cast<int>(p.div_chunk.d);
    if (hkv < p.Hkv) {
      const int2 at = find_tile(p, r - chunk * static_cast<int>(p.div_tiles.d));
      if (at.x >= 0) {
        it = packed_item(p, packed_request<KIND>(p, at.x), at.y);
        it.hkv = hkv;
      }
    }
  }
  return it;
}

// 32 bytes (a whole sector) per thread.
__device__ __forceinline__ void stg_32(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// Output rows of a tile from its slices, a warp for its 32 rows, lanes along the columns: o = sum_s o_s
// 2^(m_s - m) / sum_s l_s 2^(m_s - m). Eight rows at a time, so that their loads are in flight together.
template <int D>
__device__ __forceinline__ void join_slices(const PackedParams& p, const PackedItem& it, int warp, int lane,
                                         int rows) {
  constexpr int kCols = D / 32, kRows = 8;
  const int n = it.n_parts, hkv = it.hkv, q_row = it.q_row;
  const int64_t part0 = (static_cast<int64_t>(it.part) * p.Hkv + hkv) * kPackedRows;
  const int64_t step = static_cast<int64_t>(p.Hkv) * kPackedRows;
  const int end = min(warp * 32 + 32, rows);
  #pragma unroll 1
  for (int r0 = warp * 32; r0 < end; r0 += kRows) {
    float acc[kRows][kCols], l[kRows], m[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      m[u] = -INFINITY;
      l[u] = 0.f;
#pragma unroll
      for (int c = 0; c < kCols; ++c) acc[u][c] = 0.f;
    }
    for (int s = 0; s < n; ++s) {
      float2 ml[kRows];
      float x[kRows][kCols];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const int64_t at = part0 + s * step + min(r0 + u, end - 1);
        ml[u] = __ldcg(&p.part_ml[at]);
        const float* src = p.part_o + at * D + lane * kCols;
        if constexpr (kCols == 4) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
          x[u][0] = v.x, x[u][1] = v.y, x[u][2] = v.z, x[u][3] = v.w;
        } else {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
          x[u][0] = v.x, x[u][1] = v.y;
        }
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        if (ml[u].y == 0.f) continue;  // (no key of this row: what its accumulator holds is of no value)
        const float top = fmaxf(m[u], ml[u].x);
        const float back = ex2_approx(m[u] - top), w = ex2_approx(ml[u].x - top);
        m[u] = top;
        l[u] = fmaf(l[u], back, ml[u].y * w);
#pragma unroll
        for (int c = 0; c < kCols; ++c) acc[u][c] = fmaf(acc[u][c], back, x[u][c] * w);
      }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      if (r0 + u >= end) break;
      const int tok = static_cast<int>(p.div_g.div(r0 + u));
      __nv_bfloat16* dst = p.out + static_cast<int64_t>(q_row + tok) * p.o_stride[0] +
                           static_cast<int64_t>(hkv * p.G + r0 + u - tok * p.G) * p.o_stride[1] + lane * kCols;
      const float inv = l[u] == 0.f ? 0.f : 1.f / l[u];
      if constexpr (kCols == 4)
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(acc[u][0] * inv, acc[u][1] * inv),
                                                    pack_bf16x2(acc[u][2] * inv, acc[u][3] * inv));
      else
        *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(acc[u][0] * inv, acc[u][1] * inv);
    }
  }
}

template <int D, int KIND, bool SOFTCAP>
__device__ __forceinline__ void packed_tiles(const CUtensorMap& tmap_q, const CUtensorMap& tmap_k,
                                             const CUtensorMap& tmap_v, const PackedParams& p, int cta) {
  using Shape = PackedShape<D>;
  constexpr int kStages = Shape::kStages;
  constexpr int kBlocksD = D / 64;
  constexpr uint32_t kIdescQK = make_idesc_bf16(128, kPackedKeys, 0);
  constexpr uint32_t kIdescPV = make_idesc_bf16(128, D, 1);
  constexpr uint32_t kColO = 128;
  constexpr int kKWarp = 4, kQkWarp = 5, kVWarp = 6, kPvWarp = 7;
  constexpr bool kPages = KIND != kPackedDense;
  // A K or V block in shared memory: 8-row groups of 64-column halves, [half][group] where one copy moves
  // them all, [group][half] where a copy moves the groups of a page.
  constexpr uint32_t kHalf = kPages ? 1024 : Shape::kKVBlockBytes;         // bytes between halves
  constexpr uint32_t kGroup = kPages ? 1024 * kBlocksD : 1024;             // and between groups

  // (Aligned by declaration: every address is a constant then, and none of them takes registers.)
  extern __shared__ __align__(1024) unsigned char smem[];
  PackedBarriers* bars = reinterpret_cast<PackedBarriers*>(smem);
  unsigned char* sQ = smem + 1024;
  unsigned char* sK = sQ + Shape::kQBlockBytes * kBlocksD;
  unsigned char* sV = sK + kStages * Shape::kTileBytes;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  // ---------------- setup ----------------
  if (warp == kKWarp && lane == 0) {
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
    for (int i = 0; i < kItemSlots; ++i) {
      mbar_init(&bars->item_full[i], 1);
      mbar_init(&bars->item_empty[i], 7);  // (softmax, QK, V, PV)
    }
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->q_empty, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->v_empty[s], 1);
    }
    for (int bf = 0; bf < 2; ++bf) {
      mbar_init(&bars->s_full[bf], 1);
      mbar_init(&bars->p_full[bf], 4);
      mbar_init(&bars->s_free[bf], 1);
    }
    mbar_init(&bars->pv_done, 1);
    mbar_init(&bars->o_final, 1);
    mbar_init(&bars->o_empty, 4);
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(&bars->tmem_base, Shape::kTmemColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  pdl_wait();  // (nothing in global memory has been touched so far)

  // 128 registers per thread at two CTAs of 256: 184 for the softmax warps, 72 for the others (one
  // instruction per warpgroup, in front of the dispatch of roles).
  if (warp >= 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");

  // A wait that runs out is reported, and the waits after it are passed over: the warp runs through what
  // is left without a loop to leave in the middle (lanes that may leave one apart cost the registers that
  // bring them together again).
  bool lost = false;
  auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
    if (!lost && !mbar_wait(bar, parity)) {
      packed_timeout(p.status, where);
      lost = true;
    }
  };
  // Item number i of this CTA, once warp 4 has put it there.
  auto take_item = [&](int i, PackedItem* it) {
    wait(&bars->item_full[i % kItemSlots], (i / kItemSlots) & 1, 80);
    *it = bars->item[i % kItemSlots];
    if (__any_sync(0xffffffffu, lost)) it->count = 0;
  };
  auto free_item = [&](int i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->item_empty[i % kItemSlots]);
  };
  // Rows that see a handful of keys do not average the rounding of P away: where the first row of the tile
  // does (the start of a prompt, a tiny window), P enters the second product as two bf16, its rounding and
  // what that leaves, in the half of the S buffer that P does not need. Behind a prefix P is one bf16 whatever the
  // prefix's length, each weight within 2^-9 of its value: against 64 bits 0.0021 to 0.0024 of the outputs' size, where
  // a paged decode, which keeps two, has 0.0017. (The rows of a tile are different requests, so that one of a few
  // keys would cost all of them the second product.)
  auto is_fine = [&](const PackedItem& it) {
    if constexpr (KIND == kPackedPrefix) return false;
    int sees = it.m;
    if (p.mask_kind != LF_MASK_NONE) sees = min(sees, it.pos + 1);
    if (p.mask_kind == LF_MASK_CAUSAL_WINDOW) sees = min(sees, p.window);
    return sees < 16;
  };

  // Next place in the order (without a list there is none).
  auto take_place = [&]() -> uint32_t {
    uint32_t at = 0xffffffffu;
    if (p.items) {
      if (lane == 0) at = atomicAdd(&p.list[1], 1u);
      at = gridDim.x + __shfl_sync(0xffffffffu, at, 0);
    }
    return at;
  };

  if (warp == kKWarp || warp == kVWarp) {
    // ---------------- producers ----------------
    // The whole warp runs the loops and waits; the elected lane issues the copies.
    const bool is_k = warp == kKWarp;
    const bool elected = elect_one_sync();
    const CUtensorMap* map = is_k ? &tmap_k : &tmap_v;
    unsigned char* ring = is_k ? sK : sV;
    uint64_t* full = is_k ? bars->k_full : bars->v_full;
    uint64_t* empty = is_k ? bars->k_empty : bars->v_empty;
    auto page_of = [&](int t) { return p.page_shift >= 0 ? (t >> p.page_shift) : (t / p.page_size); };
    const int boxes = kPages ? kPackedKeys / p.box : 1;

    // K warp: takes the place of the next item as the last blocks of the present one are on their way. (Earlier, at
    // the start of the item, it is another CTA's that could start it sooner: 256 slices of 36 blocks were two each
    // for 50 of the CTAs. The blocks that are still to be computed hide the look-ups.)
    uint32_t n_list = 0, at = cta;
    auto read_item = [&](bool first) {
      PackedItem x;
      x.count = 0;
      if (p.items) {
        if (n_list > 0) x = listed_item(p, at, n_list);
      } else if (first) {
        x = own_item<KIND>(p, cta);
      }
      return x;
    };
    auto hand_on = [&](PackedItem x, int i) {
      // (A tile that sees no key is not handed on: its rows are zeros, written here.)
      while (KIND != kPackedPrefix && x.count > 0 && x.hi <= x.lo) {
        const int pieces = x.hkv < 0 ? 0 : x.count * p.G * (D / 8);
        for (int e = lane; e < pieces; e += 32) {
          const int r = e / (D / 8), t = static_cast<int>(p.div_g.div(r));
          *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(x.q_row + t) * p.o_stride[0] +
                                    static_cast<int64_t>(x.hkv * p.G + r - t * p.G) * p.o_stride[1] +
                                    (e % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
        }
        at = take_place();
        x = read_item(false);
      }
      wait(&bars->item_empty[i % kItemSlots], ((i / kItemSlots) & 1) ^ 1, 87);
      __syncwarp();
      if (lane == 0) {
        bars->item[i % kItemSlots] = x;
        mbar_arrive(&bars->item_full[i % kItemSlots]);
      }
      __syncwarp();
    };
    if (is_k) {
      if (p.items) n_list = p.list[0];
      hand_on(read_item(true), 0);
    }
    int g = 0;  // blocks
    for (int i = 0;; ++i) {
      PackedItem it;
      take_item(i, &it);
      if (!is_k) free_item(i);
      if (it.count <= 0) break;
      const int lo = it.lo, hi = it.hi;
      {
        if (is_k) {
          if (i > 0) wait(&bars->q_empty, (i - 1) & 1, 81);
          __syncwarp();
          if (elected) {
            // (A box is always tq tokens; those past the end of the request are strangers' rows or zeros.)
            mbar_arrive_expect_tx(&bars->q_full, static_cast<uint32_t>(p.tq * p.G) * 128 * kBlocksD);
#pragma unroll
            for (int kb = 0; kb < kBlocksD; ++kb)
              tma_load_5d(sQ + kb * Shape::kQBlockBytes, &tmap_q, &bars->q_full, kb * 64, 0, it.hkv, it.q_row, 0);
          }
        }
        // Table entries of the copies ("boxes"), 32 at a time, a box per lane; the next 32 are requested before
        // these are used. (Block by block the look-up took 800 clocks of each.)
        const int32_t* table = p.table + static_cast<int64_t>(it.k_from) * p.bt_stride;
        const int box_end = kPages ? min((it.m + p.box - 1) >> p.box_shift, hi * boxes) : 0;  // that hold a key
        int window = kPages ? lo * boxes / 32 : 0;
        int32_t page = 0, page_next = 0;
        // Boxes in front of all keys that a row sees (the first block may have some): their pages may be anybody's by
        // now, so their entries are not looked at, and the copy reads past the last page, which is zeros.
        const int box0 = KIND == kPackedPaged ? first_key(p, it) >> p.box_shift : 0;
        auto request = [&](int w) -> int32_t {
          const int n = w * 32 + lane;
          if (n < box0 || n >= box_end) return 0;
          const int at = page_of(n * p.box);
          return LF_BOUNDS(at >= 0 && at < p.bt_blocks, p.status, 70) ? table[at] : 0;
        };
        auto checked = [&](int32_t pg, int w) -> int32_t {
          if (KIND == kPackedPaged && w * 32 + lane < box0) return p.n_pages;
          if (pg >= 0 && pg < p.n_pages) return pg;
          if (p.status) atomicExch(p.status, LF_DEV_BAD_PAGE);
          return 0;
        };
        if constexpr (kPages) {
          page = request(window);
          page_next = request(window + 1);
          page = checked(page, window);
        }
        for (int j = lo; j < hi; ++j, ++g) {
          const int stage = g % kStages;
          wait(&empty[stage], ((g / kStages) & 1) ^ 1, 81);
          __syncwarp();
          const bool run = elected && !lost;
          unsigned char* dst = ring + stage * Shape::kTileBytes;
          if constexpr (!kPages) {
            // (Both 64-column halves in one copy: the third dimension of the map.)
            if (run) {
              mbar_arrive_expect_tx(&full[stage], Shape::kTileBytes);
              tma_load_5d(dst, map, &full[stage], 0, it.k_from + j * kPackedKeys, 0, it.hkv, 0);
            }
          } else {
            const int n0 = j * boxes;
            const int live = min(boxes, box_end - n0);  // (the rest of the last block is not fetched)
            if (run)
              mbar_arrive_expect_tx(&full[stage], static_cast<uint32_t>(live * p.box) * 128 * kBlocksD);
            // Four boxes at a time: places by shuffle, then the copies in one go. (They lie in one window: 32 is a
            // multiple of them, or they of 32.)
            for (int r0 = 0; r0 < live; r0 += 4) {
              if ((n0 + r0) / 32 != window) {
                ++window;
                page = checked(page_next, window);
                page_next = request(window + 1);
              }
              int pg[4], slot[4];
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const int n = n0 + min(r0 + u, live - 1);
                pg[u] = __shfl_sync(0xffffffffu, page, n & 31);
                slot[u] = n * p.box - page_of(n * p.box) * p.page_size;
              }
              if (run) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                  const int row = (r0 + u) * p.box;
                  if (r0 + u >= live) continue;
                  if (p.page_groups > 0) {  // 8-row groups of the whole pool are evenly spaced
                    tma_load_5d(dst + row * (128 * kBlocksD), map, &full[stage], 0, 0, 0, it.hkv,
                                pg[u] * p.page_groups + (slot[u] >> 3));
                  } else {
#pragma unroll
                    for (int kb = 0; kb < kBlocksD; ++kb)
                      tma_load_5d(dst + (row >> 3) * (1024 * kBlocksD) + kb * 1024 + (row & 7) * 128, map,
                                  &full[stage], kb * 64, slot[u], 0, it.hkv, pg[u]);
                  }
                }
              }
            }
          }
          if (is_k && j == max(lo, hi - 2)) at = take_place();
        }
        if (is_k) hand_on(read_item(false), i + 1);
      }
    }
  } else if (warp == kQkWarp) {
    // ---------------- S = Q K^T ----------------
    // The whole warp runs the loop (every lane waits on the barriers); the elected lane alone issues.
    const bool elected = elect_one_sync();
    constexpr uint32_t kStageUnits = Shape::kTileBytes >> 4;
    const uint64_t qdesc = make_smem_desc_sw128(smem_u32(sQ), 16, 1024);
    const uint64_t kdesc0 = make_smem_desc_sw128(smem_u32(sK), 16, kGroup);
    int g = 0;
    for (int i = 0;; ++i) {
      PackedItem it;
      take_item(i, &it);
      free_item(i);
      if (it.count <= 0) break;
      wait(&bars->q_full, i & 1, 82);
      for (int j = it.lo; j < it.hi; ++j, ++g) {
        const int stage = g % kStages;
        wait(&bars->k_full[stage], (g / kStages) & 1, 82);
        wait(&bars->s_free[g & 1], ((g >> 1) & 1) ^ 1, 82);
        // The lanes meet before anything is issued that lets a barrier they wait on complete its next phase.
        const bool run = __all_sync(0xffffffffu, !lost) && elected;
        tc_fence_after();
        const uint64_t kd = kdesc0 + static_cast<uint64_t>(stage * kStageUnits);
        const uint32_t d = tmem_base + (g & 1) * 64;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          mma_ss_if(run, d,
                    qdesc + static_cast<uint64_t>((ks / 4) * (Shape::kQBlockBytes >> 4) + (ks % 4) * 2),
                    kd + static_cast<uint64_t>((ks / 4) * (kHalf >> 4) + (ks % 4) * 2),
                    kIdescQK, ks > 0 ? 1u : 0u);
        tc_commit_if(run, &bars->s_full[g & 1]);
        tc_commit_if(run, &bars->k_empty[stage]);
        tc_commit_if(run && j + 1 == it.hi, &bars->q_empty);
      }
    }
  } else if (warp == kPvWarp) {
    // ---------------- O += P V ----------------
    const bool elected = elect_one_sync();
    constexpr uint32_t kStageUnits = Shape::kTileBytes >> 4;
    const uint64_t vdesc0 = make_smem_desc_sw128(smem_u32(sV), kHalf, kGroup);
    const uint32_t o_col = tmem_base + kColO;
    int g = 0;
    for (int i = 0;; ++i) {
      PackedItem it;
      take_item(i, &it);
      free_item(i);
      if (it.count <= 0) break;
      const bool fine = is_fine(it);
      if (i > 0) wait(&bars->o_empty, (i - 1) & 1, 88);
      for (int j = it.lo; j < it.hi; ++j, ++g) {
        const int stage = g % kStages;
        wait(&bars->v_full[stage], (g / kStages) & 1, 88);
        wait(&bars->p_full[g & 1], (g >> 1) & 1, 88);
        const bool run = __all_sync(0xffffffffu, !lost) && elected;
        tc_fence_after();
        const uint64_t vd = vdesc0 + static_cast<uint64_t>(stage * kStageUnits);
        const uint32_t a = tmem_base + (g & 1) * 64;
#pragma unroll
        for (int ks = 0; ks < kPackedKeys / 16; ++ks)
          mma_ts_if(run, o_col, a + ks * 8, vd + static_cast<uint64_t>(ks * (2 * kGroup >> 4)), kIdescPV,
                    ks > 0 || j > it.lo ? 1u : 0u);
        if (fine) {
#pragma unroll
          for (int ks = 0; ks < kPackedKeys / 16; ++ks)
            mma_ts_if(run, o_col, a + 32 + ks * 8, vd + static_cast<uint64_t>(ks * (2 * kGroup >> 4)), kIdescPV, 1u);
        }
        tc_commit_if(run, &bars->s_free[g & 1]);
        tc_commit_if(run, &bars->v_empty[stage]);
        // Completion points the softmax warps may wait on: the second-to-last PV (for a rescale in the last
        // block) and the last one (for the epilogue).
        tc_commit_if(run && j + 2 == it.hi, &bars->pv_done);
        tc_commit_if(run && j + 1 == it.hi, &bars->o_final);
      }
    }
  } else if (warp < 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    // ---------------- softmax warps ----------------
    const int row = warp * 32 + lane;  // of the tile == tensor-memory lane
    const uint32_t lane_addr = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t s_base = tmem_base + lane_addr;
    const uint32_t o_addr = tmem_base + lane_addr + kColO;
    int g = 0, twos = 0;  // blocks; items of two or more

    auto rescale_o = [&](int c, float alpha) {
      uint32_t orr[32];
      tmem_ld_32x32b_x32(o_addr + c * 32, orr);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; ++i) orr[i] = __float_as_uint(__uint_as_float(orr[i]) * alpha);
      tmem_st_32x32b_x32(o_addr + c * 32, orr);
    };

    for (int i = 0;; ++i) {
      // (Only what the block loop needs is held in registers; the rest is read again behind it. With all the
      // SM's memory taken as shared memory a spilled register comes from L2.)
      int nblk, c0, c_lo, c_hi, m, rows;
      bool fine;
      {
        PackedItem it;
        take_item(i, &it);
        it.count = warp_uniform(it.count);
        if (it.count <= 0) break;
        rows = it.count * p.G;
        fine = warp_uniform(is_fine(it)) != 0;
        nblk = warp_uniform(it.hi - it.lo);
        c0 = warp_uniform(it.lo) * kPackedKeys;
        m = warp_uniform(it.m);
        // Keys that this row sees: [c_lo, c_hi].
        const int tok = row < rows ? static_cast<int>(p.div_g.div(row)) : 0;
        c_lo = 0, c_hi = m - 1;
        if constexpr (KIND == kPackedPrefix) {
          if (row < rows) c_hi = min(c_hi, max(p.kv_lens[it.q_row + tok], 0) - 1);
        } else {
          const int last = it.pos + tok;
          if (p.mask_kind != LF_MASK_NONE) c_hi = min(c_hi, last);
          if (p.mask_kind == LF_MASK_CAUSAL_WINDOW) c_lo = max(0, last - (p.window - 1));
        }
      }
      bool valid = row < rows;
      const bool idle = warp_uniform(warp * 32) >= rows;  // no row of this warp is one of the tile's
      float m_used = p.m_first;  // reference that P and O are scaled by (log2 domain)
      float l_run = 0.f;

      for (int k = 0; k < nblk; ++k, ++g, c0 += kPackedKeys) {
        const uint32_t s_addr = s_base + (g & 1) * 64;
        wait(&bars->s_full[g & 1], (g >> 1) & 1, 83);
        tc_fence_after();
        if (c0 + kPackedKeys > m) {
          // V rows past the last key become zeros (the stage's next fill waits for this block's PV).
          const int stage = g % kStages;
          wait(&bars->v_full[stage], (g / kStages) & 1, 84);
          unsigned char* v = sV + stage * Shape::kTileBytes;
          const int first = m - c0;  // (0 < first < 64)
          for (int e = first * 8 + row; e < kPackedKeys * 8; e += 128)
#pragma unroll
            for (int kb = 0; kb < kBlocksD; ++kb)
              *reinterpret_cast<uint4*>(v + kb * kHalf + (e >> 6) * kGroup + (e & 63) * 16) =
                  make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
        }
        if (!idle) {
          uint32_t sr[2][32];
          tmem_ld_32x32b_x32(s_addr, sr[0]);
          tmem_ld_32x32b_x32(s_addr + 32, sr[1]);
          tmem_wait_ld();

          if constexpr (SOFTCAP) {
            // tanh(x), x = raw * a: x (1 - x^2 / 3) up to |x| = 0.125 (error below 4.1e-6), its series to
            // x^7 up to 0.4 (below 6e-6), the unit's approximation beyond. The warp takes the form that its largest
            // score asks for; columns past the last key (other requests' rows, or whatever was in the stage) have
            // no say in it, nor have rows that see no key.
            if (c0 + kPackedKeys > m) {
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (c * 32 + e >= m - c0) sr[c][e] = 0u;
            }
            const bool sees = valid && c_hi >= 0;
            float mx[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                mx[2 * c] = max3(mx[2 * c], fabsf(__uint_as_float(sr[c][e])),
                                 fabsf(__uint_as_float(sr[c][e + 1])));
                mx[2 * c + 1] = max3(mx[2 * c + 1], fabsf(__uint_as_float(sr[c][e + 2])),
                                     fabsf(__uint_as_float(sr[c][e + 3])));
              }
            const float bound = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * fabsf(p.a);
            const float a2 = p.a * p.a;
            const float b1 = a2 * (-1.f / 3.f);
            if (!__any_sync(0xffffffffu, sees && !(bound <= 0.125f))) {
              const uint64_t a_2 = pack2(p.a, p.a), b_2 = pack2(b1 * p.a, b1 * p.a);
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                  const uint64_t r = pack2u(sr[c][e], sr[c][e + 1]);
                  float t0, t1;
                  unpack2(mul2(r, fma2(mul2(r, r), b_2, a_2)), t0, t1);
                  sr[c][e] = __float_as_uint(t0);
                  sr[c][e + 1] = __float_as_uint(t1);
                }
            } else if (!__any_sync(0xffffffffu, sees && !(bound <= 0.4f))) {
              const float b2 = a2 * a2 * (2.f / 15.f);
              const float b3 = a2 * a2 * a2 * (-17.f / 315.f);
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float r = __uint_as_float(sr[c][e]), y = r * r;
                  sr[c][e] = __float_as_uint((r * p.a) * fmaf(fmaf(fmaf(y, b3, b2), y, b1), y, 1.f));
                }
            } else {
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  sr[c][e] = __float_as_uint(tanh_approx(__uint_as_float(sr[c][e]) * p.a));
            }
          }

          const int rel_lo = c_lo - c0, rel_hi = c_hi - c0;  // visible columns of this row in the block
          if (__any_sync(0xffffffffu, valid && (rel_lo > 0 || rel_hi < kPackedKeys - 1))) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              // Bit e: column c * 32 + e is visible (shifts by 32 and more give 0).
              uint32_t seen, upto;
              asm("shl.b32 %0, 0xffffffff, %1;" : "=r"(seen) : "r"(max(rel_lo - c * 32, 0)));
              asm("shl.b32 %0, 0xfffffffe, %1;" : "=r"(upto) : "r"(max(rel_hi - c * 32, 0)));
              seen = rel_hi < c * 32 ? 0u : seen & ~upto;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(seen & (1u << e))) sr[c][e] = 0xff800000u;  // -inf
            }
          }
          // Where every row of the warp has a reference, P is taken against it without looking for the
          // block's maximum first; P may then exceed 1, which bf16 and fp32 hold as exactly as any other
          // magnitude (a row sum past 2^14 takes the other pass). Row sums are taken over the bf16 that the
          // PV product sees: numerator and denominator carry the same rounding, and a row that one key
          // dominates has none.
          uint32_t pk[32];
          bool own_max = __any_sync(0xffffffffu, fine || (valid && m_used == -INFINITY));
          if (!own_max) {
            float fs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float p0 = ex2_approx(fmaf(__uint_as_float(sr[c][e]), p.c2, -m_used));
                const float p1 = ex2_approx(fmaf(__uint_as_float(sr[c][e + 1]), p.c2, -m_used));
                const uint32_t pkv = pack_bf16x2(p0, p1);
                pk[c * 16 + (e >> 1)] = pkv;
                if ((e >> 1) & 1) add_bf16x2_to_f32(fs[2], fs[3], pkv);
                else add_bf16x2_to_f32(fs[0], fs[1], pkv);
                if (e == 30) tmem_st_32x32b_x16(s_addr + c * 16, pk + c * 16);
              }
            const float sum = (fs[0] + fs[1]) + (fs[2] + fs[3]);
            own_max = __any_sync(0xffffffffu, valid && !(sum <= 16384.f));
            if (!own_max) l_run += sum;
          }
          if (own_max) {
            tmem_wait_st();
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                mx[2 * c] = max3(mx[2 * c], __uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1]));
                mx[2 * c + 1] = max3(mx[2 * c + 1], __uint_as_float(sr[c][e + 2]),
                                     __uint_as_float(sr[c][e + 3]));
              }
            const float m_new = fmaxf(m_used, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.c2);
            float alpha = 1.f;  // lazy rescale: the reference moves only when it is passed by 2^8
            if (m_new > -INFINITY && (m_used == -INFINITY || m_new - m_used > 8.f)) {
              alpha = ex2_approx(m_used - m_new);
              m_used = m_new;
            }
            if (k > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
              // O must hold every PV up to the block before: QK(g+1) is issued behind PV(g-1), so "S(g+1) is
              // ready" says so; behind an item's last block that may be another item's, or none.
              const bool last = k + 1 == nblk;
              wait(last ? &bars->pv_done : &bars->s_full[(g + 1) & 1],
                   last ? (twos & 1) : (((g + 1) >> 1) & 1), 85);
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) rescale_o(c, alpha);
            }
            const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
            float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float p0 = ex2_approx(fmaf(__uint_as_float(sr[c][e]), p.c2, neg_m));
                const float p1 = ex2_approx(fmaf(__uint_as_float(sr[c][e + 1]), p.c2, neg_m));
                const uint32_t pkv = pack_bf16x2(p0, p1);
                pk[c * 16 + (e >> 1)] = pkv;
                if ((e >> 1) & 1) add_bf16x2_to_f32(ps[2], ps[3], pkv);
                else add_bf16x2_to_f32(ps[0], ps[1], pkv);
              }
            if (fine) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                uint32_t rest[16];
#pragma unroll
                for (int f = 0; f < 16; ++f) {
                  const float p0 = ex2_approx(fmaf(__uint_as_float(sr[c][2 * f]), p.c2, neg_m));
                  const float p1 = ex2_approx(fmaf(__uint_as_float(sr[c][2 * f + 1]), p.c2, neg_m));
                  const uint32_t hi = pk[c * 16 + f];
                  rest[f] = pack_bf16x2(p0 - bf16lo_to_f32(hi), p1 - bf16hi_to_f32(hi));
                  add_bf16x2_to_f32(ps[f & 2], ps[(f & 2) + 1], rest[f]);
                }
                tmem_st_32x32b_x16(s_addr + 32 + c * 16, rest);
              }
            }
            l_run = fmaf(l_run, alpha, (ps[0] + ps[1]) + (ps[2] + ps[3]));
            tmem_st_32x32b_x32(s_addr, pk);
          }
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[g & 1]);
      }

      // ---------------- epilogue ----------------
      wait(&bars->o_final, i & 1, 86);
      if (nblk > 1) ++twos;
      tc_fence_after();
      const PackedItem& it = bars->item[i % kItemSlots];
      const int row_tok = static_cast<int>(p.div_g.div(row));
      const int head = row - row_tok * p.G;  // of the kv head's query heads
      const bool sliced = KIND == kPackedPrefix || warp_uniform(it.part) >= 0;
      // Rows of O: un-normalised with their (reference, sum) for the join, or the output (a row is D / 16 whole
      // sectors of 32 bytes; one that saw no key is zeros).
      const bool empty = l_run == 0.f;
      const float inv = empty ? 0.f : 1.f / l_run;
      if (valid && !LF_BOUNDS(it.q_row >= 0 && it.q_row + row_tok < (KIND == kPackedPrefix ? p.B : p.T) &&
                                  it.hkv >= 0 && it.hkv < p.Hkv && head < p.G,
                              p.status, 71))
        valid = false;
      float* part = nullptr;
      __nv_bfloat16* dst = nullptr;
      if (valid) {
        if (!sliced) {
          dst = p.out + static_cast<int64_t>(it.q_row + row_tok) * p.o_stride[0] +
                static_cast<int64_t>(it.hkv * p.G + head) * p.o_stride[1];
        } else {
          int64_t at;
          if constexpr (KIND == kPackedPrefix) {
            at = static_cast<int64_t>(it.index) * p.B * p.Hkv * p.G +
                 (static_cast<int64_t>(it.q_row + row_tok) * p.Hkv + it.hkv) * p.G + head;
          } else {
            at = (static_cast<int64_t>(it.part + it.index) * p.Hkv + it.hkv) * kPackedRows + row;
          }
          p.part_ml[at] = make_float2(m_used, l_run);
          part = p.part_o + at * D;
        }
      }
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (!idle) {
          tmem_ld_32x32b_x32(o_addr + c, o);
          tmem_wait_ld();
        }
        if (c + 32 == D) {  // the next item's first PV may overwrite O
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->o_empty);
        }
        if (sliced) {
          if (valid) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) stg_32(part + c + e, &o[e]);
          }
        } else if (valid) {
#pragma unroll
          for (int e = 0; e < 32; e += 16) {
            uint32_t w[8];
#pragma unroll
            for (int f = 0; f < 8; ++f)
              w[f] = empty ? 0u
                           : pack_bf16x2(__uint_as_float(o[e + 2 * f]) * inv,
                                         __uint_as_float(o[e + 2 * f + 1]) * inv);
            if (p.out_sectors) {
              stg_32(dst + c + e, w);
            } else {
              *reinterpret_cast<uint4*>(dst + c + e) = make_uint4(w[0], w[1], w[2], w[3]);
              *reinterpret_cast<uint4*>(dst + c + e + 8) = make_uint4(w[4], w[5], w[6], w[7]);
            }
          }
        }
      }
      if constexpr (KIND != kPackedPrefix) {
        if (sliced) {
          // The CTA that finishes the last slice of a tile joins them all, in order.
          __threadfence();
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (threadIdx.x == 0)
            bars->last_part = atomicAdd(&p.list[2 + it.counter * p.Hkv + it.hkv], 1u) + 1u ==
                              static_cast<uint32_t>(it.n_parts);
          asm volatile("bar.sync 1, 128;" ::: "memory");
          const bool join = warp_uniform(bars->last_part) != 0;
          asm volatile("bar.sync 1, 128;" ::: "memory");  // (the word is free again)
          if (join && !idle) {
            __threadfence();
            join_slices<D>(p, it, warp, lane, rows);
          }
        }
      }
      free_item(i);
    }
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Shape::kTmemColumns);
  }
}

// ---------------------------------------------------------------------------------------
// Host side, shared by both
// ---------------------------------------------------------------------------------------
// Score function of a call: multipliers only, or (multipliers) tanh (multipliers). Other chains have no
// kernel here.
struct PackedScore {
  bool softcap = false;
  float a = 1.f, c2 = 1.f;
  float m_first = -INFINITY;
};

inline int packed_score(float scale, int n_mod, const int32_t* op, const float* arg, PackedScore* s) {
  if (n_mod < 0 || n_mod > LF_MAX_MODS) return LF_ERR_INVALID_ARG;
  int i = 0;
  auto fold = [&](float x) {
    for (; i < n_mod && (op[i] == LF_MOD_MUL || op[i] == LF_MOD_DIV); ++i)
      x = op[i] == LF_MOD_MUL ? x * arg[i] : x / arg[i];
    return x;
  };
  const float pre = fold(scale);
  s->softcap = i < n_mod && op[i] == LF_MOD_TANH;
  if (s->softcap) {
    ++i;
    const float post = fold(1.f);
    // (tanh is odd: a negative factor behind it changes sides)
    s->a = post < 0.f ? -pre : pre;
    s->c2 = fabsf(post);
  } else {
    s->c2 = pre;
  }
  // (The series of tanh takes powers of `a` up to the sixth.)
  if (i < n_mod || !(s->c2 >= 0.f) || !(s->c2 < 1e30f) || !(fabsf(s->a) < 1e6f)) return LF_ERR_UNSUPPORTED;
  // (A factor of zero, or below the normal numbers, would turn masked scores into NaN.)
  s->c2 = fmaxf(s->c2 * kPackedLog2e, FLT_MIN);
  // Capped logits lie within c2 of zero: up to 80, rows can begin with the reference 0 instead of looking
  // for their first maximum (P from 2^-80; a row sum past 2^14 moves the reference as usual).
  if (s->softcap && s->c2 <= 80.f) s->m_first = 0.f;
  return LF_OK;
}

// Largest power of two that divides the page, up to a block: a copy of that many keys stays in one page.
inline int packed_box(int page_size) {
  int box = 1;
  while (box < kPackedKeys && page_size % (box * 2) == 0) box *= 2;
  return box;
}

// Maps of the pools [n_pages, page_size, Hkv, D] with strides (page, slot, kv head). Where both pools' groups
// of 8 slots are evenly spaced through all pages, a copy moves the groups of p->box slots with all their
// columns, by (column, slot of the group, half, kv head, group); else p->box slots of a group and 64 columns,
// by (column, slot, -, kv head, page), and p->page_groups is 0.
inline int packed_pool_maps(CUtensorMap* mk, CUtensorMap* mv, const void* k, const void* v,
                            const int64_t* k_st, const int64_t* v_st, int n_pages, int page_size, int Hkv,
                            int D, PackedParams* p) {
  const int64_t groups = static_cast<int64_t>(n_pages) * (page_size / 8);
  const bool even = page_size % 8 == 0 && groups < (1ll << 31) &&
                    (n_pages == 1 || (k_st[0] == k_st[1] * page_size && v_st[0] == v_st[1] * page_size));
  p->page_groups = even ? page_size / 8 : 0;
  p->box = packed_box(page_size);
  if (!even && p->box > 8) p->box = 8;
  p->box_shift = shift_of(p->box);
  for (int i = 0; i < 2; ++i) {
    const int64_t* st = i ? v_st : k_st;
    TileMapSpec spec;
    if (even)
      spec = {i ? v : k, {64, 8, D / 64, Hkv, groups}, {st[1], 64, st[2], 8 * st[1]}, {8, D / 64, 1, p->box / 8}};
    else
      spec = {i ? v : k, {D, page_size, 1, Hkv, n_pages}, {st[1], 0, st[2], st[0]}, {p->box, 1, 1, 1}};
    const int rc = make_map_5d(i ? mv : mk, spec);
    if (rc != LF_OK) return rc;
  }
  return LF_OK;
}

template <class Kernel>
inline int packed_configure(Kernel kernel, size_t smem, int* configured_dev) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (*configured_dev == dev) return LF_OK;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) {
    set_cuda_error(e, "cudaFuncSetAttribute(packed kernel)");
    return LF_ERR_CUDA;
  }
  *configured_dev = dev;
  return LF_OK;
}

}  // namespace lf

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
// One CTA per tile, two CTAs per SM: the start and end of one lie under the blocks of the other, which
// is what short requests are made of. 256 threads:
//   warps 0-3   softmax (one thread per score row)
//   warp  4     producer: Q once, then pairs of 64-key tiles into a ring, in the order of their use:
//               {K(lo), K(lo+1)}, {V(lo), K(lo+2)}, {V(lo+1), K(lo+3)}, ...
//   warp  5     MMA issuer: S[buf] = Q K^T, O += P V; QK of block j+2 is issued right behind PV of block j
// Tensor memory (256 columns): S of buffer b at column b * 64, P (bf16) over its first 32 columns, O at 128.
//
// What a packed batch adds to the tiles of the prefill kernels: the last key block of a request holds
// rows of the next one (or, in a page, of whoever had it before). Their scores are masked; their V rows
// are zeroed in shared memory by the softmax warps before P V, since 0 * infinity or 0 * NaN of a
// stranger would reach every row.
#pragma once

#include "lf_common.cuh"
#include "lf_tensor_map.h"

#include <float.h>

namespace lf {

constexpr int kPackedRows = 128;  // of a tile
constexpr int kPackedKeys = 64;   // of a block
constexpr int kPackedThreads = 256;
constexpr float kPackedLog2e = 1.4426950408889634f;

// Where a tile's rows and keys come from.
enum PackedKind {
  kPackedDense = 0,   // packed queries, packed keys
  kPackedPaged = 1,   // packed queries, keys through a block table
  kPackedPrefix = 2,  // one query token per request against a slice of the shared prefix; partial results
};

struct PackedParams {
  __nv_bfloat16* out;
  int64_t o_stride[2];        // (token, head)
  const int32_t* cu_q;        // [B + 1] first query token of each request
  const int32_t* cu_k;        // dense: [B + 1] first key
  const int32_t* kv_lens;     // paged, prefix: [B] keys of each request
  const int32_t* table;       // block table
  int64_t bt_stride;
  const int2* items;          // (request, tile) in the order of the launch, or null: looked up by the CTA
  const int32_t* n_items;     // how many there are
  int32_t B, T, Tk, Hkv, G;
  int32_t tq;                 // tokens (requests) per tile: 128 / G
  int32_t mask_kind, window;
  float a;                    // softcap: score = tanh(raw * a) * c2
  float c2;                   // logit in the log2 domain = score * c2; > 0
  int32_t bt_blocks, page_size, page_shift, n_pages;
  int32_t box;                // keys per copy of a paged operand: they lie in one page
  int32_t n_tiles;            // grid: tiles of a kv head (an upper bound)
  FastDiv div_chunk;          // heads of a chunk of kv heads (see the launch)
  FastDiv div_tiles;          // tiles
  FastDiv div_g;              // query heads per kv head
  // Prefix: rows [B, Hkv, G], keys [split * chunk, ...) below prefix_len.
  int32_t prefix_len, chunk, splits;
  float* part_o;              // [split][row][D]
  float2* part_ml;            // [split][row] (reference, sum)
  int32_t* status;
};

template <int D>
struct PackedShape {
  static constexpr int kStages = D == 64 ? 4 : 2;
  // Output staging (2 KB per softmax warp; with D = 64 the CTA has to stay above a third of the SM's
  // shared memory, so that a third one does not wait for tensor memory).
  static constexpr uint32_t kStaging = 4 * 2048 + 4096;
  static constexpr uint32_t kTmemColumns = 256;
  static constexpr uint32_t kQBlockBytes = kPackedRows * 128;  // [128][64] bf16
  static constexpr uint32_t kKVBlockBytes = kPackedKeys * 128;
  static constexpr uint32_t kTileBytes = kKVBlockBytes * (D / 64);
  static constexpr size_t kSmem = 1024 /*align slack*/ + 1024 /*barriers*/ + kStaging +
                                  kQBlockBytes * (D / 64) + kStages * 2 * kTileBytes;
};

struct __align__(8) PackedBarriers {
  uint64_t q_full;
  uint64_t kv_full[4];
  uint64_t kv_empty[4];
  uint64_t s_full[2];   // MMA -> softmax
  uint64_t p_full[2];   // softmax -> MMA
  uint64_t pv_done;     // second-to-last PV done
  uint64_t o_final;     // last PV done
  uint32_t tmem_base;
};

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
    r.k0 = 0;
    const int64_t held = static_cast<int64_t>(p.bt_blocks) * p.page_size;
    r.m = clamp_to(p.kv_lens[b], held > 0x7fffffff ? 0x7fffffff : static_cast<int>(held));
  }
  return r;
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

template <int D, int KIND, bool SOFTCAP>
__device__ __forceinline__ void packed_tile(const CUtensorMap& tmap_q, const CUtensorMap& tmap_k,
                                            const CUtensorMap& tmap_v, const PackedParams& p,
                                            unsigned char* smem_unaligned, int cta) {
  using Shape = PackedShape<D>;
  constexpr int kStages = Shape::kStages;
  constexpr int kBlocksD = D / 64;
  constexpr uint32_t kIdescQK = make_idesc_bf16(128, kPackedKeys, 0);
  constexpr uint32_t kIdescPV = make_idesc_bf16(128, D, 1);
  constexpr uint32_t kColO = 128;
  constexpr int kProducerWarp = 4, kMmaWarp = 5;
  constexpr bool kPages = KIND != kPackedDense;

  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~static_cast<uintptr_t>(1023));
  PackedBarriers* bars = reinterpret_cast<PackedBarriers*>(smem);
  unsigned char* sStage = smem + 1024;
  unsigned char* sQ = sStage + Shape::kStaging;
  unsigned char* sKV = sQ + Shape::kQBlockBytes * kBlocksD;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  // ---------------- which tile ----------------
  int hkv, t0, count;      // kv head; first token of the tile and how many it has
  int table_row = 0, split = 0;
  PackedRequest rq;
  int key_lo, key_hi;      // keys that some row of the tile sees
  int off = 0;             // query token i sees the keys up to i + off
  if constexpr (KIND == kPackedPrefix) {
    const int unit = static_cast<int>(p.div_tiles.div(cta));  // (kv head, split); tiles of it together
    const int tile = cta - unit * static_cast<int>(p.div_tiles.d);
    split = static_cast<int>(p.div_chunk.div(unit));          // div_chunk: kv heads
    hkv = unit - split * static_cast<int>(p.div_chunk.d);
    t0 = tile * p.tq;
    count = min(p.tq, p.B - t0);
    rq = {0, p.B, 0, 0};
    key_lo = split * p.chunk;
    key_hi = min(p.prefix_len, key_lo + p.chunk);
    rq.m = key_hi;
  } else {
    const int r = static_cast<int>(p.div_chunk.div(cta));     // place in the order of this chunk of heads
    const int head_chunk = static_cast<int>(p.div_tiles.div(r));
    hkv = head_chunk * static_cast<int>(p.div_chunk.d) + cta - r * static_cast<int>(p.div_chunk.d);
    if (hkv >= p.Hkv) return;
    const int rank = r - head_chunk * static_cast<int>(p.div_tiles.d);
    int2 at;
    if (p.items) {
      if (rank >= *p.n_items) return;
      at = p.items[rank];
    } else {
      at = find_tile(p, rank);
      if (at.x < 0) return;
    }
    rq = packed_request<KIND>(p, at.x);
    table_row = at.x;
    t0 = at.y * p.tq;
    count = min(p.tq, rq.n - t0);
    off = rq.m - rq.n;
    key_lo = 0;
    key_hi = rq.m;
    if (p.mask_kind != LF_MASK_NONE) key_hi = min(key_hi, t0 + count + off);
    if (p.mask_kind == LF_MASK_CAUSAL_WINDOW) key_lo = max(0, t0 + off - (p.window - 1));
  }
  const int rows = count * p.G;
  // Rows that see a handful of keys do not average the rounding of P away: where the first row of the tile
  // does (the start of a prompt, a tiny window), P enters the second product as two bf16, its rounding and
  // what that leaves, in the half of the S buffer that P does not need.
  bool fine = false;
  if constexpr (KIND != kPackedPrefix) {
    int sees = rq.m;
    if (p.mask_kind != LF_MASK_NONE) sees = min(sees, t0 + off + 1);
    if (p.mask_kind == LF_MASK_CAUSAL_WINDOW) sees = min(sees, p.window);
    fine = sees < 16;
  }
  const int lo = key_lo / kPackedKeys;
  const int hi = key_hi > key_lo ? (key_hi + kPackedKeys - 1) / kPackedKeys : lo;
  const int nblk = hi - lo;

  // ---------------- setup ----------------
  if (warp == kProducerWarp && lane == 0) {
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
    mbar_init(&bars->q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->kv_full[s], 1);
      mbar_init(&bars->kv_empty[s], 1);
    }
    for (int bf = 0; bf < 2; ++bf) {
      mbar_init(&bars->s_full[bf], 1);
      mbar_init(&bars->p_full[bf], 4);
    }
    mbar_init(&bars->pv_done, 1);
    mbar_init(&bars->o_final, 1);
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

  // 128 registers per thread at two CTAs of 256: 184 for the softmax warps, 72 for the others (one
  // instruction per warpgroup, in front of the dispatch of roles).
  if (warp >= 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");

  if (warp == kProducerWarp) {
    // ---------------- producer ----------------
    const bool elected = elect_one_sync();
    if (nblk > 0) {
      if (elected) {
        // (A box is always tq tokens; those past the end of the request are strangers' rows or zeros.)
        mbar_arrive_expect_tx(&bars->q_full, static_cast<uint32_t>(p.tq * p.G) * 128 * kBlocksD);
#pragma unroll
        for (int kb = 0; kb < kBlocksD; ++kb)
          tma_load_4d(sQ + kb * Shape::kQBlockBytes, &tmap_q, &bars->q_full, kb * 64, 0, hkv,
                      rq.q0 + t0);
      }
      bool ok = true;
      auto page_of = [&](int t) { return p.page_shift >= 0 ? (t >> p.page_shift) : (t / p.page_size); };
      const int32_t* table = p.table + static_cast<int64_t>(table_row) * p.bt_stride;
      const int boxes = kPages ? kPackedKeys / p.box : 1;
      // Boxes of block j that hold a key (the rest of the last block is not fetched).
      auto live_boxes = [&](int j) {
        return min(boxes, (rq.m - j * kPackedKeys + p.box - 1) / p.box);
      };
      // Table entries of a block's boxes, one or two per lane, requested a block ahead of their use.
      auto request = [&](int j, int32_t (&e)[2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = i * 32 + lane;
          e[i] = 0;
          if (j < hi && r < live_boxes(j)) e[i] = table[page_of(j * kPackedKeys + r * p.box)];
        }
      };
      // Block j of K or V into `dst`. Paged: the page ids are checked, then the elected lane issues a copy
      // per box.
      auto load = [&](const CUtensorMap* map, unsigned char* dst, uint64_t* bar, int j, int32_t (&e)[2]) {
        if constexpr (!kPages) {
          if (elected) {
#pragma unroll
            for (int kb = 0; kb < kBlocksD; ++kb)
              tma_load_4d(dst + kb * Shape::kKVBlockBytes, map, bar, kb * 64, rq.k0 + j * kPackedKeys,
                          hkv, 0);
          }
        } else {
          const int live = live_boxes(j);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (i * 32 + lane < live && (e[i] < 0 || e[i] >= p.n_pages)) {
              if (p.status) atomicExch(p.status, LF_DEV_BAD_PAGE);
              e[i] = 0;
            }
          }
          for (int r = 0; r < live; ++r) {
            const int page = __shfl_sync(0xffffffffu, r < 32 ? e[0] : e[1], r & 31);
            const int t = j * kPackedKeys + r * p.box;
            const int slot = t - page_of(t) * p.page_size;
            if (elected) {
#pragma unroll
              for (int kb = 0; kb < kBlocksD; ++kb)
                tma_load_4d(dst + kb * Shape::kKVBlockBytes + r * p.box * 128, map, bar, kb * 64, slot,
                            hkv, page);
            }
          }
        }
      };
      auto bytes = [&](int j) -> uint32_t {
        return kPages ? static_cast<uint32_t>(live_boxes(j) * p.box) * 128 * kBlocksD : Shape::kTileBytes;
      };
      int32_t ek[2] = {0, 0}, ek2[2] = {0, 0}, ev[2] = {0, 0};
      // Entries of the blocks whose V is still to come: those of K(j), K(j+1) serve V again.
      if constexpr (kPages) {
        request(lo, ev);
        request(lo + 1, ek);
        request(lo + 2, ek2);
      }
      {
        if (elected) mbar_arrive_expect_tx(&bars->kv_full[0], bytes(lo) + (nblk > 1 ? bytes(lo + 1) : 0u));
        load(&tmap_k, sKV, &bars->kv_full[0], lo, ev);
        if (nblk > 1) load(&tmap_k, sKV + Shape::kTileBytes, &bars->kv_full[0], lo + 1, ek);
      }
      for (int j = lo, n = 1; j < hi && ok; ++j, ++n) {
        const int stage = n % kStages;
        ok = mbar_wait(&bars->kv_empty[stage], ((n / kStages) & 1) ^ 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          packed_timeout(p.status, 81);
          break;
        }
        unsigned char* dst = sKV + stage * (2 * Shape::kTileBytes);
        const bool more = j + 2 < hi;
        if (elected)
          mbar_arrive_expect_tx(&bars->kv_full[stage], bytes(j) + (more ? bytes(j + 2) : 0u));
        load(&tmap_v, dst, &bars->kv_full[stage], j, ev);
        if (more) load(&tmap_k, dst + Shape::kTileBytes, &bars->kv_full[stage], j + 2, ek2);
        if constexpr (kPages) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            ev[i] = ek[i];
            ek[i] = ek2[i];
          }
          request(j + 3, ek2);
        }
      }
    }
  } else if (warp == kMmaWarp) {
    // ---------------- MMA issuer ----------------
    // The whole warp runs the loop (every lane waits on the barriers); the elected lane alone issues.
    if (nblk > 0) {
      const bool elected = elect_one_sync();
      bool ok = __all_sync(0xffffffffu, mbar_wait(&bars->q_full, 0));
      constexpr uint32_t kStageUnits = (2 * Shape::kTileBytes) >> 4;
      constexpr uint32_t kHalfUnits = Shape::kTileBytes >> 4;
      const uint64_t qdesc = make_smem_desc_sw128(smem_u32(sQ), 16, 1024);
      const uint64_t kdesc0 = make_smem_desc_sw128(smem_u32(sKV), 16, 1024);
      const uint64_t vdesc0 = make_smem_desc_sw128(smem_u32(sKV), Shape::kKVBlockBytes, 1024);
      const uint32_t o_col = tmem_base + kColO;
      auto wait_stage = [&](int n) {
        if (!mbar_wait(&bars->kv_full[n % kStages], (n / kStages) & 1)) ok = false;
        return n % kStages;
      };
      auto issue_qk = [&](int stage, int half, int kt) {
        const uint64_t kd = kdesc0 + static_cast<uint64_t>(stage * kStageUnits + half * kHalfUnits);
        const uint32_t d = tmem_base + (kt & 1) * 64;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          mma_ss_if(elected, d,
                    qdesc + static_cast<uint64_t>((ks / 4) * (Shape::kQBlockBytes >> 4) + (ks % 4) * 2),
                    kd + static_cast<uint64_t>((ks / 4) * (Shape::kKVBlockBytes >> 4) + (ks % 4) * 2),
                    kIdescQK, ks > 0 ? 1u : 0u);
        tc_commit_if(elected, &bars->s_full[kt & 1]);
      };
      if (ok) {
        const int st = wait_stage(0);
        tc_fence_after();
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
          issue_qk(st, 0, 0);
          if (nblk > 1) issue_qk(st, 1, 1);
          tc_commit_if(elected, &bars->kv_empty[st]);
        }
      }
      __syncwarp();
      for (int kt = 0; kt < nblk && ok; ++kt) {
        const int st = wait_stage(kt + 1);  // {V(kt), K(kt + 2)}
        if (ok) ok = mbar_wait(&bars->p_full[kt & 1], (kt >> 1) & 1);
        tc_fence_after();
        const uint64_t vd = vdesc0 + static_cast<uint64_t>(st * kStageUnits);
        const bool run = elected && ok;
#pragma unroll
        for (int ks = 0; ks < kPackedKeys / 16; ++ks)
          mma_ts_if(run, o_col, tmem_base + (kt & 1) * 64 + ks * 8,
                    vd + static_cast<uint64_t>(ks * (2048 >> 4)), kIdescPV, (kt > 0 || ks > 0) ? 1u : 0u);
        if (fine) {
#pragma unroll
          for (int ks = 0; ks < kPackedKeys / 16; ++ks)
            mma_ts_if(run, o_col, tmem_base + (kt & 1) * 64 + 32 + ks * 8,
                      vd + static_cast<uint64_t>(ks * (2048 >> 4)), kIdescPV, 1u);
        }
        // Completion points the softmax warps may wait on: the second-to-last PV (for a rescale in the
        // last block) and the last one (for the epilogue).
        tc_commit_if(run && kt == nblk - 2, &bars->pv_done);
        tc_commit_if(run && kt == nblk - 1, &bars->o_final);
        // The lanes meet before anything is issued that lets a barrier they wait on complete its next
        // phase, and leave together when a wait ran out.
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (kt + 2 < nblk) issue_qk(st, 1, kt + 2);
        tc_commit_if(elected, &bars->kv_empty[st]);
      }
      if (!ok) packed_timeout(p.status, 82);
    }
  } else if (warp < 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    // ---------------- softmax warps ----------------
    const int row = warp * 32 + lane;  // of the tile == tensor-memory lane
    const bool valid = row < rows;
    const int row_tok = static_cast<int>(p.div_g.div(valid ? row : 0));
    const int head = row - row_tok * p.G;  // of the kv head's query heads
    const int tok = t0 + row_tok;
    const uint32_t lane_addr = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t s_base = tmem_base + lane_addr;
    const uint32_t o_addr = tmem_base + lane_addr + kColO;
    // Keys that this row sees: [c_lo, c_hi].
    int c_lo = 0, c_hi = key_hi - 1;
    if constexpr (KIND == kPackedPrefix) {
      if (valid) c_hi = min(c_hi, p.kv_lens[tok] - 1);
    } else {
      if (p.mask_kind != LF_MASK_NONE) c_hi = min(rq.m - 1, tok + off);
      if (p.mask_kind == LF_MASK_CAUSAL_WINDOW) c_lo = max(0, tok + off - (p.window - 1));
    }
    float m_used = -INFINITY;  // reference that P and O are scaled by (log2 domain)
    float l_run = 0.f;
    bool ok = true;
    const bool idle = warp * 32 >= rows;  // no row of this warp is one of the tile's

    auto rescale_o = [&](int c, float alpha) {
      uint32_t orr[32];
      tmem_ld_32x32b_x32(o_addr + c * 32, orr);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; ++i) orr[i] = __float_as_uint(__uint_as_float(orr[i]) * alpha);
      tmem_st_32x32b_x32(o_addr + c * 32, orr);
    };
    for (int k = 0; k < nblk && ok; ++k) {
      const int c0 = (lo + k) * kPackedKeys;
      const int buf = k & 1;
      const uint32_t s_addr = s_base + buf * 64;
      if (!mbar_wait(&bars->s_full[buf], (k >> 1) & 1)) {
        packed_timeout(p.status, 83);
        ok = false;
        break;
      }
      tc_fence_after();
      if (c0 + kPackedKeys > rq.m) {
        // V rows past the last key become zeros (the stage's next fill waits for this block's PV).
        const int stage = (k + 1) % kStages;
        if (!mbar_wait(&bars->kv_full[stage], ((k + 1) / kStages) & 1)) {
          packed_timeout(p.status, 84);
          ok = false;
          break;
        }
        unsigned char* v = sKV + stage * (2 * Shape::kTileBytes);
        const int first = rq.m - c0;  // (0 < first < 64)
        for (int i = first * 8 + row; i < kPackedKeys * 8; i += 128)
#pragma unroll
          for (int kb = 0; kb < kBlocksD; ++kb)
            *reinterpret_cast<uint4*>(v + kb * Shape::kKVBlockBytes + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
      }
      if (!idle) {
        uint32_t sr[2][32];
        tmem_ld_32x32b_x32(s_addr, sr[0]);
        tmem_ld_32x32b_x32(s_addr + 32, sr[1]);
        tmem_wait_ld();
        const int rel_lo = c_lo - c0, rel_hi = c_hi - c0;  // visible columns of this row in the block
        const bool masked = valid && (rel_lo > 0 || rel_hi < kPackedKeys - 1);

        if constexpr (SOFTCAP) {
          // tanh(x), x = raw * a: x (1 - x^2 / 3) up to |x| = 0.125 (error below 4.1e-6), its series to
          // x^7 up to 0.4 (below 6e-6), the unit's approximation beyond.
          float mx[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              mx[2 * c] = max3(mx[2 * c], fabsf(__uint_as_float(sr[c][i])),
                               fabsf(__uint_as_float(sr[c][i + 1])));
              mx[2 * c + 1] = max3(mx[2 * c + 1], fabsf(__uint_as_float(sr[c][i + 2])),
                                   fabsf(__uint_as_float(sr[c][i + 3])));
            }
          const float bound = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * fabsf(p.a);
          const float a2 = p.a * p.a;
          const float b1 = a2 * (-1.f / 3.f);
          if (!__any_sync(0xffffffffu, valid && !(bound <= 0.125f))) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float r = __uint_as_float(sr[c][i]);
                sr[c][i] = __float_as_uint((r * p.a) * fmaf(r * r, b1, 1.f));
              }
          } else if (!__any_sync(0xffffffffu, valid && !(bound <= 0.4f))) {
            const float b2 = a2 * a2 * (2.f / 15.f);
            const float b3 = a2 * a2 * a2 * (-17.f / 315.f);
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float r = __uint_as_float(sr[c][i]), y = r * r;
                sr[c][i] = __float_as_uint((r * p.a) * fmaf(fmaf(fmaf(y, b3, b2), y, b1), y, 1.f));
              }
          } else {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                sr[c][i] = __float_as_uint(tanh_approx(__uint_as_float(sr[c][i]) * p.a));
          }
        }

        // Where every row of the warp has a reference and sees the whole block, P is taken against that
        // reference without looking for the block's maximum first; P may then exceed 1, which bf16 and
        // fp32 hold as exactly as any other magnitude (a row sum past 2^14 takes the other pass). Row sums
        // are taken over the bf16 that the PV product sees: numerator and denominator carry the same
        // rounding, and a row that one key dominates has none.
        uint32_t pk[32];
        bool own_max = __any_sync(0xffffffffu, fine || masked || (valid && m_used == -INFINITY));
        if (!own_max) {
          float fs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float p0 = ex2_approx(fmaf(__uint_as_float(sr[c][i]), p.c2, -m_used));
              const float p1 = ex2_approx(fmaf(__uint_as_float(sr[c][i + 1]), p.c2, -m_used));
              const uint32_t pkv = pack_bf16x2(p0, p1);
              pk[c * 16 + (i >> 1)] = pkv;
              if ((i >> 1) & 1) add_bf16x2_to_f32(fs[2], fs[3], pkv);
              else add_bf16x2_to_f32(fs[0], fs[1], pkv);
            }
          const float sum = (fs[0] + fs[1]) + (fs[2] + fs[3]);
          own_max = __any_sync(0xffffffffu, valid && !(sum <= 16384.f));
          if (!own_max) l_run += sum;
        }
        if (own_max) {
          if (__any_sync(0xffffffffu, masked)) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              // Bit i: column c * 32 + i is visible (shifts by 32 and more give 0).
              uint32_t seen, upto;
              asm("shl.b32 %0, 0xffffffff, %1;" : "=r"(seen) : "r"(max(rel_lo - c * 32, 0)));
              asm("shl.b32 %0, 0xfffffffe, %1;" : "=r"(upto) : "r"(max(rel_hi - c * 32, 0)));
              seen = rel_hi < c * 32 ? 0u : seen & ~upto;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(seen & (1u << i))) sr[c][i] = 0xff800000u;  // -inf
            }
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              mx[2 * c] = max3(mx[2 * c], __uint_as_float(sr[c][i]), __uint_as_float(sr[c][i + 1]));
              mx[2 * c + 1] = max3(mx[2 * c + 1], __uint_as_float(sr[c][i + 2]),
                                   __uint_as_float(sr[c][i + 3]));
            }
          const float m_new = fmaxf(m_used, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.c2);
          float alpha = 1.f;  // lazy rescale: the reference moves only when it is passed by 2^8
          if (m_new > -INFINITY && (m_used == -INFINITY || m_new - m_used > 8.f)) {
            alpha = ex2_approx(m_used - m_new);
            m_used = m_new;
          }
          if (k > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
            // O must hold every PV up to k-1: QK(k+1) is issued behind PV(k-1), so "S(k+1) is ready" says
            // so; in the last block there is no S(k+1).
            const bool last = k + 1 == nblk;
            if (!mbar_wait(last ? &bars->pv_done : &bars->s_full[(k + 1) & 1],
                           last ? 0u : (((k + 1) >> 1) & 1))) {
              packed_timeout(p.status, 85);
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) rescale_o(c, alpha);
          }
          const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
          float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float p0 = ex2_approx(fmaf(__uint_as_float(sr[c][i]), p.c2, neg_m));
              const float p1 = ex2_approx(fmaf(__uint_as_float(sr[c][i + 1]), p.c2, neg_m));
              const uint32_t pkv = pack_bf16x2(p0, p1);
              pk[c * 16 + (i >> 1)] = pkv;
              if ((i >> 1) & 1) add_bf16x2_to_f32(ps[2], ps[3], pkv);
              else add_bf16x2_to_f32(ps[0], ps[1], pkv);
            }
          if (fine) {
            uint32_t rest[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int c = i >> 4, e = (2 * i) & 31;
              const float p0 = ex2_approx(fmaf(__uint_as_float(sr[c][e]), p.c2, neg_m));
              const float p1 = ex2_approx(fmaf(__uint_as_float(sr[c][e + 1]), p.c2, neg_m));
              rest[i] = pack_bf16x2(p0 - bf16lo_to_f32(pk[i]), p1 - bf16hi_to_f32(pk[i]));
              add_bf16x2_to_f32(ps[i & 2], ps[(i & 2) + 1], rest[i]);
            }
            tmem_st_32x32b_x32(s_addr + 32, rest);
          }
          l_run = fmaf(l_run, alpha, (ps[0] + ps[1]) + (ps[2] + ps[3]));
        }
        tmem_st_32x32b_x32(s_addr, pk);
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->p_full[buf]);
    }

    // ---------------- epilogue ----------------
    if (nblk > 0 && ok && !mbar_wait(&bars->o_final, 0)) {
      packed_timeout(p.status, 86);
      ok = false;
    }
    tc_fence_after();
    if (ok && !idle) {
      if constexpr (KIND == kPackedPrefix) {
        // Un-normalised rows and their (reference, sum), for the join with the requests' own keys.
        const int64_t unit = (static_cast<int64_t>(tok) * p.Hkv + hkv) * p.G + head;
        const int64_t at = static_cast<int64_t>(split) * p.B * p.Hkv * p.G + unit;
        if (valid) p.part_ml[at] = make_float2(m_used, l_run);
        float* dst = p.part_o + at * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t orr[32];
          tmem_ld_32x32b_x32(o_addr + c * 32, orr);
          tmem_wait_ld();
          if (valid) {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(
                               dst + c * 32 + i),
                           "r"(orr[i]), "r"(orr[i + 1]), "r"(orr[i + 2]), "r"(orr[i + 3]),
                           "r"(orr[i + 4]), "r"(orr[i + 5]), "r"(orr[i + 6]), "r"(orr[i + 7])
                           : "memory");
          }
        }
      } else {
        // 32 columns of 32 rows at a time go through a swizzled 2 KB buffer of the warp, so that a store
        // instruction writes eight 64-byte row segments. A row that saw no key is zeros.
        const float inv = 1.f / l_run;
        const bool empty = l_run == 0.f || nblk == 0;
        unsigned char* stage = sStage + warp * 2048;
        const int64_t row_off = valid ? static_cast<int64_t>(rq.q0 + tok) * p.o_stride[0] +
                                            static_cast<int64_t>(hkv * p.G + head) * p.o_stride[1]
                                      : -1;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t orr[32];
          tmem_ld_32x32b_x32(o_addr + c * 32, orr);
          tmem_wait_ld();
#pragma unroll
          for (int q = 0; q < 4; ++q) {  // piece q of row r sits at position q ^ ((r >> 1) & 3)
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = empty ? 0u
                           : pack_bf16x2(__uint_as_float(orr[8 * q + 2 * e]) * inv,
                                         __uint_as_float(orr[8 * q + 2 * e + 1]) * inv);
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
#pragma unroll
          for (int rr = 0; rr < 4; ++rr) {
            const int r = rr * 8 + (lane >> 2), q = lane & 3;
            const uint4 w = *reinterpret_cast<const uint4*>(stage + r * 64 + ((q ^ ((r >> 1) & 3)) << 4));
            const int64_t o = __shfl_sync(0xffffffffu, row_off, r);
            if (o >= 0) *reinterpret_cast<uint4*>(p.out + o + c * 32 + q * 8) = w;
          }
          __syncwarp();
        }
      }
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
  return LF_OK;
}

inline bool packed_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Largest power of two that divides the page, up to a block: a copy of that many keys stays in one page.
inline int packed_box(int page_size) {
  int box = 1;
  while (box < kPackedKeys && page_size % (box * 2) == 0) box *= 2;
  return box;
}

inline int packed_page_shift(int page_size) {
  for (int sh = 0; sh < 31; ++sh)
    if ((1 << sh) == page_size) return sh;
  return -1;
}

// Map of a pool [n_pages, page_size, Hkv, D] with strides (page, slot, kv head) for boxes of `box` slots.
inline int packed_pool_map(CUtensorMap* map, const void* pool, const int64_t* st, int n_pages, int page_size,
                           int Hkv, int D, int box) {
  return make_map_4d(map, TileMapSpec{pool, {D, page_size, Hkv, n_pages}, {st[1], st[2], st[0]}, {box, 1, 1}});
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

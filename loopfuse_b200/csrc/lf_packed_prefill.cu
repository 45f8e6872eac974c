// Packed prefill: causal attention of a batch of prompts of different lengths, their tokens one after
// the other in one tensor, with keys packed the same way or read from the paged cache. The tiles are
// those of lf_packed.cuh; this file has the order they are launched in and the host code.
#include "lf_packed.cuh"

#include <algorithm>
#include <type_traits>

namespace lf {

template <int D, int KIND, bool SOFTCAP>
__global__ void __launch_bounds__(kPackedThreads, 2)
    packed_prefill_kernel(const __grid_constant__ CUtensorMap tmap_q,
                          const __grid_constant__ CUtensorMap tmap_k,
                          const __grid_constant__ CUtensorMap tmap_v, const PackedParams p) {
  pdl_trigger();
  packed_tiles<D, KIND, SOFTCAP>(tmap_q, tmap_k, tmap_v, p, blockIdx.x);
}

// The list of items of a batch: its tiles, longest first, whosever they are (counting sort by key blocks;
// with the requests one after the other the last one's longest tile would start when the rest is nearly
// done), and those that are long next to what a CTA has to do in all cut into slices of their keys (a
// few new tokens behind a long context are a few tiles). One CTA; among items of one length the order is
// arbitrary, and no result depends on it. 7 us, 9 where slices are compared, which the tiles wait for: 32 chunks of up
// to 512 tokens behind up to 4096 take 90 us with it.
constexpr int kOrderThreads = 1024;
constexpr int kOrderLevels = 1024;
constexpr int kOrderRequests = 8192;  // in shared memory; larger batches keep the requests' order, are not cut, and
                                      // each CTA looks its tile up in the offsets, 32 requests at a time
constexpr int kWholeBlocks = 32;      // tiles of up to 2048 keys are never cut: a prompt of that length has
                                      // the same result in every batch
constexpr int kSliceBlocks = 16;      // at least, since a slice costs the store and the join of its rows
constexpr int kItemBlocks = 8;        // about what the start, the store and the join of a slice take, in blocks
constexpr int kOrderChoices = 8;      // lengths of slices that are compared

template <int KIND>
__global__ void __launch_bounds__(kOrderThreads)
    packed_order_kernel(const PackedParams p, PackedItem* items, const int max_items, const int max_parts,
                        const int n_slots) {
  extern __shared__ int32_t s_first[];  // [B + 1] first tile of each request
  __shared__ int32_t s_level[kOrderLevels];
  __shared__ long long s_warp[kOrderThreads / 32];
  __shared__ unsigned long long s_blocks;
  __shared__ int32_t s_longest, s_parts, s_cut;
  __shared__ int32_t s_slice[kOrderChoices], s_long[kOrderChoices], s_long_blocks[kOrderChoices];
  __shared__ long long s_cost[kOrderChoices];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  s_level[tid] = 0;
  if (tid == 0) {
    s_longest = s_parts = s_cut = 0;
    s_blocks = 0;
  }
  __syncthreads();
  pdl_wait();
  // Exclusive sums over the threads of the CTA; `all` gets the total. (In 64 bits: offsets out of order can let
  // every request hold the whole batch.)
  auto scan = [&](int v, long long* all) {
    long long incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += x;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    long long warps = s_warp[lane];  // (as many warps as lanes)
    const long long own = __shfl_sync(0xffffffffu, warps, warp);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, warps, d);
      if (lane >= d) warps += x;
    }
    __syncthreads();
    *all = __shfl_sync(0xffffffffu, warps, 31);
    return __shfl_sync(0xffffffffu, warps, warp) - own + incl - v;
  };
  // (Tiles past n_tiles, which requests in order do not have, are left out.)
  long long base = 0;
  for (int b0 = 0; b0 < p.B; b0 += kOrderThreads) {
    const int b = b0 + tid;
    int tiles = 0;
    if (b < p.B) {
      const PackedRequest r = packed_request<KIND>(p, b);
      tiles = (r.n + p.tq - 1) / p.tq;
    }
    long long all;
    const long long first = scan(tiles, &all);
    if (b < p.B) s_first[b] = static_cast<int32_t>(min(base + first, static_cast<long long>(p.n_tiles)));
    base += all;
  }
  __syncthreads();
  const int n = static_cast<int>(min(base, static_cast<long long>(p.n_tiles)));
  auto item_of = [&](int e) {
    int lo = 0, hi = p.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_first[mid] <= e) lo = mid;
      else hi = mid - 1;
    }
    return packed_item(p, packed_request<KIND>(p, lo), e - s_first[lo]);
  };
  // (A thread's first tile is looked up once; most batches have no second.)
  PackedItem mine_first = {};
  if (tid < n) mine_first = item_of(tid);
  auto item_at = [&](int e) { return e == tid ? mine_first : item_of(e); };
  // How much there is, and so how long a slice may be.
  {
    int longest = 0;
    unsigned long long blocks = 0;
    for (int e = tid; e < n; e += kOrderThreads) {
      const PackedItem it = item_at(e);
      longest = max(longest, it.hi - it.lo);
      blocks += it.hi - it.lo;
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
      longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, d));
      blocks += __shfl_xor_sync(0xffffffffu, blocks, d);
    }
    if (lane == 0) {
      atomicMax(&s_longest, longest);
      atomicAdd(&s_blocks, blocks);
    }
  }
  __syncthreads();
  // Slices of 0.8 to 1.5 of a CTA's share: as long as makes the whole shortest, if that is either what there
  // is over all CTAs or the rounds that the long items take on them, whichever is more. (Shorter ones are more
  // items than they bring balance. With 0.8 always, the 128 tiles of 512 tokens behind 4096 are 384 items for 296
  // CTAs: 99 us, and 68 now.)
  if (tid < kOrderChoices) {
    const long long share = (static_cast<long long>(s_blocks) * p.Hkv * (8 + tid) + 10ll * n_slots - 1) / (10ll * n_slots);
    s_slice[tid] = static_cast<int>(min(max(share, static_cast<long long>(kSliceBlocks)), 1ll << 28));
    s_long[tid] = s_long_blocks[tid] = 0;
  }
  __syncthreads();
  auto whole_of = [&](int slice) { return max(kWholeBlocks, slice + slice / 4); };
  int choice = 0;
  if (s_longest > whole_of(s_slice[0])) {
    int items_of[kOrderChoices] = {}, blocks_of[kOrderChoices] = {};  // long items, and the longest's blocks
    for (int e = tid; e < n; e += kOrderThreads) {
      const PackedItem it = item_at(e);
      const int blocks = it.hi - it.lo;
      if (blocks <= kWholeBlocks) continue;
#pragma unroll
      for (int c = 0; c < kOrderChoices; ++c) {
        const int slice = s_slice[c], parts = blocks > whole_of(slice) ? (blocks + slice - 1) / slice : 1;
        items_of[c] += parts;
        blocks_of[c] = max(blocks_of[c], (blocks + parts - 1) / parts);
      }
    }
#pragma unroll
    for (int c = 0; c < kOrderChoices; ++c) {
      const int items = __reduce_add_sync(0xffffffffu, items_of[c]);
      const int blocks = __reduce_max_sync(0xffffffffu, blocks_of[c]);
      if (lane == 0 && items) {
        atomicAdd(&s_long[c], items);
        atomicMax(&s_long_blocks[c], blocks);
      }
    }
    __syncthreads();
    if (tid < kOrderChoices) {
      const long long items = static_cast<long long>(s_long[tid]) * p.Hkv;
      const long long rounds = (items + n_slots - 1) / n_slots;
      const long long spread = static_cast<long long>(s_blocks) * p.Hkv + items * kItemBlocks;
      s_cost[tid] = max(spread, rounds * (s_long_blocks[tid] + kItemBlocks) * n_slots);
    }
    __syncthreads();
#pragma unroll
    for (int c = 1; c < kOrderChoices; ++c)
      if (s_cost[c] < s_cost[choice]) choice = c;
  }
  const int slice = s_slice[choice], whole = whole_of(slice);
  auto parts_of = [&](int blocks) { return blocks > whole ? (blocks + slice - 1) / slice : 1; };
  int shift = 0;
  while ((s_longest >> shift) >= kOrderLevels) ++shift;
  auto level_of = [&](int blocks) {  // longest first
    return kOrderLevels - 1 - min(blocks >> shift, kOrderLevels - 1);
  };
  for (int e = tid; e < n; e += kOrderThreads) {
    const PackedItem it = item_at(e);
    const int blocks = it.hi - it.lo, parts = parts_of(blocks);
    atomicAdd(&s_level[level_of((blocks + parts - 1) / parts)], parts);
  }
  __syncthreads();
  long long n_items;
  const int mine = static_cast<int>(scan(s_level[tid], &n_items));
  s_level[tid] = mine;
  __syncthreads();
  for (int e = tid; e < n; e += kOrderThreads) {
    PackedItem it = item_at(e);
    const int lo = it.lo, blocks = it.hi - it.lo, parts = parts_of(blocks);
    const int at = atomicAdd(&s_level[level_of((blocks + parts - 1) / parts)], parts);
    if (parts > 1) {
      it.part = atomicAdd(&s_parts, parts);
      it.counter = atomicAdd(&s_cut, 1);
      it.n_parts = parts;
    }
    // (The host's room follows from the lengths of slices; see lf_packed_workspace_bytes.)
    if (at + parts > max_items || (parts > 1 && it.part + parts > max_parts)) continue;
    for (int s = 0; s < parts; ++s) {
      it.index = s;
      it.lo = lo + static_cast<int>(static_cast<long long>(blocks) * s / parts);
      it.hi = lo + static_cast<int>(static_cast<long long>(blocks) * (s + 1) / parts);
      items[at + s] = it;
    }
    if (parts > 1)
      for (int h = 0; h < p.Hkv; ++h) p.list[2 + it.counter * p.Hkv + h] = 0;
  }
  if (tid == 0) {
    p.list[0] = static_cast<uint32_t>(min(n_items, static_cast<long long>(max_items)));
    p.list[1] = 0;
  }
}

static int sm_count() {
  static thread_local int cached_dev = -1, cached = 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev != cached_dev) {
    cudaDeviceGetAttribute(&cached, cudaDevAttrMultiProcessorCount, dev);
    cached_dev = dev;
  }
  return cached > 0 ? cached : 148;
}

// Tiles of a kv head that a batch has at most: whatever the lengths, each request has one partly filled.
static int64_t most_tiles(int32_t B, int32_t T, int32_t tq) { return T / tq + std::min(B, T); }

// Whether a batch gets a list, and the room that it needs: batches of more tiles than two per SM, and
// those whose tiles can be long. `max_keys`: keys that a request has at most. The others start all at
// once, and a launch ahead of them would cost more than an order brings.
struct PackedList {
  bool used = false;
  int64_t max_items = 0, max_parts = 0;  // (of a kv head)
  size_t head_bytes = 0, item_bytes = 0, part_bytes = 0;
  size_t bytes() const { return used ? head_bytes + item_bytes + part_bytes : 0; }
};
static PackedList plan_list(int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t D, int64_t max_keys) {
  PackedList l;
  const int64_t sms = sm_count(), tiles = most_tiles(B, T, kPackedRows / (Hq / Hkv));
  const bool cuts = max_keys > static_cast<int64_t>(kWholeBlocks) * kPackedKeys;
  l.used = B <= kOrderRequests && (cuts || (tiles * Hkv > 2 * sms && B > 1));
  if (!l.used) return l;
  // Slices: a tile of n blocks has ceil(n / slice) with slice >= 0.8 of a CTA's share W / (2 sms) and n >
  // 1.25 slice, so all heads' together are at most W / slice + W / (1.25 slice) = 4.5 sms.
  l.max_parts = cuts ? (9 * sms / 2 + Hkv) / Hkv + 1 : 0;
  l.max_items = tiles + l.max_parts;
  l.head_bytes = ((2 + static_cast<size_t>(l.max_parts) / 2 * Hkv) * 4 + 127) / 128 * 128;
  l.item_bytes = (static_cast<size_t>(l.max_items) * sizeof(PackedItem) + 127) / 128 * 128;
  l.part_bytes = static_cast<size_t>(l.max_parts) * Hkv * kPackedRows * (D + 2) * 4;
  return l;
}

// Keys that a request has at most, and that all have together.
static int64_t most_keys(const LfPackedArgs* a, int64_t* together) {
  if (!a->block_table) {
    *together = a->Tk;
    return a->Tk;
  }
  const int64_t held = static_cast<int64_t>(a->bt_blocks) * a->page_size;
  *together = std::min(held * a->B, static_cast<int64_t>(a->n_pages) * a->page_size);
  return held;
}

template <int D, int KIND, bool SOFTCAP>
static int launch_packed(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                         const PackedParams& p, unsigned grid, cudaStream_t st) {
  using Shape = PackedShape<D>;
  static thread_local int configured_dev = -1;
  const auto kernel = packed_prefill_kernel<D, KIND, SOFTCAP>;
  const int rc = packed_configure(kernel, Shape::kSmem, &configured_dev);
  if (rc != LF_OK) return rc;
  launch_pdl(kernel, dim3(grid), kPackedThreads, Shape::kSmem, st, mq, mk, mv, p);
  return check_launch("packed_prefill_kernel");
}

template <int KIND>
static int launch_order(const PackedParams& p, PackedItem* items, const PackedList& l, cudaStream_t st) {
  const size_t smem = (static_cast<size_t>(p.B) + 1) * sizeof(int32_t);
  launch_pdl(packed_order_kernel<KIND>, dim3(1), kOrderThreads, smem, st, p, items,
             static_cast<int>(l.max_items), static_cast<int>(l.max_parts), 2 * sm_count());
  return check_launch("packed_order_kernel");
}

}  // namespace lf

extern "C" {

size_t lf_packed_workspace_bytes(const LfPackedArgs* a) {
  using namespace lf;
  if (!a || a->B <= 0 || a->T <= 0 || a->Hkv <= 0 || a->Hq <= 0 || a->Hq % a->Hkv ||
      a->Hq / a->Hkv > kPackedRows)
    return 0;
  int64_t together;
  return plan_list(a->B, a->T, a->Hq, a->Hkv, a->D, most_keys(a, &together)).bytes();
}

int lf_packed_prefill_bf16(const LfPackedArgs* a, void* stream) {
  using namespace lf;
  if (!a || a->B <= 0 || a->T < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv) return LF_ERR_INVALID_ARG;
  if (a->D != 64 && a->D != 128) return LF_ERR_UNSUPPORTED;
  const bool paged = a->block_table != nullptr;
  if (a->mask_kind < LF_MASK_NONE || a->mask_kind > LF_MASK_CAUSAL_WINDOW) return LF_ERR_INVALID_ARG;
  if (a->mask_kind == LF_MASK_CAUSAL_WINDOW && a->window <= 0) return LF_ERR_INVALID_ARG;
  if (paged ? (a->page_size <= 0 || a->n_pages <= 0 || a->bt_blocks <= 0) : a->Tk < 0)
    return LF_ERR_INVALID_ARG;
  if (a->T > kMostKeys || (!paged && a->Tk > kMostKeys)) return LF_ERR_TOO_LARGE;
  const int G = a->Hq / a->Hkv;
  if (G > kPackedRows) return LF_ERR_UNSUPPORTED;
  PackedScore score;
  int rc = packed_score(a->scale, a->n_mod, a->mod_op, a->mod_arg, &score);
  if (rc != LF_OK) return rc;
  if (a->T == 0) return LF_OK;
  if (!a->q || !a->out || !a->cu_q || (paged ? !a->kv_lens : !a->cu_k)) return LF_ERR_INVALID_ARG;
  // (No key at all: maps of one row of q that nothing is read through.)
  const bool no_keys = !paged && a->Tk == 0;
  const void* kv[2] = {no_keys ? a->q : a->k, no_keys ? a->q : a->v};
  if (!kv[0] || !kv[1]) return LF_ERR_INVALID_ARG;
  if (!packed_aligned(a->q) || !packed_aligned(kv[0]) || !packed_aligned(kv[1]) || !packed_aligned(a->out))
    return LF_ERR_ALIGNMENT;
  if (a->o_stride[0] % 8 || a->o_stride[1] % 8) return LF_ERR_ALIGNMENT;

  PackedParams p = {};
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.o_stride[0] = a->o_stride[0];
  p.o_stride[1] = a->o_stride[1];
  p.out_sectors = reinterpret_cast<uintptr_t>(a->out) % 32 == 0 && a->o_stride[0] % 16 == 0 && a->o_stride[1] % 16 == 0;
  p.cu_q = a->cu_q;
  p.cu_k = a->cu_k;
  p.kv_lens = a->kv_lens;
  p.table = a->block_table;
  p.bt_stride = a->bt_stride;
  p.B = a->B;
  p.T = a->T;
  p.Tk = a->Tk;
  p.Hkv = a->Hkv;
  p.G = G;
  p.tq = kPackedRows / G;
  p.mask_kind = a->mask_kind;
  // (No request has more keys, and the first key of a query, `pos - (window - 1)` with pos from -2^30 up, stays
  // within 32 bits.)
  p.window = std::min(a->window, kMostKeys);
  p.a = score.a;
  p.c2 = score.c2;
  p.m_first = score.m_first;
  p.bt_blocks = a->bt_blocks;
  p.page_size = paged ? a->page_size : 1;
  p.page_shift = packed_page_shift(p.page_size);
  p.n_pages = a->n_pages;
  p.status = a->status;

  CUtensorMap mq, mk, mv;
  rc = make_map_5d(&mq, TileMapSpec{a->q, {a->D, G, a->Hkv, a->T, 1},
                                    {a->q_stride[1], a->q_stride[1] * G, a->q_stride[0], 0}, {G, 1, p.tq, 1}});
  if (rc == LF_OK && paged)
    rc = packed_pool_maps(&mk, &mv, kv[0], kv[1], a->k_stride, a->v_stride, a->n_pages, a->page_size, a->Hkv,
                          a->D, &p);
  for (int i = 0; i < 2 && rc == LF_OK && !paged; ++i) {
    const int64_t* st = i ? a->v_stride : a->k_stride;
    // (By column, token, half, kv head.)
    rc = make_map_5d(i ? &mv : &mk, TileMapSpec{kv[i], {64, std::max(a->Tk, 1), a->D / 64, a->Hkv, 1},
                                                {st[0], 64, st[1], 0}, {kPackedKeys, a->D / 64, 1, 1}});
  }
  if (rc != LF_OK) return rc;

  const int64_t tiles = most_tiles(a->B, a->T, p.tq);
  int64_t keys;
  const int64_t max_keys = most_keys(a, &keys);
  const PackedList list = plan_list(a->B, a->T, a->Hq, a->Hkv, a->D, max_keys);
  // The heads of a chunk run together: as many as keep their K and V in half of L2, since the tiles that
  // read them do so at different times.
  const int64_t fit = std::max<int64_t>(1, (64ll << 20) / std::max<int64_t>(1, keys * a->D * 4));
  const int64_t chunks = (a->Hkv + fit - 1) / fit;
  const int64_t per_chunk = (a->Hkv + chunks - 1) / chunks;
  if ((tiles + list.max_parts) * per_chunk * chunks > 0x7fffffff - 4096) return LF_ERR_TOO_LARGE;
  p.n_tiles = static_cast<int32_t>(tiles);
  p.div_chunk = FastDiv::make(static_cast<int32_t>(per_chunk));
  p.div_tiles = FastDiv::make(p.n_tiles);
  p.div_g = FastDiv::make(G);
  int64_t grid = tiles * per_chunk * chunks;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (list.used) {
    if (!a->workspace || a->workspace_bytes < list.bytes()) return LF_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(a->workspace) & 31u) return LF_ERR_ALIGNMENT;  // (32-byte stores)
    char* ws = static_cast<char*>(a->workspace);
    PackedItem* items = reinterpret_cast<PackedItem*>(ws + list.head_bytes);
    p.list = reinterpret_cast<uint32_t*>(ws);
    p.part_o = reinterpret_cast<float*>(ws + list.head_bytes + list.item_bytes);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + list.max_parts * a->Hkv * kPackedRows * a->D);
    rc = paged ? launch_order<kPackedPaged>(p, items, list, st)
               : launch_order<kPackedDense>(p, items, list, st);
    if (rc != LF_OK) return rc;
    p.items = items;
    grid = std::min<int64_t>(grid + list.max_parts * per_chunk * chunks, 2ll * sm_count());
  }
  auto with_d = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (paged)
      return score.softcap ? launch_packed<D, kPackedPaged, true>(mq, mk, mv, p, static_cast<unsigned>(grid), st)
                           : launch_packed<D, kPackedPaged, false>(mq, mk, mv, p, static_cast<unsigned>(grid), st);
    return score.softcap ? launch_packed<D, kPackedDense, true>(mq, mk, mv, p, static_cast<unsigned>(grid), st)
                         : launch_packed<D, kPackedDense, false>(mq, mk, mv, p, static_cast<unsigned>(grid), st);
  };
  return a->D == 128 ? with_d(std::integral_constant<int, 128>{}) : with_d(std::integral_constant<int, 64>{});
}

}  // extern "C"

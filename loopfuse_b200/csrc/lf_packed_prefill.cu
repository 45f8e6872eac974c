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
  extern __shared__ unsigned char smem[];
  pdl_trigger();
  pdl_wait();
  packed_tile<D, KIND, SOFTCAP>(tmap_q, tmap_k, tmap_v, p, smem, blockIdx.x);
}

// Order of the tiles of a batch that does not fit the machine at once: longest first, whosever they are
// (counting sort by key blocks). With the requests one after the other the last one's longest tile would
// start when the rest is nearly done. One CTA; among tiles of one length the order is arbitrary, and no
// result depends on it.
constexpr int kOrderThreads = 1024;
constexpr int kOrderLevels = 1024;
constexpr int kOrderRequests = 8192;  // in shared memory; larger batches keep the requests' order

template <int KIND>
__global__ void __launch_bounds__(kOrderThreads)
    packed_order_kernel(const PackedParams p, int2* items, int32_t* n_items) {
  extern __shared__ int32_t s_first[];  // [B + 1] first tile of each request
  __shared__ int32_t s_level[kOrderLevels];
  __shared__ int32_t s_warp[kOrderThreads / 32];
  __shared__ int32_t s_longest;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  s_level[tid] = 0;
  if (tid == 0) s_longest = 0;
  __syncthreads();
  pdl_wait();
  // Exclusive sums over the threads of the CTA; `all` gets the total.
  auto scan = [&](int v, int* all) {
    int incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += x;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < kOrderThreads / 32; ++w) {
      const int x = s_warp[w];
      if (w < warp) before += x;
      total += x;
    }
    __syncthreads();
    *all = total;
    return before + incl - v;
  };
  int base = 0, longest = 0;
  for (int b0 = 0; b0 < p.B; b0 += kOrderThreads) {
    const int b = b0 + tid;
    int tiles = 0;
    if (b < p.B) {
      const PackedRequest r = packed_request<KIND>(p, b);
      tiles = (r.n + p.tq - 1) / p.tq;
      longest = max(longest, r.m);
    }
    int all;
    const int first = scan(tiles, &all);
    if (b < p.B) s_first[b] = base + first;
    base += all;
  }
  const int n = min(base, p.n_tiles);
  atomicMax(&s_longest, longest);
  __syncthreads();
  int shift = 0;
  while ((((s_longest + kPackedKeys - 1) / kPackedKeys) >> shift) >= kOrderLevels) ++shift;

  auto tile_of = [&](int e) {
    int lo = 0, hi = p.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_first[mid] <= e) lo = mid;
      else hi = mid - 1;
    }
    return make_int2(lo, e - s_first[lo]);
  };
  auto level_of = [&](int2 at) {  // longest first: level 0
    const PackedRequest r = packed_request<KIND>(p, at.x);
    const int t0 = at.y * p.tq, off = r.m - r.n;
    int last = r.m, first = 0;
    if (p.mask_kind != LF_MASK_NONE) last = min(last, min(t0 + p.tq, r.n) + off);
    if (p.mask_kind == LF_MASK_CAUSAL_WINDOW) first = max(0, t0 + off - (p.window - 1));
    const int blocks = last > first ? (last + kPackedKeys - 1) / kPackedKeys - first / kPackedKeys : 0;
    return kOrderLevels - 1 - min(blocks >> shift, kOrderLevels - 1);
  };
  for (int e = tid; e < n; e += kOrderThreads) atomicAdd(&s_level[level_of(tile_of(e))], 1);
  __syncthreads();
  int all;
  const int mine = scan(s_level[tid], &all);
  s_level[tid] = mine;
  __syncthreads();
  for (int e = tid; e < n; e += kOrderThreads) {
    const int2 at = tile_of(e);
    items[atomicAdd(&s_level[level_of(at)], 1)] = at;
  }
  if (tid == 0) *n_items = n;
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

// Batches of more tiles than two per SM are ordered; the others start all at once.
static bool is_ordered(int64_t tiles, int32_t Hkv, int32_t B) {
  return tiles * Hkv > 2ll * sm_count() && B <= kOrderRequests && B > 1;
}

constexpr size_t kOrderHeader = 16;

template <int D, int KIND, bool SOFTCAP>
static int launch_packed(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                         const PackedParams& p, unsigned grid, cudaStream_t st) {
  using Shape = PackedShape<D>;
  static_assert(2 * (Shape::kSmem + 1024) <= 233472 && 3 * (Shape::kSmem + 1024) > 233472,
                "two CTAs per SM, for its 512 columns of tensor memory");
  static thread_local int configured_dev = -1;
  const auto kernel = packed_prefill_kernel<D, KIND, SOFTCAP>;
  const int rc = packed_configure(kernel, Shape::kSmem, &configured_dev);
  if (rc != LF_OK) return rc;
  launch_pdl(kernel, dim3(grid), kPackedThreads, Shape::kSmem, st, mq, mk, mv, p);
  return check_launch("packed_prefill_kernel");
}

template <int KIND>
static int launch_order(const PackedParams& p, int2* items, int32_t* n_items, cudaStream_t st) {
  const size_t smem = (static_cast<size_t>(p.B) + 1) * sizeof(int32_t);
  launch_pdl(packed_order_kernel<KIND>, dim3(1), kOrderThreads, smem, st, p, items, n_items);
  return check_launch("packed_order_kernel");
}

}  // namespace lf

extern "C" {

size_t lf_packed_workspace_bytes(int32_t B, int32_t T, int32_t Hq, int32_t Hkv) {
  using namespace lf;
  if (B <= 0 || T <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > kPackedRows) return 0;
  const int64_t tiles = most_tiles(B, T, kPackedRows / (Hq / Hkv));
  return is_ordered(tiles, Hkv, B) ? kOrderHeader + static_cast<size_t>(tiles) * sizeof(int2) : 0;
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
  p.window = a->window;
  p.a = score.a;
  p.c2 = score.c2;
  p.bt_blocks = a->bt_blocks;
  p.page_size = paged ? a->page_size : 1;
  p.page_shift = packed_page_shift(p.page_size);
  p.n_pages = a->n_pages;
  p.box = packed_box(p.page_size);
  p.status = a->status;

  CUtensorMap mq, mk, mv;
  rc = make_map_4d(&mq, TileMapSpec{a->q, {a->D, G, a->Hkv, a->T},
                                    {a->q_stride[1], a->q_stride[1] * G, a->q_stride[0]}, {G, 1, p.tq}});
  for (int i = 0; i < 2 && rc == LF_OK; ++i) {
    CUtensorMap* map = i ? &mv : &mk;
    const int64_t* st = i ? a->v_stride : a->k_stride;
    rc = paged ? packed_pool_map(map, kv[i], st, a->n_pages, a->page_size, a->Hkv, a->D, p.box)
               : make_map_4d(map, TileMapSpec{kv[i], {a->D, std::max(a->Tk, 1), a->Hkv, 1},
                                              {st[0], st[1], 0}, {kPackedKeys, 1, 1}});
  }
  if (rc != LF_OK) return rc;

  const int64_t tiles = most_tiles(a->B, a->T, p.tq);
  const bool ordered = is_ordered(tiles, a->Hkv, a->B);
  // The heads of a chunk run together: as many as keep their K and V in half of L2, since the tiles that
  // read them do so at different times.
  const int64_t keys = paged ? std::min<int64_t>(static_cast<int64_t>(a->n_pages) * a->page_size,
                                                 static_cast<int64_t>(a->B) * a->bt_blocks * a->page_size)
                             : a->Tk;
  const int64_t fit = (64ll << 20) / std::max<int64_t>(1, keys * a->D * 4);
  const int64_t chunks = (a->Hkv + std::max<int64_t>(fit, 1) - 1) / std::max<int64_t>(fit, 1);
  const int64_t per_chunk = (a->Hkv + chunks - 1) / chunks;
  if (tiles * per_chunk * chunks > 0x7fffffff) return LF_ERR_TOO_LARGE;
  p.n_tiles = static_cast<int32_t>(tiles);
  p.div_chunk = FastDiv::make(static_cast<int32_t>(per_chunk));
  p.div_tiles = FastDiv::make(p.n_tiles);
  p.div_g = FastDiv::make(G);
  const unsigned grid = static_cast<unsigned>(tiles * per_chunk * chunks);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (ordered) {
    if (!a->workspace || a->workspace_bytes < lf_packed_workspace_bytes(a->B, a->T, a->Hq, a->Hkv))
      return LF_ERR_WORKSPACE;
    if (!packed_aligned(a->workspace)) return LF_ERR_ALIGNMENT;
    int32_t* n_items = static_cast<int32_t*>(a->workspace);
    int2* items = reinterpret_cast<int2*>(static_cast<char*>(a->workspace) + kOrderHeader);
    rc = paged ? launch_order<kPackedPaged>(p, items, n_items, st)
               : launch_order<kPackedDense>(p, items, n_items, st);
    if (rc != LF_OK) return rc;
    p.items = items;
    p.n_items = n_items;
  }
  auto with_d = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (paged)
      return score.softcap ? launch_packed<D, kPackedPaged, true>(mq, mk, mv, p, grid, st)
                           : launch_packed<D, kPackedPaged, false>(mq, mk, mv, p, grid, st);
    return score.softcap ? launch_packed<D, kPackedDense, true>(mq, mk, mv, p, grid, st)
                         : launch_packed<D, kPackedDense, false>(mq, mk, mv, p, grid, st);
  };
  return a->D == 128 ? with_d(std::integral_constant<int, 128>{}) : with_d(std::integral_constant<int, 64>{});
}

}  // extern "C"

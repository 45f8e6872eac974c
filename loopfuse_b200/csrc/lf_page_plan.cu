// The start of a serving step over a paged cache: which pages the new tokens of a batch of requests of
// different lengths take, where each of them goes (plan_pages_kernel), and the store of their K/V rows
// to those places (kv_append_packed_kernel).
//
//   before_b = ceil(kv_b / P), after_b = ceil((kv_b + new_b) / P)        pages of request b
//   first_b  = sum of (after - before) over the requests ahead of b     its first page in the free list
//   table[b, c] = free[first_b + c - before_b]                          before_b <= c < after_b
//   token t of the packed batch, cu_b <= t < cu_{b+1}:  pos = kv_b + t - cu_b,
//   slot = table[b, pos / P] * P + pos % P
#include "lf_common.cuh"

namespace lf {

struct PlanParams {
  const int32_t* kv_lens;
  const int32_t* new_lens;
  const int32_t* free_pages;
  int32_t* table;
  int32_t* cu;
  int32_t* seq_lens;
  int32_t* slots;
  int32_t* positions;
  int32_t* pages_used;
  int32_t* status;
  int64_t bt_stride;
  int32_t B, n_free, bt_blocks, page_size, page_shift, num_tokens;
};

constexpr int kPlanThreads = 512;
constexpr int kMaxLength = 1 << 30;  // of a request, so that no sum of two lengths passes 32 bits

// Every CTA adds up all the lengths by itself (a few KB from L2) and then places its share of the new
// pages and tokens: no launch and no wait between the two halves. Old entries of the table are read and
// new ones written, never the same ones, so the CTAs do not depend on each other. Bound by latency, of the launch,
// the sums and a search per token: 512 requests of up to 2048 new tokens 5.4 us in a graph, 64 requests of one token
// 4.1. A call from Python is bound by the host, 6.5 to 7 us for its checks, the output tensors and the launch.
__global__ void __launch_bounds__(kPlanThreads) plan_pages_kernel(const PlanParams p) {
  extern __shared__ int32_t s_plan[];
  int32_t* s_cu = s_plan;               // [B + 1] first token of each request
  int32_t* s_page = s_plan + p.B + 1;   // [B + 1] first new page
  __shared__ long long s_warp[2][kPlanThreads / 32];
  __shared__ int s_bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_bad = 0;
  __syncthreads();
  pdl_trigger();
  pdl_wait();
  auto pages_of = [&](int n) {
    const uint32_t up = static_cast<uint32_t>(n) + static_cast<uint32_t>(p.page_size) - 1u;
    return static_cast<int>(p.page_shift >= 0 ? up >> p.page_shift
                                              : up / static_cast<uint32_t>(p.page_size));
  };
  auto clamp_len = [&](int n, int most) {
    if (n < 0 || n > most) s_bad = 1;
    return min(max(n, 0), most);
  };
  // Sums in 64 bits: lengths that make no sense add up to more than any buffer holds. Tokens past num_tokens are
  // dropped; where there are some, a second pass takes pages for the tokens that are left.
  long long tokens_before, pages_before, pages_asked = 0;
  for (bool cut = false;; cut = true) {
    tokens_before = pages_before = 0;
    for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
      const int b = b0 + tid;
      int held = 0, fresh = 0;
      if (b < p.B) {
        held = clamp_len(p.kv_lens[b], kMaxLength);
        fresh = cut ? s_cu[b + 1] - s_cu[b] : clamp_len(p.new_lens[b], kMaxLength - 1);
      }
      long long tok = fresh, pg = pages_of(held + fresh) - pages_of(held);
      const long long my_tok = tok, my_pg = pg;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, tok, d);
        const long long c = __shfl_up_sync(0xffffffffu, pg, d);
        if (lane >= d) {
          tok += a;
          pg += c;
        }
      }
      if (lane == 31) {
        s_warp[0][warp] = tok;
        s_warp[1][warp] = pg;
      }
      __syncthreads();
      long long wt = 0, wp = 0, all_t = 0, all_p = 0;
#pragma unroll
      for (int w = 0; w < kPlanThreads / 32; ++w) {
        if (w < warp) {
          wt += s_warp[0][w];
          wp += s_warp[1][w];
        }
        all_t += s_warp[0][w];
        all_p += s_warp[1][w];
      }
      if (b < p.B) {
        const long long t0 = tokens_before + wt + tok - my_tok;
        s_cu[b] = static_cast<int32_t>(min(t0, static_cast<long long>(p.num_tokens)));
        s_page[b] = static_cast<int32_t>(min(pages_before + wp + pg - my_pg, 0x7fffffffll));
      }
      tokens_before += all_t;
      pages_before += all_p;
      __syncthreads();
    }
    if (tid == 0) {
      s_cu[p.B] = static_cast<int32_t>(min(tokens_before, static_cast<long long>(p.num_tokens)));
      s_page[p.B] = static_cast<int32_t>(min(pages_before, 0x7fffffffll));
    }
    __syncthreads();
    if (!cut) pages_asked = pages_before;
    if (cut || tokens_before <= p.num_tokens) break;
    if (tid == 0) s_bad = 1;
  }
  const int n_tokens = s_cu[p.B], n_pages = s_page[p.B];
  if (tid == 0 && blockIdx.x == 0) {
    // (Where pages run out: what the lengths ask for, dropped tokens included.)
    *p.pages_used = n_pages > p.n_free ? static_cast<int32_t>(min(pages_asked, 0x7fffffffll)) : n_pages;
    if (p.status && s_bad) atomicCAS(p.status, 0, LF_DEV_BAD_LENGTHS);
    if (p.status && n_pages > p.n_free) atomicCAS(p.status, 0, LF_DEV_BAD_PAGE);
  }

  // Request that entry i of a list belongs to, by the requests' first entries (the last of those that
  // start at or before i: the ones ahead of it with the same start are empty).
  auto owner = [&](const int32_t* first, int i) {
    int lo = 0, hi = p.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  const int step = gridDim.x * kPlanThreads, start = blockIdx.x * kPlanThreads + tid;
  for (int b = start; b <= p.B; b += step) {
    p.cu[b] = s_cu[b];
    if (b < p.B)
      p.seq_lens[b] = min(max(p.kv_lens[b], 0), kMaxLength) + (s_cu[b + 1] - s_cu[b]);
  }
  for (int e = start; e < n_pages; e += step) {  // (no more than tokens: 2^30)
    const int b = owner(s_page, e);
    const int c = pages_of(min(max(p.kv_lens[b], 0), kMaxLength)) + (e - s_page[b]);
    if (c < p.bt_blocks) p.table[b * p.bt_stride + c] = e < p.n_free ? p.free_pages[e] : -1;
    else if (p.status) atomicCAS(p.status, 0, LF_DEV_BAD_PAGE);  // the table is too narrow
  }
  for (int t = start; t < p.num_tokens; t += step) {
    int slot = -1, pos = 0;
    if (t < n_tokens) {
      const int b = owner(s_cu, t);
      if (!LF_BOUNDS(t >= s_cu[b] && t < s_cu[b + 1], p.status, 74)) continue;
      const int held = min(max(p.kv_lens[b], 0), kMaxLength);
      pos = held + (t - s_cu[b]);
      const int blk = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
      const int old = pages_of(held);
      int page = -1;
      if (blk < p.bt_blocks) {
        const int e = s_page[b] + (blk - old);
        if (blk < old) page = p.table[b * p.bt_stride + blk];
        else if (e < p.n_free) page = p.free_pages[e];
      }
      if (page >= 0 && page <= (0x7fffffff - p.page_size + 1) / p.page_size)
        slot = page * p.page_size + (pos - blk * p.page_size);
      else if (p.status) atomicCAS(p.status, 0, LF_DEV_BAD_PAGE);
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
}

struct AppendPackedParams {
  const __nv_bfloat16* k_new;
  const __nv_bfloat16* v_new;
  __nv_bfloat16* k_pool;
  __nv_bfloat16* v_pool;
  const int32_t* slots;
  int64_t kn_stride[2], vn_stride[2];  // (token, kv head)
  int64_t kp_stride[3], vp_stride[3];  // (page, slot, kv head)
  int32_t n_slots, page_size, page_shift;
  uint32_t total;                      // 16-byte pieces of the new K rows
  FastDiv div_token, div_head;         // pieces per token, per row
  int32_t* status;
};

// One thread moves one 16-byte piece of a K row and the same piece of the V row. Consecutive threads
// take consecutive pieces, then heads, then tokens: whole lines on both sides, since a token's heads lie
// next to each other in a page. Pure data movement, bound by HBM for prompts and by latency for a token
// per request. 54 thousand tokens of 8 heads of 128: 70 us, 6.3 TB/s in both directions together.
__global__ void __launch_bounds__(256) kv_append_packed_kernel(const AppendPackedParams p) {
  pdl_trigger();
  pdl_wait();
  const uint32_t step = gridDim.x * 256u;
  for (uint32_t gid = blockIdx.x * 256u + threadIdx.x; gid < p.total; gid += step) {
    const uint32_t t = p.div_token.div(gid);
    const uint32_t piece = gid - t * p.div_token.d;
    const uint32_t h = p.div_head.div(piece);
    const uint32_t c = piece - h * p.div_head.d;
    const int slot = p.slots[t];
    if (slot < 0) continue;      // a padding row
    if (slot >= p.n_slots) {     // never write outside the pool
      if (p.status) atomicExch(p.status, LF_DEV_BAD_PAGE);
      continue;
    }
    if (!LF_BOUNDS(t < p.total / p.div_token.d && h * p.div_head.d < p.div_token.d, p.status, 73)) continue;
    const int page = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
    const int at = slot - page * p.page_size;
    const uint4 kx = ldg_stream_16(p.k_new + t * p.kn_stride[0] + h * p.kn_stride[1] + c * 8);
    const uint4 vx = ldg_stream_16(p.v_new + t * p.vn_stride[0] + h * p.vn_stride[1] + c * 8);
    *reinterpret_cast<uint4*>(p.k_pool + page * p.kp_stride[0] + at * p.kp_stride[1] +
                              h * p.kp_stride[2] + c * 8) = kx;
    *reinterpret_cast<uint4*>(p.v_pool + page * p.vp_stride[0] + at * p.vp_stride[1] +
                              h * p.vp_stride[2] + c * 8) = vx;
  }
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static int shift_of(int page_size) {
  for (int sh = 0; sh < 31; ++sh)
    if ((1 << sh) == page_size) return sh;
  return -1;
}

static int sm_count_or(int fallback) {
  int dev = 0, n = fallback;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

}  // namespace lf

extern "C" {

int lf_plan_pages(const LfPagePlanArgs* a, void* stream) {
  using namespace lf;
  if (!a || !a->kv_lens || !a->new_lens || !a->block_table || !a->cu_seqlens || !a->seq_lens ||
      !a->pages_used || (a->num_tokens > 0 && (!a->slots || !a->positions)) ||
      (a->n_free > 0 && !a->free_pages))
    return LF_ERR_INVALID_ARG;
  if (a->B <= 0 || a->n_free < 0 || a->bt_blocks <= 0 || a->page_size <= 0 || a->num_tokens < 0)
    return LF_ERR_INVALID_ARG;
  if (a->B > LF_MAX_REQUESTS || a->num_tokens > kMaxLength || a->page_size > kMaxLength)
    return LF_ERR_TOO_LARGE;
  PlanParams p;
  p.kv_lens = a->kv_lens;
  p.new_lens = a->new_lens;
  p.free_pages = a->free_pages;
  p.table = a->block_table;
  p.cu = a->cu_seqlens;
  p.seq_lens = a->seq_lens;
  p.slots = a->slots;
  p.positions = a->positions;
  p.pages_used = a->pages_used;
  p.status = a->status;
  p.bt_stride = a->bt_stride;
  p.B = a->B;
  p.n_free = a->n_free;
  p.bt_blocks = a->bt_blocks;
  p.page_size = a->page_size;
  p.page_shift = shift_of(a->page_size);
  p.num_tokens = a->num_tokens;
  const size_t smem = 2 * (static_cast<size_t>(a->B) + 1) * sizeof(int32_t);
  static thread_local int configured_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (smem > 48 * 1024 - 1024 && configured_dev != dev) {
    const cudaError_t e =
        cudaFuncSetAttribute(plan_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             2 * (LF_MAX_REQUESTS + 1) * static_cast<int>(sizeof(int32_t)));
    if (e != cudaSuccess) {
      set_cuda_error(e, "cudaFuncSetAttribute(plan_pages_kernel)");
      return LF_ERR_CUDA;
    }
    configured_dev = dev;
  }
  int64_t blocks = (static_cast<int64_t>(a->num_tokens) + kPlanThreads - 1) / kPlanThreads;
  const int64_t most = sm_count_or(148);
  blocks = blocks < 1 ? 1 : blocks > most ? most : blocks;
  launch_pdl(plan_pages_kernel, dim3(static_cast<unsigned>(blocks)), kPlanThreads, smem,
             static_cast<cudaStream_t>(stream), p);
  return check_launch("plan_pages_kernel");
}

int lf_kv_append_packed_bf16(const LfKvAppendPackedArgs* a, void* stream) {
  using namespace lf;
  if (!a || a->T < 0 || a->Hkv <= 0 || a->page_size <= 0 || a->n_pages <= 0) return LF_ERR_INVALID_ARG;
  if (a->D != 64 && a->D != 128) return LF_ERR_UNSUPPORTED;
  if (a->T == 0) return LF_OK;
  if (!a->k_new || !a->v_new || !a->k_pool || !a->v_pool || !a->slots) return LF_ERR_INVALID_ARG;
  if (!aligned16(a->k_new) || !aligned16(a->v_new) || !aligned16(a->k_pool) || !aligned16(a->v_pool))
    return LF_ERR_ALIGNMENT;
  for (int i = 0; i < 3; ++i)
    if ((i < 2 && (a->kn_stride[i] % 8 || a->vn_stride[i] % 8)) || a->kp_stride[i] % 8 ||
        a->vp_stride[i] % 8)
      return LF_ERR_ALIGNMENT;
  const int64_t total = static_cast<int64_t>(a->T) * a->Hkv * (a->D / 8);
  const int64_t n_slots = static_cast<int64_t>(a->n_pages) * a->page_size;
  if (total > 0x7fffffff - (1 << 24) || n_slots > 0x7fffffff) return LF_ERR_TOO_LARGE;
  AppendPackedParams p;
  p.k_new = static_cast<const __nv_bfloat16*>(a->k_new);
  p.v_new = static_cast<const __nv_bfloat16*>(a->v_new);
  p.k_pool = static_cast<__nv_bfloat16*>(a->k_pool);
  p.v_pool = static_cast<__nv_bfloat16*>(a->v_pool);
  p.slots = a->slots;
  for (int i = 0; i < 3; ++i) {
    if (i < 2) {
      p.kn_stride[i] = a->kn_stride[i];
      p.vn_stride[i] = a->vn_stride[i];
    }
    p.kp_stride[i] = a->kp_stride[i];
    p.vp_stride[i] = a->vp_stride[i];
  }
  p.n_slots = static_cast<int32_t>(n_slots);
  p.page_size = a->page_size;
  p.page_shift = shift_of(a->page_size);
  p.total = static_cast<uint32_t>(total);
  p.div_token = FastDiv::make(a->Hkv * (a->D / 8));
  p.div_head = FastDiv::make(a->D / 8);
  p.status = a->status;
  int64_t blocks = (total + 255) / 256;
  const int64_t cap = static_cast<int64_t>(sm_count_or(148)) * 32;
  if (blocks > cap) blocks = cap;
  launch_pdl(kv_append_packed_kernel, dim3(static_cast<unsigned>(blocks)), 256, 0,
             static_cast<cudaStream_t>(stream), p);
  return check_launch("kv_append_packed_kernel");
}

}  // extern "C"

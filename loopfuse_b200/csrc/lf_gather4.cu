// Keys and values of requests from a 4-bit cache, as packed bf16 rows: y_d = z + s (c_d - 8).
//
// The way from a 4-bit cache to the attention of prompts: chunks of several tokens are bound by their products, so
// their keys are unpacked once and read as ordinary packed keys by all heads' tiles. Bound by HBM: 5/8 byte
// read and 2 written per value.
#include "lf_cache4.cuh"

namespace lf {

struct Gather4Params {
  const char* k_pool;
  const char* v_pool;
  __nv_bfloat16* k_out;
  __nv_bfloat16* v_out;
  const int32_t* table;
  const int32_t* cu;
  int64_t bt_stride;
  int64_t kp_stride[3], vp_stride[3], ko_stride[2], vo_stride[2];
  int32_t B, T, Hkv, page_size, page_shift, n_pages, bt_blocks;
  int32_t* status;
};

__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// z + s (c - 8) for the codes at bits 0..3 of both halves, each with one rounding: 128 + c has its code in the last bits
// of its significand, and c - 8 is exact.
__device__ __forceinline__ uint32_t value2(uint32_t codes, uint32_t s, uint32_t z) {
  const uint32_t c = fma_bf16x2((codes & 0x000f000fu) | 0x43004300u, 0x3f803f80u, 0xc308c308u);  // 1 x (128 + c) - 136
  return fma_bf16x2(c, s, z);
}

// Tokens of a warp, CTAs of an SM, rows of a lane whose loads are in flight together. 55 thousand tokens of 8 heads,
// D = 128: 51 us; three CTAs of two rows 53 (four of them 59), eight tokens 58, sixteen 61.
constexpr int kGatherTokens = 4, kGatherCtas = 2, kGatherRows = 4;

template <int N>
__device__ __forceinline__ void ldg_words(const char* p, uint32_t (&x)[N]) {
  static_assert(N == 2 || N == 4, "pieces of 8 or 16 bytes");
  if constexpr (N == 4) {
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
    x[0] = r.x, x[1] = r.y, x[2] = r.z, x[3] = r.w;
  } else {
    const uint2 r = __ldg(reinterpret_cast<const uint2*>(p));
    x[0] = r.x, x[1] = r.y;
  }
}

// The request that row t belongs to: the first whose rows end behind it, or B. 32 ends are looked at at a time.
__device__ __forceinline__ int request_of(const int32_t* cu, int B, int t, int lane) {
  int lo = 0, n = B;
  for (;;) {
    const int step = (n + 31) >> 5, at = lo + (lane + 1) * step - 1;
    const bool behind = at < lo + n && cu[at + 1] <= t;
    const int skipped = __popc(__ballot_sync(0xffffffffu, behind)) * step;
    n = min(step - (step > 1 ? 1 : 0), n - skipped);
    lo += skipped;
    if (step == 1 || n <= 0) return lo;
  }
}

// A warp takes four tokens and all their heads, four lanes a row: a lane has a piece of a record, which holds eight
// columns of every group, and so reads 16 bytes (D = 64: 8) and writes 16 for each group, next to its neighbours'.
template <int D>
__global__ void __launch_bounds__(256, kGatherCtas) gather4_kernel(const Gather4Params p) {
  using R = Record4<D>;
  constexpr int NG = R::kGroups;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * kGatherTokens;
  if (first >= p.T) return;
  // Lane u: page and slot of token first + u.
  int page = -1, slot = 0;  // -1: a row that no request has; -2: no page
  {
    const int t = static_cast<int>(first) + lane;  // (T is 2^30 at most)
    bool open = lane < kGatherTokens && t < p.T;
    for (unsigned todo; (todo = __ballot_sync(0xffffffffu, open)) != 0;) {  // a request of the tokens at a time
      const int t0 = static_cast<int>(first) + __ffs(todo) - 1;
      const int b = request_of(p.cu, p.B, t0, lane);
      if (b >= p.B) break;
      const int from = max(p.cu[b], 0), end = p.cu[b + 1];
      if (open && from <= t && t < end) {
        const int at = t - from, block = p.page_shift >= 0 ? at >> p.page_shift : at / p.page_size;
        slot = at - block * p.page_size;
        if (!LF_BOUNDS(b >= 0 && at >= 0 && slot >= 0 && slot < p.page_size, p.status, 79)) slot = 0;
        page = block < p.bt_blocks ? p.table[b * p.bt_stride + block] : -1;
        if (page < 0 || page >= p.n_pages) {
          if (p.status) atomicCAS(p.status, 0, LF_DEV_BAD_PAGE);
          page = -2;
        }
      }
      open = open && t >= end && t != t0;
    }
  }
  const int i = lane & 3;
  const int u = (lane >> 2) % kGatherTokens;
  const int64_t pg = __shfl_sync(0xffffffffu, page, u);
  const int sl = __shfl_sync(0xffffffffu, slot, u);
  if (pg == -1) return;
  const char* kr = p.k_pool + max(pg, int64_t(0)) * p.kp_stride[0] + sl * p.kp_stride[1];
  const char* vr = p.v_pool + max(pg, int64_t(0)) * p.vp_stride[0] + sl * p.vp_stride[1];
  __nv_bfloat16* ko = p.k_out + (first + u) * p.ko_stride[0] + 8 * i;
  __nv_bfloat16* vo = p.v_out + (first + u) * p.vo_stride[0] + 8 * i;
#pragma unroll kGatherRows
  for (int h = (lane >> 2) / kGatherTokens; h < p.Hkv; h += 8 / kGatherTokens) {
    uint32_t kc[NG], vc[NG], km[NG], vm[NG];  // codes; scales, then midpoints
    ldg_words<NG>(kr + h * p.kp_stride[2] + i * R::kKeyPiece, kc);
    ldg_words<NG>(kr + h * p.kp_stride[2] + R::kScales, km);
    ldg_words<NG>(vr + h * p.vp_stride[2] + 2 * i * R::kValuePiece, vc);
    ldg_words<NG>(vr + h * p.vp_stride[2] + R::kScales, vm);
    uint4 ky[NG], vy[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {  // a key's word: columns e and e + 4 in its halves
      const uint32_t sel = g & 1 ? 0x3232u : 0x1010u;
      const uint32_t s = __byte_perm(km[g / 2], 0, sel), z = __byte_perm(km[NG / 2 + g / 2], 0, sel);
      uint32_t r[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = value2(kc[g] >> (4 * e), s, z);
      ky[g] = make_uint4(__byte_perm(r[0], r[1], 0x5410), __byte_perm(r[2], r[3], 0x5410),
                         __byte_perm(r[0], r[1], 0x7632), __byte_perm(r[2], r[3], 0x7632));
    }
#pragma unroll
    for (int g = 0; g < NG; g += 2) {  // a value's word: a column of groups g and g + 1 in its halves; two pieces
      const uint32_t s = vm[g / 2], z = vm[NG / 2 + g / 2];
      uint32_t r[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        r[e] = value2(vc[g / 2] >> (4 * e), s, z);
        r[4 + e] = value2(vc[NG / 2 + g / 2] >> (4 * e), s, z);
      }
      vy[g] = make_uint4(__byte_perm(r[0], r[1], 0x5410), __byte_perm(r[2], r[3], 0x5410),
                         __byte_perm(r[4], r[5], 0x5410), __byte_perm(r[6], r[7], 0x5410));
      vy[g + 1] = make_uint4(__byte_perm(r[0], r[1], 0x7632), __byte_perm(r[2], r[3], 0x7632),
                             __byte_perm(r[4], r[5], 0x7632), __byte_perm(r[6], r[7], 0x7632));
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if (pg < 0) ky[g] = vy[g] = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4*>(ko + h * p.ko_stride[1] + 32 * g) = ky[g];
      *reinterpret_cast<uint4*>(vo + h * p.vo_stride[1] + 32 * g) = vy[g];
    }
  }
}

}  // namespace lf

extern "C" int lf_kv_gather_4bit(const LfGather4Args* a, void* stream) {
  using namespace lf;
  if (!a || a->B <= 0 || a->T < 0 || a->Hkv <= 0 || a->page_size <= 0 || a->n_pages <= 0 || a->bt_blocks <= 0)
    return LF_ERR_INVALID_ARG;
  if (a->T == 0) return LF_OK;  // (empty tensors have no addresses)
  if (!a->k_pool || !a->v_pool || !a->k_out || !a->v_out || !a->block_table || !a->cu_k) return LF_ERR_INVALID_ARG;
  if (a->D != 64 && a->D != 128) return LF_ERR_UNSUPPORTED;
  if (a->Hkv > (1 << 20) || a->T > (1 << 30)) return LF_ERR_TOO_LARGE;
  if (!record4_aligned(a->k_pool, a->kp_stride, a->D) || !record4_aligned(a->v_pool, a->vp_stride, a->D))
    return LF_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(a->k_out) | reinterpret_cast<uintptr_t>(a->v_out)) & 15u) return LF_ERR_ALIGNMENT;
  for (int i = 0; i < 2; ++i)
    if (a->ko_stride[i] % 8 || a->vo_stride[i] % 8) return LF_ERR_ALIGNMENT;
  Gather4Params p = {};
  p.k_pool = static_cast<const char*>(a->k_pool);
  p.v_pool = static_cast<const char*>(a->v_pool);
  p.k_out = static_cast<__nv_bfloat16*>(a->k_out);
  p.v_out = static_cast<__nv_bfloat16*>(a->v_out);
  p.table = a->block_table;
  p.cu = a->cu_k;
  p.bt_stride = a->bt_stride;
  for (int i = 0; i < 3; ++i) {
    p.kp_stride[i] = a->kp_stride[i];
    p.vp_stride[i] = a->vp_stride[i];
  }
  for (int i = 0; i < 2; ++i) {
    p.ko_stride[i] = a->ko_stride[i];
    p.vo_stride[i] = a->vo_stride[i];
  }
  p.B = a->B;
  p.T = a->T;
  p.Hkv = a->Hkv;
  p.page_size = a->page_size;
  p.page_shift = shift_of(a->page_size);
  p.n_pages = a->n_pages;
  p.bt_blocks = a->bt_blocks;
  p.status = a->status;
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(a->T) + 8 * kGatherTokens - 1) / (8 * kGatherTokens));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->D == 128)
    launch_pdl(gather4_kernel<128>, dim3(grid), 256, 0, st, p);
  else
    launch_pdl(gather4_kernel<64>, dim3(grid), 256, 0, st, p);
  return check_launch("gather4_kernel");
}

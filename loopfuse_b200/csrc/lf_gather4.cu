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

constexpr int kGatherTokens = 4;  // of a warp

template <int D>
__device__ __forceinline__ uint4 decode8(uint32_t codes, const char* rec, int g) {
  using R = Record4<D>;
  const float s = bf16lo_to_f32(__ldg(reinterpret_cast<const unsigned short*>(rec + R::kScales + 2 * g)));
  const float z = bf16lo_to_f32(__ldg(reinterpret_cast<const unsigned short*>(rec + R::kMids + 2 * g)));
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)  // (the product is exact: one rounding in fp32, then the one to bf16)
    y[e] = fmaf(s, static_cast<float>(static_cast<int>((codes >> (4 * e)) & 15u) - 8), z);
  return make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                    pack_bf16x2(y[6], y[7]));
}

// A warp takes four tokens and all their heads; D / 8 lanes a row, so that consecutive slots of a head are read
// together.
template <int D>
__global__ void __launch_bounds__(256) gather4_kernel(const Gather4Params p) {
  using R = Record4<D>;
  constexpr int LPR = D / 8, RPW = 32 / LPR;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * kGatherTokens;
  if (first >= p.T) return;
  // Lane l: page and slot of token first + l % 4. Its request is the first that ends behind it.
  int page = -1, slot = 0;  // -1: a row that no request has; -2: no page
  {
    const int64_t t = first + lane % kGatherTokens;
    int lo = 0, hi = p.B;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (p.cu[mid + 1] > t) hi = mid;
      else lo = mid + 1;
    }
    if (t < p.T && lo < p.B) {
      const int from = max(p.cu[lo], 0);
      if (from <= t && p.cu[lo + 1] > t) {
        const int at = static_cast<int>(t) - from;
        const int block = p.page_shift >= 0 ? at >> p.page_shift : at / p.page_size;
        slot = at - block * p.page_size;
        page = block < p.bt_blocks ? p.table[lo * p.bt_stride + block] : -1;
        if (page < 0 || page >= p.n_pages) {
          if (p.status) atomicCAS(p.status, 0, LF_DEV_BAD_PAGE);
          page = -2;
        }
      }
    }
  }
  const int sub = lane % LPR, g = sub >> 2, i = sub & 3;
#pragma unroll 4
  for (int r0 = 0; r0 < kGatherTokens * p.Hkv; r0 += RPW) {
    const int r = r0 + lane / LPR;  // (four rows a head: all lanes have one)
    const int u = r % kGatherTokens, h = r / kGatherTokens;
    const int64_t pg = __shfl_sync(0xffffffffu, page, u);
    const int sl = __shfl_sync(0xffffffffu, slot, u);
    if (pg == -1) continue;
    uint4 ky = make_uint4(0u, 0u, 0u, 0u), vy = ky;
    if (pg >= 0) {
      const char* kr = p.k_pool + pg * p.kp_stride[0] + sl * p.kp_stride[1] + h * p.kp_stride[2];
      const char* vr = p.v_pool + pg * p.vp_stride[0] + sl * p.vp_stride[1] + h * p.vp_stride[2];
      const uint32_t kc = __ldg(reinterpret_cast<const uint32_t*>(kr + i * R::kKeyPiece + 4 * g));
      const uint32_t v0 = __ldg(reinterpret_cast<const unsigned short*>(vr + 2 * i * R::kValuePiece + 2 * g));
      const uint32_t v1 = __ldg(reinterpret_cast<const unsigned short*>(vr + (2 * i + 1) * R::kValuePiece + 2 * g));
      ky = decode8<D>(kc, kr, g);
      vy = decode8<D>(v0 | v1 << 16, vr, g);
    }
    const int64_t t = first + u;
    *reinterpret_cast<uint4*>(p.k_out + t * p.ko_stride[0] + h * p.ko_stride[1] + 8 * sub) = ky;
    *reinterpret_cast<uint4*>(p.v_out + t * p.vo_stride[0] + h * p.vo_stride[1] + 8 * sub) = vy;
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
  p.page_shift = cache_page_shift(a->page_size);
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

// Norm of each query and key head, rotation by position, and the append of the result to a paged cache of
// bf16 or of 4-bit records, in one pass over q, k and v.
//
//   x'_d = x_d * rsqrt(mean(x^2) + eps) * w_d
//   y_i = x'_i cos - x'_j sin,  y_j = x'_j cos + x'_i sin     (cos, sin: of the row's position and of i)
//   4 bits, per group of 32 columns: s = (max - min) / 15, z = min + 8 s, c = rint((y - z) / s) + 8
//
// Bound by HBM: every row is read once and written once; the arithmetic is some twenty operations per value.
#include "lf_cache4.cuh"

namespace lf {

struct RotaryParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  __nv_bfloat16* q_out;
  __nv_bfloat16* k_out;
  char* k_pool;
  char* v_pool;
  const int32_t* slots;
  const int32_t* positions;
  const float* table;
  const void* q_weight;
  const void* k_weight;
  int64_t table_stride;
  int64_t q_stride[2], k_stride[2], v_stride[2], qo_stride[2], ko_stride[2];
  int64_t kp_stride[3], vp_stride[3];  // bytes
  FastDiv div_parts;                   // parts of a token: runs of heads of q, then of k, then of v
  uint32_t items;                      // tokens times parts
  int32_t q_parts, k_parts;
  int32_t Hq, Hkv, rot, n_positions, interleaved, q_weight_f32, k_weight_f32;
  int32_t n_slots, page_size, page_shift;
  float eps;
  int32_t* status;
};

// (Plain loads: outputs may be the inputs.)
__device__ __forceinline__ uint4 ld_stream_16(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p)
               : "memory");
  return r;
}

__device__ __forceinline__ void unpack8(const uint4& r, float (&x)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16lo_to_f32(w[i]);
    x[2 * i + 1] = bf16hi_to_f32(w[i]);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                    pack_bf16x2(x[6], x[7]));
}

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
  x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// Largest and smallest that let a NaN through, so that it reaches the group's scale.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// The eight columns of a lane as codes of 4 bits, the first in the lowest bits; scale and midpoint of the group,
// which four neighbouring lanes share. Each step is rounded once (no fused product, no approximate
// division), so that a row has one encoding.
__device__ __forceinline__ uint32_t encode8(const float (&y)[8], uint16_t* scale, uint16_t* mid) {
  float lo = y[0], hi = y[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo = min_nan(lo, y[e]);
    hi = max_nan(hi, y[e]);
  }
#pragma unroll
  for (int d = 1; d <= 2; d <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, d));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, d));
  }
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f));
  const float s = __bfloat162float(sb);
  const __nv_bfloat16 zb = __float2bfloat16_rn(__fadd_rn(lo, __fmul_rn(8.f, s)));
  const float z = __bfloat162float(zb);
  const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = __fadd_rn(rintf(__fmul_rn(__fsub_rn(y[e], z), inv)), 8.f);
    w |= static_cast<uint32_t>(fminf(fmaxf(t, 0.f), 15.f)) << (4 * e);  // (a NaN becomes 0: its group has a NaN scale)
  }
  *scale = __bfloat16_as_ushort(sb);
  *mid = __bfloat16_as_ushort(zb);
  return w;
}

enum RotaryStore { kStoreRows = 0, kStorePool16 = 1, kStorePool4 = 2 };

// An item is a token and HEADS neighbouring heads of q, k or v, for D / 8 lanes with eight columns each: what a
// position needs of the table is read once for the heads, and their loads are in flight together.
template <int D, int HEADS, int STORE>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  constexpr int LPR = D / 8;  // lanes of a row
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, sub = lane % LPR;
  const uint32_t index = blockIdx.x * (256u / LPR) + threadIdx.x / LPR;
  const bool here = index < p.items;  // (the others compute along: rows exchange values across lanes)
  const uint32_t item = here ? index : p.items - 1;
  const uint32_t t = p.div_parts.div(item);
  const int part = static_cast<int>(item - t * p.div_parts.d);
  const bool is_q = part < p.q_parts;
  const bool is_v = STORE != kStoreRows && part >= p.q_parts + p.k_parts;
  const int heads = is_q ? p.Hq : p.Hkv;
  const int h0 = (is_q ? part : is_v ? part - p.q_parts - p.k_parts : part - p.q_parts) * HEADS;
  const __nv_bfloat16* src = is_q ? p.q + t * p.q_stride[0] : is_v ? p.v + t * p.v_stride[0]
                                                                  : p.k + t * p.k_stride[0];
  const int64_t src_head = is_q ? p.q_stride[1] : is_v ? p.v_stride[1] : p.k_stride[1];
  uint4 raw[HEADS];
#pragma unroll
  for (int u = 0; u < HEADS; ++u) {
    raw[u] = make_uint4(0u, 0u, 0u, 0u);
    if (here && h0 + u < heads) raw[u] = ld_stream_16(src + (h0 + u) * src_head + 8 * sub);
  }

  // Cosines and sines of this lane's columns.
  const int half = p.rot / 2;
  const bool turned = !is_v && 8 * sub < p.rot;
  float cs[8], sn[8];
  int partner = lane;
  float sign = 1.f;
  if (turned) {
    int pos = p.positions[t];
    if (pos < 0 || pos >= p.n_positions) {
      if (p.status && here) atomicCAS(p.status, 0, LF_DEV_BAD_POSITION);
      pos = min(max(pos, 0), p.n_positions - 1);
    }
    const float* row = p.table + pos * p.table_stride;
    if (p.interleaved) {
      const float4 c4 = *reinterpret_cast<const float4*>(row + 4 * sub);
      const float4 s4 = *reinterpret_cast<const float4*>(row + half + 4 * sub);
      cs[0] = cs[1] = c4.x, cs[2] = cs[3] = c4.y, cs[4] = cs[5] = c4.z, cs[6] = cs[7] = c4.w;
      sn[0] = sn[1] = s4.x, sn[2] = sn[3] = s4.y, sn[4] = sn[5] = s4.z, sn[6] = sn[7] = s4.w;
    } else {
      const bool first = 8 * sub < half;
      const int i = first ? 8 * sub : 8 * sub - half;
      load8(row + i, cs);
      load8(row + half + i, sn);
      partner = first ? lane + half / 8 : lane - half / 8;
      sign = first ? -1.f : 1.f;
    }
  }
  float weight[8];
  const void* wp = is_q ? p.q_weight : is_v ? nullptr : p.k_weight;
  if (wp) {
    if (is_q ? p.q_weight_f32 : p.k_weight_f32) {
      load8(static_cast<const float*>(wp) + 8 * sub, weight);
    } else {
      unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(wp) + 8 * sub), weight);
    }
  }
  // Where a cache row goes.
  bool stored = here;
  int64_t page = 0;
  int slot = 0;
  if constexpr (STORE != kStoreRows) {
    if (!is_q) {
      const int at = p.slots[t];
      stored = here && at >= 0 && at < p.n_slots;  // (negative: a row of the padding)
      if (stored) {
        page = p.page_shift >= 0 ? at >> p.page_shift : at / p.page_size;
        slot = at - static_cast<int>(page) * p.page_size;
      } else if (here && at >= 0 && p.status) {
        atomicCAS(p.status, 0, LF_DEV_BAD_PAGE);
      }
    }
  }

#pragma unroll
  for (int u = 0; u < HEADS; ++u) {
    float x[8], y[8];
    unpack8(raw[u], x);
    if (p.q_weight || p.k_weight) {  // (the same for all lanes)
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
      for (int d = 1; d < LPR; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
      if (wp) {
        const float r = rsqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * r * weight[e];
      }
    }
    if (p.interleaved) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        y[e] = turned ? __fsub_rn(__fmul_rn(x[e], cs[e]), __fmul_rn(x[e + 1], sn[e])) : x[e];
        y[e + 1] = turned ? __fadd_rn(__fmul_rn(x[e + 1], cs[e]), __fmul_rn(x[e], sn[e])) : x[e + 1];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = __shfl_sync(0xffffffffu, x[e], partner);
        y[e] = turned ? __fadd_rn(__fmul_rn(x[e], cs[e]), __fmul_rn(sign * other, sn[e])) : x[e];
      }
    }
    const int h = h0 + u;
    const bool store = stored && h < heads;
    if constexpr (STORE == kStorePool4) {
      using R = Record4<D>;
      uint16_t scale, mid;
      const uint32_t w = encode8(y, &scale, &mid);
      const int g = sub >> 2, i = sub & 3;
      // (A value's two halfwords lie in different pieces: lanes of neighbouring groups trade one for one, and each
      // stores a word.)
      const uint32_t traded = __shfl_xor_sync(0xffffffffu, (g & 1) ? w & 0xffffu : w >> 16, 4);
      if (!is_q && store) {
        const int64_t* st = is_v ? p.vp_stride : p.kp_stride;
        char* rec = (is_v ? p.v_pool : p.k_pool) + page * st[0] + slot * st[1] + h * st[2];
        if (is_v) {
          const uint32_t both = (g & 1) ? traded | (w & 0xffff0000u) : (w & 0xffffu) | traded << 16;
          *reinterpret_cast<uint32_t*>(rec + (2 * i + (g & 1)) * R::kValuePiece + 4 * (g >> 1)) = both;
        } else {
          *reinterpret_cast<uint32_t*>(rec + i * R::kKeyPiece + 4 * g) = w;
        }
        if (i < 2) *reinterpret_cast<uint16_t*>(rec + (i ? R::kMids : R::kScales) + 2 * g) = i ? mid : scale;
      }
      if (is_q && store)
        *reinterpret_cast<uint4*>(p.q_out + t * p.qo_stride[0] + h * p.qo_stride[1] + 8 * sub) = pack8(y);
    } else if (store) {
      char* dst;
      if (is_q)
        dst = reinterpret_cast<char*>(p.q_out + t * p.qo_stride[0] + h * p.qo_stride[1]);
      else if constexpr (STORE == kStoreRows)
        dst = reinterpret_cast<char*>(p.k_out + t * p.ko_stride[0] + h * p.ko_stride[1]);
      else if (is_v)
        dst = p.v_pool + page * p.vp_stride[0] + slot * p.vp_stride[1] + h * p.vp_stride[2];
      else
        dst = p.k_pool + page * p.kp_stride[0] + slot * p.kp_stride[1] + h * p.kp_stride[2];
      *reinterpret_cast<uint4*>(dst + 16 * sub) = pack8(y);
    }
  }
}

static bool rotary_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int D, int HEADS>
static void launch_rotary(const RotaryParams& p, int store, unsigned grid, cudaStream_t st) {
  if (store == kStoreRows)
    launch_pdl(rotary_kernel<D, HEADS, kStoreRows>, dim3(grid), 256, 0, st, p);
  else if (store == kStorePool16)
    launch_pdl(rotary_kernel<D, HEADS, kStorePool16>, dim3(grid), 256, 0, st, p);
  else
    launch_pdl(rotary_kernel<D, HEADS, kStorePool4>, dim3(grid), 256, 0, st, p);
}

}  // namespace lf

extern "C" int lf_rotary_bf16(const LfRotaryArgs* a, void* stream) {
  using namespace lf;
  if (!a || a->T < 0 || a->Hkv <= 0 || a->n_positions <= 0) return LF_ERR_INVALID_ARG;
  if (a->T == 0) return LF_OK;  // (empty tensors have no addresses)
  if (!a->k || !a->positions || !a->table) return LF_ERR_INVALID_ARG;
  const bool pools = a->k_pool != nullptr;
  if (a->q && (a->Hq <= 0 || !a->q_out)) return LF_ERR_INVALID_ARG;
  if (pools ? !a->v || !a->v_pool || !a->slots || a->page_size <= 0 || a->n_pages <= 0 : !a->k_out)
    return LF_ERR_INVALID_ARG;
  if (a->D != 64 && a->D != 128) return LF_ERR_UNSUPPORTED;
  if (a->rot <= 0 || a->rot > a->D || a->rot % 16) return LF_ERR_UNSUPPORTED;
  if (pools && a->bits != 16 && a->bits != 4) return LF_ERR_UNSUPPORTED;
  if (!(a->eps >= 0.f)) return LF_ERR_INVALID_ARG;
  const bool four = pools && a->bits == 4;
  for (const void* ptr : {a->q, a->k, a->v, static_cast<const void*>(a->q_out), static_cast<const void*>(a->k_out),
                          static_cast<const void*>(a->table), a->q_weight, a->k_weight})
    if (!rotary_aligned(ptr)) return LF_ERR_ALIGNMENT;
  for (int i = 0; i < 2; ++i) {
    if (a->k_stride[i] % 8) return LF_ERR_ALIGNMENT;
    if (a->q && (a->q_stride[i] % 8 || a->qo_stride[i] % 8)) return LF_ERR_ALIGNMENT;
    if (pools ? a->v_stride[i] % 8 : a->ko_stride[i] % 8) return LF_ERR_ALIGNMENT;
  }
  if (a->table_stride % 4) return LF_ERR_ALIGNMENT;
  if (four) {
    if (!record4_aligned(a->k_pool, a->kp_stride, a->D) || !record4_aligned(a->v_pool, a->vp_stride, a->D))
      return LF_ERR_ALIGNMENT;
  } else if (pools) {
    if (!rotary_aligned(a->k_pool) || !rotary_aligned(a->v_pool)) return LF_ERR_ALIGNMENT;
    for (int i = 0; i < 3; ++i)
      if (a->kp_stride[i] % 8 || a->vp_stride[i] % 8) return LF_ERR_ALIGNMENT;
  }
  if (pools && static_cast<int64_t>(a->n_pages) * a->page_size > 0x7fffffff) return LF_ERR_TOO_LARGE;

  RotaryParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.k = static_cast<const __nv_bfloat16*>(a->k);
  p.v = static_cast<const __nv_bfloat16*>(a->v);
  p.q_out = static_cast<__nv_bfloat16*>(a->q_out);
  p.k_out = static_cast<__nv_bfloat16*>(a->k_out);
  p.k_pool = static_cast<char*>(a->k_pool);
  p.v_pool = static_cast<char*>(a->v_pool);
  p.slots = a->slots;
  p.positions = a->positions;
  p.table = a->table;
  p.q_weight = a->q ? a->q_weight : nullptr;
  p.k_weight = a->k_weight;
  p.table_stride = a->table_stride;
  for (int i = 0; i < 2; ++i) {
    p.q_stride[i] = a->q_stride[i];
    p.k_stride[i] = a->k_stride[i];
    p.v_stride[i] = a->v_stride[i];
    p.qo_stride[i] = a->qo_stride[i];
    p.ko_stride[i] = a->ko_stride[i];
  }
  for (int i = 0; i < 3; ++i) {
    p.kp_stride[i] = a->kp_stride[i] * (four ? 1 : 2);
    p.vp_stride[i] = a->vp_stride[i] * (four ? 1 : 2);
  }
  p.Hq = a->q ? a->Hq : 0;
  p.Hkv = a->Hkv;
  p.rot = a->rot;
  p.n_positions = a->n_positions;
  p.interleaved = a->interleaved;
  p.q_weight_f32 = a->q_weight_f32;
  p.k_weight_f32 = a->k_weight_f32;
  p.eps = a->eps;
  p.status = a->status;
  if (pools) {
    p.n_slots = a->n_pages * a->page_size;
    p.page_size = a->page_size;
    p.page_shift = cache_page_shift(a->page_size);
  }
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  // Four heads an item; one where that leaves threads without work.
  const int64_t rows = static_cast<int64_t>(a->T) * (p.Hq + (pools ? 2 : 1) * p.Hkv);
  const int heads = rows * (a->D / 8) <= 2048ll * sms ? 1 : 4;
  p.q_parts = (p.Hq + heads - 1) / heads;
  p.k_parts = (p.Hkv + heads - 1) / heads;
  const int64_t parts = p.q_parts + static_cast<int64_t>(pools ? 2 : 1) * p.k_parts;
  if (parts * a->T > 0x7fffffff) return LF_ERR_TOO_LARGE;
  p.div_parts = FastDiv::make(static_cast<int32_t>(parts));
  p.items = static_cast<uint32_t>(parts * a->T);
  const unsigned per_cta = 256u / (a->D / 8);
  const unsigned grid = (p.items + per_cta - 1) / per_cta;
  const int store = !pools ? kStoreRows : four ? kStorePool4 : kStorePool16;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->D == 128)
    (heads == 1 ? launch_rotary<128, 1> : launch_rotary<128, 4>)(p, store, grid, st);
  else
    (heads == 1 ? launch_rotary<64, 1> : launch_rotary<64, 4>)(p, store, grid, st);
  return check_launch("rotary_kernel");
}

// Norm of each query and key head, rotation by position, and the append of the result to a paged cache of
// bf16 or of 4-bit records, in one pass over q, k and v.
//
//   x'_d = x_d * rsqrt(mean(x^2) + eps) * w_d
//   y_i = x'_i cos - x'_j sin,  y_j = x'_j cos + x'_i sin     (cos, sin: of the row's position and of i)
//   4 bits, per group of 32 columns: s = (max - min) / 15, z = min + 8 s, c = rint((y - z) / s) + 8
//
// Bound by HBM: every row is read once and written once; the arithmetic is some twenty operations per value.
#include "lf_cache4.cuh"

#include <type_traits>

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
  int32_t Hq, Hkv, rot, n_positions, q_weight_f32, k_weight_f32;
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

__device__ __forceinline__ void load4(const float* p, float* x) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
}
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  load4(p, x);
  load4(p + 4, x + 4);
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

// Scale and midpoint of a group from its smallest and largest value. Each step is rounded once (no fused product, no
// approximate division), so that a row has one encoding.
struct Group4 {
  uint16_t scale, mid;
  float z, inv;
};
__device__ __forceinline__ Group4 group_of(float lo, float hi) {
  Group4 g;
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f));
  const float s = __bfloat162float(sb);
  const __nv_bfloat16 zb = __float2bfloat16_rn(__fadd_rn(lo, __fmul_rn(8.f, s)));
  g.z = __bfloat162float(zb);
  g.inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
  g.scale = __bfloat16_as_ushort(sb);
  g.mid = __bfloat16_as_ushort(zb);
  return g;
}

__device__ __forceinline__ void range8(const float (&y)[8], float& lo, float& hi) {
  auto min3_nan = [](float a, float b, float c) {
    float d;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
  };
  auto max3_nan = [](float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
  };
  lo = min_nan(min3_nan(min3_nan(y[0], y[1], y[2]), y[3], y[4]), min3_nan(y[5], y[6], y[7]));
  hi = max_nan(max3_nan(max3_nan(y[0], y[1], y[2]), y[3], y[4]), max3_nan(y[5], y[6], y[7]));
}

// Eight columns as codes of 4 bits, the first in the lowest bits. A number in -8..7 plus 1.5 2^23 + 8 has its nearest
// whole number, plus 8, in its last bits (ties to even, as rint), above constant ones that the sum takes off. (A NaN
// becomes 0: its group has a NaN scale.)
__device__ __forceinline__ uint32_t codes8(const float (&y)[8], const Group4& g) {
  const uint64_t z2 = pack2(-g.z, -g.z), inv2 = pack2(g.inv, g.inv), magic = pack2(12582920.f, 12582920.f);
  uint32_t u[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float a, b;
    unpack2(mul2(add2(pack2(y[e], y[e + 1]), z2), inv2), a, b);
    a = fminf(fmaxf(a, -8.f), 7.f);
    b = fminf(fmaxf(b, -8.f), 7.f);
    unpack2(add2(pack2(a, b), magic), a, b);
    u[e] = __float_as_uint(a);
    u[e + 1] = __float_as_uint(b);
  }
  uint32_t w = u[7];
#pragma unroll
  for (int e = 6; e >= 0; --e) w = w * 16u + u[e];
  return w - 0x4b400000u * 0x11111111u;
}

// Heads of an item, and CTAs of an SM, with a norm and without: 21 thousand rows of 40 heads with a norm, four heads and
// three CTAs 78 us, two and four 80; the append of 33 thousand rows, two and four 124, four and three 126. (Chosen on
// whole rotations without pools. Normed forms of four heads spill 24 to 140 bytes a thread at these registers, most of
// them where a part is turned and pools are written: the append of 33 thousand rows with a norm takes 150 us whole, 156 in
// pairs, 172 for a part, where it takes 127 to 131 without.)
constexpr int rotary_heads(bool norm) { return norm ? 4 : 2; }
constexpr int rotary_ctas(bool norm) { return norm ? 3 : 4; }

enum RotaryStore { kStoreRows = 0, kStorePool16 = 1, kStorePool4 = 2 };  // where keys go

// An item is a token and HEADS neighbouring heads of q, k or v, for D / 16 lanes with two pieces of eight columns each:
// what a position needs of the table is read once for the heads, and their loads are in flight together. The pieces are
// such that what is turned together is in one lane, so that products go in pairs and nothing is traded between lanes:
//   kWhole, i with i + D / 2      pieces 8 l and D / 2 + 8 l, as for values
//   kPart, i with i + rot / 2     pieces 8 l and rot / 2 + 8 l; columns that are not turned: two neighbours
//   kPairs, 2 i with 2 i + 1      pieces 8 l and D / 2 + 8 l
// For 4 bits, a group of 32 columns is one piece of four lanes, or both pieces of two. (kWhole is kPart with rot = D, where
// known places save registers: 21 thousand rows of 40 heads with a norm 78 us instead of 82, a 4-bit append and gather of
// 22 thousand 56 instead of 62.)
enum RotaryLayout { kWhole = 0, kPart = 1, kPairs = 2 };
template <int D, int HEADS, int STORE, bool NORM, int LAYOUT>
__global__ void __launch_bounds__(256, rotary_ctas(NORM)) rotary_kernel(const RotaryParams p) {
  constexpr int LPR = D / 16;  // lanes of a row
  constexpr bool PAIRS = LAYOUT == kPairs;
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
  // First columns of the pieces; whether they are turned; whether a piece is a part of a group, or both are.
  const int half = LAYOUT == kWhole ? D / 2 : p.rot / 2;
  const bool split = LAYOUT != kPart || is_v;
  int ca = 8 * sub, cb = D / 2 + 8 * sub;
  const bool turned = !is_v && (LAYOUT == kWhole || ca < (PAIRS ? p.rot : half));
  [[maybe_unused]] const bool turned_b = PAIRS && !is_v && cb < p.rot;
  if (!split) {
    ca = turned ? 8 * sub : p.rot + 16 * (sub - half / 8);
    cb = turned ? half + 8 * sub : ca + 8;
  }
  [[maybe_unused]] const bool piece = split || (turned && half % 32 == 0);
  const __nv_bfloat16* src = is_q ? p.q + t * p.q_stride[0] : is_v ? p.v + t * p.v_stride[0]
                                                                  : p.k + t * p.k_stride[0];
  const int64_t src_head = is_q ? p.q_stride[1] : is_v ? p.v_stride[1] : p.k_stride[1];
  src += h0 * src_head;
  uint4 raw[HEADS][2];
#pragma unroll
  for (int u = 0; u < HEADS; ++u) {
    raw[u][0] = raw[u][1] = make_uint4(0u, 0u, 0u, 0u);
    if (here && h0 + u < heads) {
      raw[u][0] = ld_stream_16(src + u * src_head + ca);
      raw[u][1] = ld_stream_16(src + u * src_head + cb);
    }
  }
  // Cosines and sines of columns that are turned together; PAIRS: four of each piece.
  float cs[8], sn[8];
  if (turned || turned_b) {
    int pos = p.positions[t];
    if (pos < 0 || pos >= p.n_positions) {
      if (p.status && here) atomicCAS(p.status, 0, LF_DEV_BAD_POSITION);
      pos = min(max(pos, 0), p.n_positions - 1);
    }
    const float* row = p.table + pos * p.table_stride;
    if constexpr (PAIRS) {
      const int ia = ca / 2, ib = turned_b ? cb / 2 : ia;
      load4(row + ia, cs);
      load4(row + ib, cs + 4);
      load4(row + half + ia, sn);
      load4(row + half + ib, sn + 4);
    } else {
      load8(row + ca, cs);
      load8(row + half + ca, sn);
    }
  }
  const void* wp = !NORM || is_v ? nullptr : is_q ? p.q_weight : p.k_weight;
  const bool f32 = is_q ? p.q_weight_f32 : p.k_weight_f32;
  auto weights_of = [&](int at, float (&w)[8]) {
    if (f32)
      load8(static_cast<const float*>(wp) + at, w);
    else
      unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(wp) + at), w);
  };
  // Where the rows go.
  bool stored = here;
  char* dst;
  int64_t dst_head;
  if (is_q || STORE == kStoreRows) {
    dst = reinterpret_cast<char*>(is_q ? p.q_out + t * p.qo_stride[0] : p.k_out + t * p.ko_stride[0]);
    dst_head = 2 * (is_q ? p.qo_stride[1] : p.ko_stride[1]);
  } else {
    const int at = p.slots[t];
    stored = here && at >= 0 && at < p.n_slots;  // (negative: a row of the padding)
    if (here && at >= p.n_slots && p.status) atomicCAS(p.status, 0, LF_DEV_BAD_PAGE);
    const int safe = stored ? at : 0;
    const int page = p.page_shift >= 0 ? safe >> p.page_shift : safe / p.page_size;
    const int slot = safe - page * p.page_size;
    dst = is_v ? p.v_pool + page * p.vp_stride[0] + slot * p.vp_stride[1]
               : p.k_pool + page * p.kp_stride[0] + slot * p.kp_stride[1];
    dst_head = is_v ? p.vp_stride[2] : p.kp_stride[2];
  }
  dst += h0 * dst_head;
  if (!LF_BOUNDS(t < p.items / p.div_parts.d && h0 < heads && ca + 8 <= D && cb + 8 <= D, p.status, 78)) stored = false;

#pragma unroll
  for (int u = 0; u < HEADS; ++u) {
    float x[8], y[8];
    unpack8(raw[u][0], x);
    unpack8(raw[u][1], y);
    if constexpr (NORM) {
      uint64_t sum2 = 0;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint64_t a = pack2(x[e], x[e + 1]), b = pack2(y[e], y[e + 1]);
        sum2 = fma2(b, b, fma2(a, a, sum2));
      }
      float ss, odd;
      unpack2(sum2, ss, odd);
      ss += odd;
#pragma unroll
      for (int d = 1; d < LPR; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
      if (wp) {
        const float r = rsqrtf(ss * (1.f / D) + p.eps);
        const uint64_t r2 = pack2(r, r);
        auto scale = [&](float (&v)[8], const float (&by)[8]) {
#pragma unroll
          for (int e = 0; e < 8; e += 2)
            unpack2(mul2(mul2(pack2(v[e], v[e + 1]), r2), pack2(by[e], by[e + 1])), v[e], v[e + 1]);
        };
        float weight[8];  // (read again for each head: in registers all along they cost more than that)
        weights_of(ca, weight);
        scale(x, weight);
        weights_of(cb, weight);
        scale(y, weight);
      }
    }
    // (Each product and sum rounded once: pairs of products would be fused with the sums.)
    if constexpr (PAIRS) {
      auto turn = [](float (&v)[8], const float* c, const float* s) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = v[2 * e], b = v[2 * e + 1];
          v[2 * e] = __fsub_rn(__fmul_rn(a, c[e]), __fmul_rn(b, s[e]));
          v[2 * e + 1] = __fadd_rn(__fmul_rn(b, c[e]), __fmul_rn(a, s[e]));
        }
      };
      if (turned) turn(x, cs, sn);
      if (turned_b) turn(y, cs + 4, sn + 4);
    } else if (turned) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint64_t ac = pack2(__fmul_rn(x[e], cs[e]), __fmul_rn(x[e + 1], cs[e + 1]));
        const uint64_t bs = pack2(__fmul_rn(y[e], -sn[e]), __fmul_rn(y[e + 1], -sn[e + 1]));
        const uint64_t bc = pack2(__fmul_rn(y[e], cs[e]), __fmul_rn(y[e + 1], cs[e + 1]));
        const uint64_t as = pack2(__fmul_rn(x[e], sn[e]), __fmul_rn(x[e + 1], sn[e + 1]));
        unpack2(add2(ac, bs), x[e], x[e + 1]);
        unpack2(add2(bc, as), y[e], y[e + 1]);
      }
    }
    const bool store = stored && h0 + u < heads;
    char* to = dst + u * dst_head;
    if (STORE == kStorePool4) {
      using R = Record4<D>;
      float lo[2], hi[2];
      range8(x, lo[0], hi[0]);
      range8(y, lo[1], hi[1]);
      // A lane makes one group, of either piece or of both, and has the other's numbers from the lane that makes that.
      const bool second = piece && (sub & 2);
      float low = piece ? (second ? lo[1] : lo[0]) : min_nan(lo[0], lo[1]);
      float high = piece ? (second ? hi[1] : hi[0]) : max_nan(hi[0], hi[1]);
      const float low2 = __shfl_xor_sync(0xffffffffu, second ? lo[0] : lo[1], 2);
      const float high2 = __shfl_xor_sync(0xffffffffu, second ? hi[0] : hi[1], 2);
      if (piece) {
        low = min_nan(low, low2);
        high = max_nan(high, high2);
      }
      low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, 1));
      high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, 1));
      const Group4 mine = group_of(low, high);
      Group4 gx = mine, gy = mine;
      {
        const float z = __shfl_xor_sync(0xffffffffu, mine.z, 2), inv = __shfl_xor_sync(0xffffffffu, mine.inv, 2);
        if (piece) {
          gx.z = second ? z : mine.z, gx.inv = second ? inv : mine.inv;
          gy.z = second ? mine.z : z, gy.inv = second ? mine.inv : inv;
        }
      }
      if (!is_q) {
        const uint32_t wx = codes8(x, gx), wy = codes8(y, gy);
        const int ga = ca / 32, ia = ca / 8 % 4, gb = cb / 32, ib = cb / 8 % 4;
        if (store) {
          if (is_v) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              char* pa = to + (2 * ia + j) * R::kValuePiece + 2 * ga;
              char* pb = to + (2 * ib + j) * R::kValuePiece + 2 * gb;
              *reinterpret_cast<uint16_t*>(pa) = static_cast<uint16_t>(wx >> (16 * j));
              *reinterpret_cast<uint16_t*>(pb) = static_cast<uint16_t>(wy >> (16 * j));
            }
          } else {
            *reinterpret_cast<uint32_t*>(to + ia * R::kKeyPiece + 4 * ga) = wx;
            *reinterpret_cast<uint32_t*>(to + ib * R::kKeyPiece + 4 * gb) = wy;
          }
          // (A lane each for the scale and the midpoint of a group.)
          *reinterpret_cast<uint16_t*>(to + (sub & 1 ? R::kMids : R::kScales) + 2 * (second ? gb : ga)) =
              sub & 1 ? mine.mid : mine.scale;
        }
        continue;
      }
    }
    if (store) {
      *reinterpret_cast<uint4*>(to + 2 * ca) = pack8(x);
      *reinterpret_cast<uint4*>(to + 2 * cb) = pack8(y);
    }
  }
}

// The same for keys of 4 bits of which a part is turned whose halves are neither whole groups of 32 columns nor lie in one:
// a lane has eight neighbouring columns, four lanes are a group, and what is turned together is traded between lanes.
// (21 thousand rows of 40 heads, D = 128, to bf16 with the norm: 108 us in this layout, 78 in the other.)
template <int D>
__global__ void __launch_bounds__(256) rotary_odd_kernel(const RotaryParams p) {
  constexpr int HEADS = 4;
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
  const bool is_v = part >= p.q_parts + p.k_parts;
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
    const bool first = 8 * sub < half;
    const int i = first ? 8 * sub : 8 * sub - half;
    load8(row + i, cs);
    load8(row + half + i, sn);
    partner = first ? lane + half / 8 : lane - half / 8;
    sign = first ? -1.f : 1.f;
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
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float other = __shfl_sync(0xffffffffu, x[e], partner);
      y[e] = turned ? __fadd_rn(__fmul_rn(x[e], cs[e]), __fmul_rn(sign * other, sn[e])) : x[e];
    }
    const int h = h0 + u;
    const bool store = stored && h < heads;
    using R = Record4<D>;
    float lo, hi;
    range8(y, lo, hi);
#pragma unroll
    for (int d = 1; d <= 2; d <<= 1) {  // (four lanes a group)
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, d));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, d));
    }
    const Group4 group = group_of(lo, hi);
    const uint32_t w = codes8(y, group);
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
      if (i < 2) *reinterpret_cast<uint16_t*>(rec + (i ? R::kMids : R::kScales) + 2 * g) = i ? group.mid : group.scale;
    }
    if (is_q && store)
      *reinterpret_cast<uint4*>(p.q_out + t * p.qo_stride[0] + h * p.qo_stride[1] + 8 * sub) = pack8(y);
  }
}

template <int D, int STORE, int LAYOUT>
static void launch_rotary(const RotaryParams& p, bool few, unsigned grid, cudaStream_t st) {
  const auto normed = few ? rotary_kernel<D, 1, STORE, true, LAYOUT>
                          : rotary_kernel<D, rotary_heads(true), STORE, true, LAYOUT>;
  const auto plain = few ? rotary_kernel<D, 1, STORE, false, LAYOUT>
                         : rotary_kernel<D, rotary_heads(false), STORE, false, LAYOUT>;
  launch_pdl(p.q_weight || p.k_weight ? normed : plain, dim3(grid), 256, 0, st, p);
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
    if (!aligned_16(ptr)) return LF_ERR_ALIGNMENT;
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
    if (!aligned_16(a->k_pool) || !aligned_16(a->v_pool)) return LF_ERR_ALIGNMENT;
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
  p.q_weight_f32 = a->q_weight_f32;
  p.k_weight_f32 = a->k_weight_f32;
  p.eps = a->eps;
  p.status = a->status;
  if (pools) {
    p.n_slots = a->n_pages * a->page_size;
    p.page_size = a->page_size;
    p.page_shift = shift_of(a->page_size);
  }
  static thread_local int cached_dev = -1, sms = 148;
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev != cached_dev) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms = 148;
    cached_dev = dev;
  }
  // Several heads an item: what is read for the token serves them all. One where that leaves threads without work.
  const int store = !pools ? kStoreRows : four ? kStorePool4 : kStorePool16;
  const bool norm = p.q_weight || p.k_weight;
  const bool odd = four && !a->interleaved && a->rot > 32 && a->rot % 64 != 0;
  const int lanes = a->D / (odd ? 8 : 16);
  const int64_t rows = static_cast<int64_t>(a->T) * (p.Hq + (pools ? 2 : 1) * p.Hkv);
  const bool few = rows * lanes <= 2048ll * sms;
  const int heads = odd ? 4 : few ? 1 : rotary_heads(norm);
  p.q_parts = (p.Hq + heads - 1) / heads;
  p.k_parts = (p.Hkv + heads - 1) / heads;
  const int64_t parts = p.q_parts + static_cast<int64_t>(pools ? 2 : 1) * p.k_parts;
  if (parts * a->T > 0x7fffffff) return LF_ERR_TOO_LARGE;
  p.div_parts = FastDiv::make(static_cast<int32_t>(parts));
  p.items = static_cast<uint32_t>(parts * a->T);
  const unsigned per_cta = 256u / lanes;
  const unsigned grid = (p.items + per_cta - 1) / per_cta;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto pick = [&](auto d, auto to) {
    constexpr int D = decltype(d)::value, STORE = decltype(to)::value;
    const auto run = a->interleaved ? launch_rotary<D, STORE, kPairs>
                     : a->rot == D  ? launch_rotary<D, STORE, kWhole>
                                    : launch_rotary<D, STORE, kPart>;
    run(p, few, grid, st);
  };
  auto with_d = [&](auto d) {
    if (odd)
      launch_pdl(rotary_odd_kernel<decltype(d)::value>, dim3(grid), 256, 0, st, p);
    else if (store == kStoreRows)
      pick(d, std::integral_constant<int, kStoreRows>{});
    else if (store == kStorePool16)
      pick(d, std::integral_constant<int, kStorePool16>{});
    else
      pick(d, std::integral_constant<int, kStorePool4>{});
  };
  if (a->D == 128)
    with_d(std::integral_constant<int, 128>{});
  else
    with_d(std::integral_constant<int, 64>{});
  return check_launch("rotary_kernel");
}

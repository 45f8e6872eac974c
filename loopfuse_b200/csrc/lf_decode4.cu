// Decode attention over a 4-bit paged cache: one query token per request, requests of any lengths.
//
// With codes c, scales s and midpoints z of the groups g of 32 columns (include/lf_sm100.h has the format),
//   score_j = sum_g sK_jg (q_g . (cK_jg - 8)) + sum_g zK_jg sum(q_g)
//   o       = sum_g sum_j (p_j sV_jg) (cV_jg - 8) + sum_g sum_j p_j zV_jg,    p_j = 2^(score_j - m),
// so a cache row is never unpacked to its values: the codes become bf16 by setting an exponent above them
// (128 + c, or 16 + c three bits up), which a matrix instruction takes as they are; scales are applied to the
// scores of a group and to the weights, and what the exponents added comes off where it was added: a group's scores
// start at minus that times the sums of q, and the weights meet the same constants, negative, in a product of their own.
//
// Bound by HBM, 5/8 byte per value: an SM has to take some 40 values a clock, so the instructions per value count
// (a quarter of one per lane and key value, as much per value of V).
#include "lf_cache4.cuh"
#include "lf_join.cuh"
#include "lf_packed.cuh"

#include <algorithm>
#include <type_traits>

namespace lf {

constexpr int kD4Warps = 4;
constexpr int kD4Stages = 3;   // groups of a warp's ring: two are copied while one is computed
constexpr int kD4Group = 32;   // tokens that a warp takes at a time
constexpr int kD4Run = 1;      // groups of a warp, at least
constexpr int kD4Ctas = 3;     // of an SM

struct Decode4Params {
  const __nv_bfloat16* q;
  const char* k;
  const char* v;
  int64_t q_stride[3], k_stride[3], v_stride[3];  // (b, kv head, g); bytes of (page, slot, kv head)
  const int32_t* table;
  int64_t bt_stride;
  const int32_t* seq_lens;
  int32_t B, G;
  int32_t heads;       // units of a request: kv heads times groups of 8 query heads
  FastDiv div_groups;  // groups of query heads
  int32_t window, max_len;
  int32_t bt_blocks, page_size, page_shift, n_pages;
  float a, c2;
  // Part of warp w for unit u: at place w + u, which no other pair has, since both only grow along the row
  // of groups; [place][8 query heads][D], (maximum, sum), and the warps that a unit's groups went to.
  float* part_o;
  float2* part_ml;
  int2* warps;
  int32_t* status;
};

__device__ __forceinline__ void mma_bf16(float& d0, float& d1, float& d2, float& d3, uint32_t a0, uint32_t a1,
                                         uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d0), "+f"(d1), "+f"(d2), "+f"(d3)
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 matrix of 16-bit values held by a warp, two neighbours of a row per lane.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Codes at bits 0..3 of both halves of a word -> 128 + c as bf16; at bits 3..6 -> 16 + c.
__device__ __forceinline__ uint32_t code_128(uint32_t w) { return (w & 0x000f000fu) | 0x43004300u; }
__device__ __forceinline__ uint32_t code_16(uint32_t w) { return (w & 0x00780078u) | 0x41804180u; }
constexpr float kOff128 = 136.f, kOff16 = 24.f;  // what has to come off, so that c - 8 is left

template <int BYTES>
__device__ __forceinline__ void cp_async_piece(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    cp_async_16(dst, src);
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

// The first key of a unit's groups: that of the window, or of the sixteen it lies in (pages of 16 and more then
// hold whole halves of a group).
__device__ __forceinline__ int first_token(int end, int window) {
  return window > 0 && end > window ? (end - window) & ~15 : 0;
}

// Thirty-two tokens of a unit, as a warp has them in hand.
struct D4Group {
  int b, head;  // request; kv head and group of query heads. b < 0: no more
  int t, end;   // first token, end of the unit
};

// All units' groups of 32 tokens are one row, of which warp `w` of `n_warps` has an equal run, whatever the
// requests' lengths; page look-ups, copies and products of following groups overlap across units.
//
// Products, m16n8k16 with the eight query heads as its columns:
//   scores  rows: 16 keys, 8 code columns of each per lane. Lane (g, c) = (lane / 4, lane % 4) has keys g and
//           g + 8 and reads their piece c, whose word of a column group feeds two instructions; its four scores
//           are keys g, g + 8 of query heads 2c, 2c + 1.
//   output  rows: 16 columns of V, inner dimension: 16 keys. Lane (g, c) reads piece g of keys 2c, 2c + 1, 2c + 8,
//           2c + 9 and pairs halfwords of two keys. The weights, times the scale of a column group and rounded to
//           bf16, get from the first product's layout to the second's by two 8 x 8 transposes.
template <int D, bool SOFTCAP>
__global__ void __launch_bounds__(kD4Warps * 32, kD4Ctas) decode4_kernel(const Decode4Params p) {
  using R = Record4<D>;
  constexpr int NG = R::kGroups;
  constexpr int kHalf = kD4Group * R::kBytes;  // keys, then values
  constexpr int kStageBytes = 2 * kHalf;
  constexpr int kPieces = R::kBytes / R::kAlign;  // of a record: 5
  static_assert(kPieces * kD4Group % 32 == 0, "a group's pieces are dealt out evenly");
  extern __shared__ __align__(1024) unsigned char smem[];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  // (Runs go round the CTAs first, then their warps: few of them are spread over all SMs.)
  const int w = warp * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x);
  const int n_warps = static_cast<int>(gridDim.x) * kD4Warps;

  // Groups of the requests [b0, b0 + 32), one per lane; those of a unit.
  int b0 = 0, groups = 0;
  auto load_groups = [&](int from) {
    b0 = from;
    const int end = b0 + lane < p.B ? own_end(p.seq_lens, b0 + lane, p.max_len) : 0;
    groups = end > 0 ? (end - first_token(end, p.window) + kD4Group - 1) / kD4Group : 0;
  };
  long long all = 0;
#pragma unroll 4
  for (int from = 0; from < p.B; from += 32) {
    load_groups(from);
    all += groups;
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
  all *= p.heads;
  const long long run = max((all + n_warps - 1) / n_warps, static_cast<long long>(kD4Run));
  long long left = min(all - w * run, run);  // groups of this warp
  if (left <= 0) return;
  D4Group now;
  {
    long long skip = w * run;  // of the requests ahead, then of the units ahead
    long long incl = 0;
    unsigned past = 0;
    for (int from = 0; from < p.B && !past; from += 32) {
      if (from) skip -= __shfl_sync(0xffffffffu, incl, 31);
      load_groups(from);
      incl = static_cast<long long>(groups) * p.heads;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += x;
      }
      past = __ballot_sync(0xffffffffu, incl > skip);
    }
    const int l = __ffs(past) - 1;
    const int n = __shfl_sync(0xffffffffu, groups, l);
    const long long into = skip - __shfl_sync(0xffffffffu, incl, l) + static_cast<long long>(n) * p.heads;
    now.b = b0 + l;
    now.head = static_cast<int>(into / n);
    now.end = own_end(p.seq_lens, now.b, p.max_len);
    now.t = first_token(now.end, p.window) + static_cast<int>(into - static_cast<long long>(now.head) * n) * kD4Group;
  }
  // The group behind x, while this warp has any.
  auto next_group = [&](const D4Group& x) {
    D4Group y = x;
    if (--left <= 0) {
      y.b = -1;
      return y;
    }
    y.t += kD4Group;
    if (y.t < y.end) return y;
    y.t = first_token(y.end, p.window);
    if (++y.head < p.heads) return y;
    y.head = 0;
    for (;;) {  // the next request that has keys
      const unsigned some = __ballot_sync(0xffffffffu, groups > 0 && b0 + lane > y.b);
      if (some) {
        y.b = b0 + __ffs(some) - 1;
        y.end = own_end(p.seq_lens, y.b, p.max_len);
        y.t = first_token(y.end, p.window);
        return y;
      }
      load_groups(b0 + 32);
    }
  };
  auto kv_head = [&](int head, int* g0) {
    const int kvh = static_cast<int>(p.div_groups.div(head));
    *g0 = (head - kvh * static_cast<int>(p.div_groups.d)) * kOwnHeads;
    return kvh;
  };

  auto page_of = [&](int t) { return p.page_shift >= 0 ? (t >> p.page_shift) : (t / p.page_size); };
  // The token that this lane finds for a group: rows past the end repeat the last, rows in front of the window
  // its first.
  auto token_of = [&](const D4Group& x) {
    const int from = p.window > 0 ? max(x.end - p.window, 0) : 0;
    return max(min(x.t + lane, x.end - 1), from);
  };
  auto look_up = [&](const D4Group& x) {
    if (x.b < 0) return 0;
    const int at = page_of(token_of(x));
    if (!LF_BOUNDS(x.b < p.B && x.head < p.heads && at >= 0 && at < p.bt_blocks, p.status, 75)) return 0;
    return p.table[x.b * p.bt_stride + at];
  };
  unsigned char* ring = smem + warp * (kD4Stages * kStageBytes);
  const uint32_t ring_u32 = smem_u32(ring);
  auto copy_group = [&](const D4Group& x, int stage, int page) {
    if (x.b >= 0) {
      int g0;
      const int kvh = kv_head(x.head, &g0);
      const int t = token_of(x);
      if (page < 0 || page >= p.n_pages) {
        if (p.status) atomicExch(p.status, LF_DEV_BAD_PAGE);
        page = 0;
      }
      int slot = t - page_of(t) * p.page_size;
      if (!LF_BOUNDS(slot >= 0 && slot < p.page_size && stage >= 0 && stage < kD4Stages, p.status, 76)) slot = 0;
      const char* krow = p.k + kvh * p.k_stride[2] + page * p.k_stride[0] + slot * p.k_stride[1];
      const char* vrow = p.v + kvh * p.v_stride[2] + page * p.v_stride[0] + slot * p.v_stride[1];
      const uint32_t dst = ring_u32 + stage * kStageBytes;
#pragma unroll
      for (int i = 0; i < kPieces * kD4Group / 32; ++i) {
        const int id = lane + 32 * i, row = id / kPieces, piece = id - row * kPieces;
        const char* kp = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(krow), row));
        const char* vp = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(vrow), row));
        cp_async_piece<R::kAlign>(dst + id * R::kAlign, kp + piece * R::kAlign);
        cp_async_piece<R::kAlign>(dst + kHalf + id * R::kAlign, vp + piece * R::kAlign);
      }
    }
    cp_async_commit();
  };

  // The query heads of a unit: columns of the first product, in the order that the codes have; what the
  // accumulators of a column group start at (heads 2c, 2c + 1); and the sums of the columns, which go with the
  // midpoints, as three bf16 each.
  uint32_t qf[NG][4];
  float start[NG][2];
  uint32_t sum_b0 = 0, sum_b1 = 0;
  auto load_q = [&](const D4Group& x) {
    int g0;
    const int kvh = kv_head(x.head, &g0);
    float sum[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      uint4 r = make_uint4(0u, 0u, 0u, 0u);
      if (g0 + g < p.G)
        r = *reinterpret_cast<const uint4*>(p.q + x.b * p.q_stride[0] + kvh * p.q_stride[1] +
                                            (g0 + g) * p.q_stride[2] + 32 * n + 8 * c);
      qf[n][0] = __byte_perm(r.x, r.z, 0x5410);  // columns 0 and 4 of the eight
      qf[n][1] = __byte_perm(r.x, r.z, 0x7632);  // 1, 5
      qf[n][2] = __byte_perm(r.y, r.w, 0x5410);  // 2, 6
      qf[n][3] = __byte_perm(r.y, r.w, 0x7632);  // 3, 7
      float even = bf16lo_to_f32(r.x) + bf16lo_to_f32(r.y) + bf16lo_to_f32(r.z) + bf16lo_to_f32(r.w);
      float odd = bf16hi_to_f32(r.x) + bf16hi_to_f32(r.y) + bf16hi_to_f32(r.z) + bf16hi_to_f32(r.w);
#pragma unroll
      for (int d = 1; d <= 2; d <<= 1) {
        even += __shfl_xor_sync(0xffffffffu, even, d);
        odd += __shfl_xor_sync(0xffffffffu, odd, d);
      }
      sum[n] = even + odd;
      const float off = -(kOff128 * even + kOff16 * odd);
      start[n][0] = __shfl_sync(0xffffffffu, off, 8 * c);
      start[n][1] = __shfl_sync(0xffffffffu, off, 8 * c + 4);
    }
    // Inner index 2c, 2c + 1 (and 8 more) of the midpoints' product: a pair of column groups, and a part of the sums.
    uint32_t part[3][NG / 2];
#pragma unroll
    for (int n = 0; n < NG / 2; ++n) {
      float x0 = sum[2 * n], x1 = sum[2 * n + 1];
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        part[i][n] = pack_bf16x2(x0, x1);
        x0 -= bf16lo_to_f32(part[i][n]);
        x1 -= bf16hi_to_f32(part[i][n]);
      }
    }
    if constexpr (NG == 4) {
      sum_b0 = c == 0 ? part[0][0] : c == 1 ? part[0][1] : c == 2 ? part[1][0] : part[1][1];
      sum_b1 = c == 0 ? part[2][0] : c == 1 ? part[2][1] : 0u;
    } else {
      sum_b0 = c == 0 ? part[0][0] : c == 1 ? part[1][0] : c == 2 ? part[2][0] : 0u;
      sum_b1 = 0u;
    }
  };

  // now: computed; then, later: being copied; ahead, last: their pages are being looked up.
  static_assert(kD4Stages == 3, "two groups are copied while one is computed");
  D4Group then = next_group(now), later = next_group(then);
  load_q(now);
  {
    const int pg0 = look_up(now), pg1 = look_up(then);
    copy_group(now, 0, pg0);
    copy_group(then, 1, pg1);
  }
  D4Group ahead = next_group(later);
  int page = look_up(later), page_ahead = look_up(ahead);

  // Query heads 2c, 2c + 1.
  float m_run[2], l_run[2], mids[NG][2];
  float o[2 * NG][4];  // rows of instruction 2n + h: columns 32 n + 4 g + 2 h, then + 1; each for both heads
  auto clear = [&] {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      m_run[r] = -INFINITY;
      l_run[r] = 0.f;
#pragma unroll
      for (int n = 0; n < NG; ++n) mids[n][r] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < 2 * NG; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  };
  clear();

  for (int it = 0; now.b >= 0; it = it == 2 ? 0 : it + 1) {
    copy_group(later, it == 0 ? 2 : it - 1, page);
    const D4Group last = next_group(ahead);
    page = page_ahead;
    page_ahead = look_up(last);
    cp_async_wait<kD4Stages - 1>();
    __syncwarp();
    const unsigned char* stage = ring + it * kStageBytes;

    float sc[2][4];  // [half of the group]: key g (two heads), key g + 8
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned char* k0 = stage + (16 * h + g) * R::kBytes;
      const unsigned char* k1 = k0 + 8 * R::kBytes;
      uint32_t w0[NG], w1[NG], s0[NG / 2], s1[NG / 2];
      if constexpr (NG == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(k0 + 16 * c), y = *reinterpret_cast<const uint4*>(k1 + 16 * c);
        w0[0] = x.x, w0[1] = x.y, w0[2] = x.z, w0[3] = x.w;
        w1[0] = y.x, w1[1] = y.y, w1[2] = y.z, w1[3] = y.w;
        const uint2 u = *reinterpret_cast<const uint2*>(k0 + R::kScales), v = *reinterpret_cast<const uint2*>(k1 + R::kScales);
        s0[0] = u.x, s0[1] = u.y, s1[0] = v.x, s1[1] = v.y;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(k0 + 8 * c), y = *reinterpret_cast<const uint2*>(k1 + 8 * c);
        w0[0] = x.x, w0[1] = x.y;
        w1[0] = y.x, w1[1] = y.y;
        s0[0] = *reinterpret_cast<const uint32_t*>(k0 + R::kScales);
        s1[0] = *reinterpret_cast<const uint32_t*>(k1 + R::kScales);
      }
      const int pair = NG == 4 ? 4 * (c & 1) : 0;
      const uint32_t z0 = *reinterpret_cast<const uint32_t*>(k0 + R::kMids + pair);
      const uint32_t z1 = *reinterpret_cast<const uint32_t*>(k1 + R::kMids + pair);
      float x0 = 0.f, x1 = 0.f, x2 = 0.f, x3 = 0.f;
      mma_bf16(x0, x1, x2, x3, z0, z1, z0, z1, sum_b0, sum_b1);
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float y0 = start[n][0], y1 = start[n][1], y2 = start[n][0], y3 = start[n][1];
        mma_bf16(y0, y1, y2, y3, code_128(w0[n]), code_128(w1[n]), code_16(w0[n] >> 1), code_16(w1[n] >> 1),
                 qf[n][0], qf[n][1]);
        mma_bf16(y0, y1, y2, y3, code_128(w0[n] >> 8), code_128(w1[n] >> 8), code_16(w0[n] >> 9),
                 code_16(w1[n] >> 9), qf[n][2], qf[n][3]);
        const float a = n & 1 ? bf16hi_to_f32(s0[n / 2]) : bf16lo_to_f32(s0[n / 2]);
        const float b = n & 1 ? bf16hi_to_f32(s1[n / 2]) : bf16lo_to_f32(s1[n / 2]);
        x0 = fmaf(a, y0, x0);
        x1 = fmaf(a, y1, x1);
        x2 = fmaf(b, y2, x2);
        x3 = fmaf(b, y3, x3);
      }
      sc[h][0] = x0, sc[h][1] = x1, sc[h][2] = x2, sc[h][3] = x3;
    }

    const int from = p.window > 0 ? now.end - p.window : 0;
    const bool edge = now.t < from || now.t + kD4Group > now.end;
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float s = sc[h][e];
        if constexpr (SOFTCAP) s = tanh_approx(s * p.a);  // (the unit's, within 2^-11, as in decode)
        s *= p.c2;
        if (edge) {
          const int t = now.t + 16 * h + g + 8 * (e >> 1);
          if (t < from || t >= now.end) s = -INFINITY;
        }
        sc[h][e] = s;
        mx[e & 1] = fmaxf(mx[e & 1], s);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int d = 4; d <= 16; d <<= 1) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], d));
      mx[r] = fmaxf(mx[r], m_run[r]);
    }
    const float m_safe[2] = {mx[0] == -INFINITY ? 0.f : mx[0], mx[1] == -INFINITY ? 0.f : mx[1]};
    if (__any_sync(0xffffffffu, mx[0] > m_run[0] || mx[1] > m_run[1])) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float alpha = ex2_approx(m_run[r] - m_safe[r]);
        m_run[r] = mx[r];
        l_run[r] *= alpha;
#pragma unroll
        for (int n = 0; n < NG; ++n) mids[n][r] *= alpha;
#pragma unroll
        for (int n = 0; n < 2 * NG; ++n) {
          o[n][r] *= alpha;
          o[n][2 + r] *= alpha;
        }
      }
    }

#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float pr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pr[e] = ex2_approx(sc[h][e] - m_safe[e & 1]);
        l_run[e & 1] += pr[e];  // this lane's share; the keys are summed at the end of the unit
      }
      const unsigned char* v = stage + kHalf + 16 * h * R::kBytes;
      const unsigned char* m0 = v + g * R::kBytes + R::kScales;
      const unsigned char* m1 = m0 + 8 * R::kBytes;
      uint32_t s0[NG], s1[NG];  // scales, then midpoints, of keys g and g + 8
      if constexpr (NG == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(m0), y = *reinterpret_cast<const uint4*>(m1);
        s0[0] = x.x, s0[1] = x.y, s0[2] = x.z, s0[3] = x.w;
        s1[0] = y.x, s1[1] = y.y, s1[2] = y.z, s1[3] = y.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(m0), y = *reinterpret_cast<const uint2*>(m1);
        s0[0] = x.x, s0[1] = x.y;
        s1[0] = y.x, s1[1] = y.y;
      }
      // Codes of keys 2c, 2c + 1, 2c + 8, 2c + 9: [key][pair of column groups].
      uint32_t cv[4][NG / 2];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const unsigned char* at = v + (2 * c + (r & 1) + 8 * (r >> 1)) * R::kBytes + g * R::kValuePiece;
        if constexpr (NG == 4) {
          const uint2 x = *reinterpret_cast<const uint2*>(at);
          cv[r][0] = x.x, cv[r][1] = x.y;
        } else {
          cv[r][0] = *reinterpret_cast<const uint32_t*>(at);
        }
      }
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const float a = n & 1 ? bf16hi_to_f32(s0[n / 2]) : bf16lo_to_f32(s0[n / 2]);
        const float b = n & 1 ? bf16hi_to_f32(s1[n / 2]) : bf16lo_to_f32(s1[n / 2]);
        const float za = n & 1 ? bf16hi_to_f32(s0[NG / 2 + n / 2]) : bf16lo_to_f32(s0[NG / 2 + n / 2]);
        const float zb = n & 1 ? bf16hi_to_f32(s1[NG / 2 + n / 2]) : bf16lo_to_f32(s1[NG / 2 + n / 2]);
#pragma unroll
        for (int r = 0; r < 2; ++r) mids[n][r] = fmaf(pr[r], za, fmaf(pr[2 + r], zb, mids[n][r]));
        const uint32_t pb0 = transpose_8x8(pack_bf16x2(pr[0] * a, pr[1] * a));
        const uint32_t pb1 = transpose_8x8(pack_bf16x2(pr[2] * b, pr[3] * b));
        const uint32_t sel = n & 1 ? 0x7632u : 0x5410u;
        const uint32_t x = __byte_perm(cv[0][n / 2], cv[1][n / 2], sel);
        const uint32_t y = __byte_perm(cv[2][n / 2], cv[3][n / 2], sel);
        // (What the exponents added comes off step by step: over a long run the sum of the weights, times 136, would
        // leave few bits for what is left. 65536 keys, against fp64: 0.015 with one correction at the end, 0.0022.)
        constexpr uint32_t kMinus128 = 0xc308c308u, kMinus16 = 0xc1c0c1c0u;  // -136, -24
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float(&d)[4] = o[2 * n + e];
          mma_bf16(d[0], d[1], d[2], d[3], kMinus128, kMinus16, kMinus128, kMinus16, pb0, pb1);
          mma_bf16(d[0], d[1], d[2], d[3], code_128(x >> 8 * e), code_16(x >> (8 * e + 1)), code_128(y >> 8 * e),
                   code_16(y >> (8 * e + 1)), pb0, pb1);
        }
      }
    }

    const int unit = now.b * p.heads + now.head;
    if (lane == 0) {  // where the join finds the unit's parts
      if (now.t == first_token(now.end, p.window)) p.warps[unit].x = w;
      if (now.t + kD4Group >= now.end) p.warps[unit].y = w;
    }
    if (then.b != now.b || then.head != now.head) {
      // This warp is done with the unit: its rows and their (maximum, sum) go to the join.
      int g0;
      kv_head(now.head, &g0);
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) {
          l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], d);
#pragma unroll
          for (int n = 0; n < NG; ++n) mids[n][r] += __shfl_xor_sync(0xffffffffu, mids[n][r], d);
        }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (g0 + 2 * c + r < p.G) {
          const int64_t at = (static_cast<int64_t>(w) + unit) * kOwnHeads + 2 * c + r;
          float* dst = p.part_o + at * D + 4 * g;
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            const float z = mids[n][r];
            *reinterpret_cast<float4*>(dst + 32 * n) =
                make_float4(o[2 * n][r] + z, o[2 * n][2 + r] + z, o[2 * n + 1][r] + z, o[2 * n + 1][2 + r] + z);
          }
          if (g == 0) p.part_ml[at] = make_float2(m_run[r], l_run[r]);
        }
      }
      clear();
      if (then.b >= 0) load_q(then);
    }
    __syncwarp();  // every lane is done with this stage before it is refilled
    now = then;
    then = later;
    later = ahead;
    ahead = last;
  }
  cp_async_wait<0>();
}

// How a call is cut, and the room for its parts.
struct Decode4Cut {
  int ctas = 0, heads = 1;
  int64_t units = 0;
  size_t parts = 0;  // rows
  size_t bytes(int D) const { return parts * (D + 2) * sizeof(float) + units * sizeof(int2); }
};

static Decode4Cut cut_decode4(int B, int Hkv, int G, int window, int max_len) {
  static thread_local int cached_dev = -1, cached = 148;
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev != cached_dev) {
    if (cudaDeviceGetAttribute(&cached, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) cached = 148;
    cached_dev = dev;
  }
  Decode4Cut c;
  if (max_len <= 0) return c;
  c.heads = Hkv * ((G + kOwnHeads - 1) / kOwnHeads);
  c.units = static_cast<int64_t>(B) * c.heads;
  const int64_t seen = window > 0 ? std::min<int64_t>(max_len, static_cast<int64_t>(window) + 15) : max_len;
  const int64_t runs = (c.units * ((seen + kD4Group - 1) / kD4Group) + kD4Run - 1) / kD4Run;
  c.ctas = static_cast<int>(std::min<int64_t>(runs, static_cast<int64_t>(kD4Ctas) * cached));
  c.parts = static_cast<size_t>(c.units + c.ctas * kD4Warps) * kOwnHeads;
  return c;
}

template <int D, bool SOFTCAP>
static int launch_decode4(const Decode4Params& p, unsigned grid, cudaStream_t st) {
  constexpr size_t smem = static_cast<size_t>(kD4Warps) * kD4Stages * 2 * kD4Group * Record4<D>::kBytes;
  static thread_local int configured_dev = -1;
  const auto kernel = decode4_kernel<D, SOFTCAP>;
  const int rc = packed_configure(kernel, smem, &configured_dev);
  if (rc != LF_OK) return rc;
  launch_pdl(kernel, dim3(grid), kD4Warps * 32, smem, st, p);
  return check_launch("decode4_kernel");
}

}  // namespace lf

extern "C" {

size_t lf_decode_4bit_workspace_bytes(int32_t B, int32_t Hkv, int32_t G, int32_t D, int32_t window,
                                      int32_t max_seq_len) {
  using namespace lf;
  if (B <= 0 || Hkv <= 0 || G <= 0 || G > kPackedRows || D <= 0 || window < 0 || max_seq_len < 0) return 0;
  return cut_decode4(B, Hkv, G, window, max_seq_len).bytes(D);
}

int lf_decode_4bit(const LfDecode4Args* a, void* stream) {
  using namespace lf;
  if (!a || !a->q || !a->k || !a->v || !a->out || !a->block_table || !a->seq_lens) return LF_ERR_INVALID_ARG;
  if (a->B <= 0 || a->Hkv <= 0 || a->G <= 0 || a->page_size <= 0 || a->n_pages <= 0 || a->bt_blocks <= 0 ||
      a->window < 0 || a->max_seq_len < 0)
    return LF_ERR_INVALID_ARG;
  if (a->D != 64 && a->D != 128) return LF_ERR_UNSUPPORTED;
  if (a->G > kPackedRows) return LF_ERR_UNSUPPORTED;
  if (a->max_seq_len > static_cast<int64_t>(a->bt_blocks) * a->page_size) return LF_ERR_INVALID_ARG;
  if (a->max_seq_len > kMostKeys) return LF_ERR_TOO_LARGE;
  PackedScore score;
  const int rc = packed_score(a->scale, a->n_mod, a->mod_op, a->mod_arg, &score);
  if (rc != LF_OK) return rc;
  const int head_groups = (a->G + kOwnHeads - 1) / kOwnHeads;
  if (a->B > 65535 || static_cast<int64_t>(a->B) * a->Hkv * head_groups > (1 << 26)) return LF_ERR_TOO_LARGE;
  if (!packed_aligned(a->q) || !packed_aligned(a->out) || !record4_aligned(a->k, a->k_stride, a->D) ||
      !record4_aligned(a->v, a->v_stride, a->D))
    return LF_ERR_ALIGNMENT;
  for (int i = 0; i < 3; ++i)
    if (a->q_stride[i] % 8 || a->o_stride[i] % 4) return LF_ERR_ALIGNMENT;
  const Decode4Cut cut = cut_decode4(a->B, a->Hkv, a->G, a->window, a->max_seq_len);
  const size_t need = cut.bytes(a->D);
  if (need && (!a->workspace || a->workspace_bytes < need)) return LF_ERR_WORKSPACE;
  if (!packed_aligned(a->workspace)) return LF_ERR_ALIGNMENT;

  Decode4Params p = {};
  JoinParams pj = {};
  p.part_o = static_cast<float*>(a->workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + cut.parts * a->D);
  p.warps = reinterpret_cast<int2*>(p.part_ml + cut.parts);
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.k = static_cast<const char*>(a->k);
  p.v = static_cast<const char*>(a->v);
  for (int i = 0; i < 3; ++i) {
    p.q_stride[i] = a->q_stride[i];
    p.k_stride[i] = a->k_stride[i];
    p.v_stride[i] = a->v_stride[i];
    pj.o_stride[i] = a->o_stride[i];
  }
  p.table = a->block_table;
  p.bt_stride = a->bt_stride;
  p.seq_lens = pj.seq_lens = a->seq_lens;
  p.B = a->B;
  p.G = pj.G = a->G;
  p.heads = a->Hkv * head_groups;
  p.div_groups = FastDiv::make(head_groups);
  p.window = a->window;
  p.max_len = pj.max_len = a->max_seq_len;
  p.bt_blocks = a->bt_blocks;
  p.page_size = a->page_size;
  p.page_shift = cache_page_shift(a->page_size);
  p.n_pages = a->n_pages;
  p.a = score.a;
  p.c2 = score.c2;
  p.status = pj.status = a->status;
  pj.own_o = p.part_o;
  pj.own_ml = p.part_ml;
  pj.warps = p.warps;
  pj.Hkv = a->Hkv;
  pj.groups = head_groups;
  pj.out = static_cast<__nv_bfloat16*>(a->out);
  pj.rows = static_cast<int64_t>(a->B) * a->Hkv * a->G;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto with_d = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (cut.ctas > 0) {
      const int r = (score.softcap ? launch_decode4<D, true> : launch_decode4<D, false>)(
          p, static_cast<unsigned>(cut.ctas), st);
      if (r != LF_OK) return r;
    }
    launch_pdl(join_kernel<D>, dim3(static_cast<unsigned>((pj.rows + 3) / 4)), 128, 0, st, pj);
    return check_launch("join_kernel");
  };
  return a->D == 128 ? with_d(std::integral_constant<int, 128>{}) : with_d(std::integral_constant<int, 64>{});
}

}  // extern "C"

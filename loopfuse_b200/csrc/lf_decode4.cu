// Decode attention over a 4-bit paged cache: one query token per request, requests of any lengths.
//
// With codes c, scales s and midpoints z of the groups g of 32 columns (include/lf_sm100.h has the format),
//   score_j = sum_g sK_jg (q_g . (cK_jg - 8)) + sum_g zK_jg sum(q_g)
//   o       = sum_g sum_j (p_j sV_jg) cV_jg + sum_g sum_j p_j (zV_jg - 8 sV_jg),    p_j = 2^(score_j - m),
// so a cache row is never unpacked to its values. A code in bits 0..3 (4..7) of an fp16 whose other bits are zero is
// the subnormal number c 2^-24 (16 c 2^-24), which a matrix instruction multiplies exactly: one AND makes two operands
// of codes, and the products, in fp32, are ordinary numbers again. Query rows, times a power of two that brings them
// into fp16's range, are exact as well. Scales are applied to the scores of a group and to the weights.
//
// Bound by HBM, 5/8 byte per value, if the instructions keep up: an SM has to take some 40 values a clock. They do not
// quite, though no pipe is full (issue slots 57 %, integer 49 %, tensor 21 %): the chains of dependent instructions in
// 2.7 warps a scheduler, at 168 registers, leave slots empty. 16 requests of up to 65536 keys, 32 heads on 8, D = 128:
// 149 to 165 us from box to box, 4.4 to 4.9 TB/s (bytes once at HBM's rate 112); 64 of up to 4096 38 to 42 (19).
// Built before: codes with an exponent set above them, 128 + c and 16 + c three bits up, 187 us where this took 149 (7
// operations for 8 codes where this takes 5, and offsets that cost long sums their last bits: an error of 0.015); codes
// as subnormal bf16, as fast, with an error of 0.0024 from the weights' rounding where this has 0.0017; c - 8 by a
// product of the weights with a constant in each step, 155.
#include "lf_cache4.cuh"
#include "lf_packed.cuh"

#include <float.h>

#include <algorithm>
#include <type_traits>

namespace lf {

constexpr int kD4Warps = 4, kD4DirectWarps = 8;  // of a CTA
constexpr int d4_warps(bool direct) { return direct ? kD4DirectWarps : kD4Warps; }
constexpr int kD4DirectGroups = 2 * kD4DirectWarps;  // of the longest unit, for DIRECT
constexpr int kD4Stages = 2;  // groups of a warp's ring: one is copied while one is computed
constexpr int kD4Group = 32;  // tokens that a warp takes at a time
constexpr int kD4Run = 1;     // groups of a warp, at least
constexpr int kD4Heads = 8;   // query heads that a warp computes together: the columns of a matrix instruction
constexpr int kD4Scan = 128;  // up to so many requests, the join adds their lengths up itself
// CTAs of an SM: as many as fit without spilled registers (D = 128, 16 requests of up to 65536 keys: four 157 us, three
// 149; D = 64, 32 of 8192: three 63, four 52), but for a softcap over pages of any kind at D = 128, which spills a word.
constexpr int d4_ctas(int D) { return D == 128 ? 3 : 4; }

struct Decode4Params {
  const __nv_bfloat16* q;
  const char* k;
  const char* v;
  int64_t q_stride[3], k_stride[3], v_stride[3];  // (b, kv head, g); bytes of (page, slot, kv head)
  int32_t even_stride[4];  // EVEN: page and kv head of keys, then of values
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
  uint32_t n_warps;
  __nv_bfloat16* out;
  int64_t o_stride[3];
  int32_t* status;

  // Keys of a request that count: never more than the caller said.
  __device__ __forceinline__ int length(int b) const { return min(max(seq_lens[b], 0), max_len); }
  // Of those, the first that the groups begin with: that of the sixteen which the window's first lies in (pages of
  // 16, 32, ... then hold whole halves of a group).
  __device__ __forceinline__ int first_token(int end) const {
    return window > 0 && end > window ? (end - window) & ~15 : 0;
  }
  __device__ __forceinline__ int groups_of(int end) const {
    return end > 0 ? (end - first_token(end) + kD4Group - 1) / kD4Group : 0;
  }
  // Groups of a warp, when all units have `all` (the host sees to it that they are fewer than 2^31).
  __device__ __forceinline__ uint32_t run(uint32_t all) const {
    return max((all + n_warps - 1) / n_warps, static_cast<uint32_t>(kD4Run));
  }
};

struct Acc {
  float x[4];
};
// Products of bf16 and of fp16.
__device__ __forceinline__ Acc mma_bf16(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                        const Acc& c) {
  Acc d;
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d.x[0]), "=f"(d.x[1]), "=f"(d.x[2]), "=f"(d.x[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c.x[0]), "f"(c.x[1]), "f"(c.x[2]), "f"(c.x[3]));
  return d;
}

__device__ __forceinline__ Acc mma_f16(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                       const Acc& c) {
  Acc d;
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d.x[0]), "=f"(d.x[1]), "=f"(d.x[2]), "=f"(d.x[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c.x[0]), "f"(c.x[1]), "f"(c.x[2]), "f"(c.x[3]));
  return d;
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// 2^(field - 127), field in 1..254; 1 / x for such an x.
__device__ __forceinline__ float power(int field) { return __int_as_float(field << 23); }
__device__ __forceinline__ float over(float x) { return __int_as_float(0x7f000000 - __float_as_int(x)); }

// Transpose of an 8 x 8 matrix of 16-bit values held by a warp, two neighbours of a row per lane.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The codes of both halves of a word as fp16: nibbles 0 and 4 in units of 2^-24, 1 and 5 in units of 2^-20.
__device__ __forceinline__ uint32_t codes_even(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t codes_odd(uint32_t w) { return w & 0x00f000f0u; }
// Weights are at most 2^4 (the reference of a row moves when a score rises further above it), a scale times its column
// group's factor at most 2^11, so that their product is an fp16: with all its 11 bits down to 2^-22 of the group's largest
// scale, and half a step, 2^-33 of that scale, off below. (The factor follows the largest scale alone: with the weights in
// it, every rise of a score would move it.)
constexpr float kRise = 4.f;
constexpr int kFactor = 11;
constexpr int kLargestFactorLog2 = 125;  // of a column group
constexpr int kLargestSumLog2 = 100;     // of what becomes a column's sum at a time
constexpr float kLargestSum = 0x1p100f;
constexpr int kMeet = 16;  // groups after which the sums of codes and bottoms meet (8 and 64: within 1 %)

template <int BYTES>
__device__ __forceinline__ void cp_async_piece(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    cp_async_16(dst, src);
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

template <int N>
__device__ __forceinline__ void lds_words(const unsigned char* p, uint32_t (&x)[N]) {
  if constexpr (N == 4) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    x[0] = r.x, x[1] = r.y, x[2] = r.z, x[3] = r.w;
  } else if constexpr (N == 2) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    x[0] = r.x, x[1] = r.y;
  } else {
    x[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// A place in the row of all units' groups: a group of 32 tokens of a unit.
struct D4Walk {
  int b, head;  // request; kv head and group of query heads
  int t, end;   // first token of the group, end of the unit

  // The unit behind this one; there has to be one.
  __device__ __forceinline__ void next_unit(const Decode4Params& p, int lane) {
    t = p.first_token(end);
    if (++head < p.heads) return;
    head = 0;
    for (++b;; b += 32) {  // the next request that has keys
      const int n = b + lane < p.B ? p.length(b + lane) : 0;
      const unsigned some = __ballot_sync(0xffffffffu, n > 0);
      if (some) {
        const int l = __ffs(some) - 1;
        b += l;
        end = __shfl_sync(0xffffffffu, n, l);
        t = p.first_token(end);
        return;
      }
      if (b + 32 >= p.B) {  // (lengths that change under the call end here)
        b = p.B - 1;
        return;
      }
    }
  }
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
//           fp16, get from the first product's layout to the second's by two 8 x 8 transposes.
//
// DIRECT: a CTA has one unit, its warps equal runs of that, and joins them itself: one launch where the units are few
// and short.
// EVEN: pages of a power of two of slots, 16 or more, whose rows lie next to each other: half a group is then one run
// of bytes, and its place takes few operations (a lane's own row for each piece took 60 of a group's 820).
template <int D, bool SOFTCAP, bool EVEN, bool DIRECT>
__global__ void __launch_bounds__(d4_warps(DIRECT) * 32, DIRECT ? 1 : d4_ctas(D))
    decode4_kernel(const Decode4Params p) {
  constexpr int WARPS = DIRECT ? kD4DirectWarps : kD4Warps;
  using R = Record4<D>;
  constexpr int NG = R::kGroups;
  constexpr int kHalf = kD4Group * R::kBytes;  // keys, then values
  constexpr int kStageBytes = 2 * kHalf;
  constexpr int kPieces = R::kBytes / R::kAlign;  // of a record: 5
  static_assert(kPieces * kD4Group % 32 == 0, "a group's pieces are dealt out evenly");
  extern __shared__ __align__(1024) unsigned char smem[];
  pdl_wait();
  pdl_trigger();  // (behind the wait: the join reads lengths before its own)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  // (Runs go round the CTAs first, then their warps: few of them are spread over all SMs.)
  const uint32_t w = warp * gridDim.x + blockIdx.x;

  D4Walk at;  // what is computed
  int left;   // groups of this warp
  if constexpr (DIRECT) {
    at.b = blockIdx.x / p.heads;
    at.head = blockIdx.x - at.b * p.heads;
    at.end = p.length(at.b);
    const int all = p.groups_of(at.end), run = (all + WARPS - 1) / WARPS;
    at.t = p.first_token(at.end) + warp * run * kD4Group;
    left = max(min(all - warp * run, run), 0);
    if (p.status && at.head == 0 && threadIdx.x == 0) {
      const int len = p.seq_lens[at.b];
      if (len < 0 || len > p.max_len) atomicCAS(p.status, 0, LF_DEV_BAD_LENGTHS);
    }
  } else {
    // Groups of the requests [b, b + 32), one per lane.
    auto groups_at = [&](int b) { return b + lane < p.B ? static_cast<uint32_t>(p.groups_of(p.length(b + lane))) : 0u; };
    uint32_t all = 0, groups = 0;
#pragma unroll 4
    for (int b = 0; b < p.B; b += 32) {
      groups = groups_at(b);
      all += groups;
    }
    all = __reduce_add_sync(0xffffffffu, all) * p.heads;
    const uint32_t run = p.run(all);
    if (all <= w * run) return;  // (run times the warps is below 2^31 and 2^31 more)
    left = static_cast<int>(min(all - w * run, run));
    {
      uint32_t skip = w * run;  // of the requests ahead, then of the units ahead
      uint32_t incl = 0;
      unsigned past = 0;
      int from = 0;
      for (int b = 0; b < p.B && !past; b += 32) {
        if (b) skip -= __shfl_sync(0xffffffffu, incl, 31);
        if (p.B > 32) groups = groups_at(b);
        from = b;
        incl = groups * p.heads;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const uint32_t x = __shfl_up_sync(0xffffffffu, incl, d);
          if (lane >= d) incl += x;
        }
        past = __ballot_sync(0xffffffffu, incl > skip);
      }
      const int l = __ffs(past) - 1;
      const uint32_t n = __shfl_sync(0xffffffffu, groups, l);
      const uint32_t into = skip - __shfl_sync(0xffffffffu, incl, l) + n * p.heads;
      at.b = from + l;
      at.head = static_cast<int>(into / n);
      at.end = p.length(at.b);
      at.t = p.first_token(at.end) + static_cast<int>(into - at.head * n) * kD4Group;
    }
  }
  auto kv_head = [&](int head, int* g0) {
    const int kvh = static_cast<int>(p.div_groups.div(head));
    *g0 = (head - kvh * static_cast<int>(p.div_groups.d)) * kD4Heads;
    return kvh;
  };

  // Where a group lies. EVEN: the pages of its halves and the first row of each (of a half past the end, rows that are
  // there). Else this lane's row: rows past the end repeat the last, rows in front of the window its first.
  struct Place {
    int page[2], slot[2], kvh;
  };
  D4Walk ahead = at;  // what is looked up
  int unseen = left, ignored;
  int kvh_ahead = kv_head(ahead.head, &ignored);
  auto look_up = [&] {
    Place x = {{0, 0}, {0, 0}, kvh_ahead};
    if (unseen <= 0) return x;
    const int32_t* row = p.table + ahead.b * p.bt_stride;
    if constexpr (EVEN) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = min(ahead.t + 16 * h, ahead.end - 1), block = t >> p.page_shift;
        x.slot[h] = (t & (p.page_size - 1)) & ~15;
        if (LF_BOUNDS(ahead.b < p.B && ahead.head < p.heads && t >= 0 && block < p.bt_blocks, p.status, 75))
          x.page[h] = row[block];
      }
    } else {
      const int t = max(min(ahead.t + lane, ahead.end - 1), p.window > 0 ? ahead.end - p.window : 0);
      const int block = p.page_shift >= 0 ? t >> p.page_shift : t / p.page_size;
      x.slot[0] = t - block * p.page_size;
      if (LF_BOUNDS(ahead.b < p.B && ahead.head < p.heads && t >= 0 && block < p.bt_blocks, p.status, 76))
        x.page[0] = row[block];
    }
    --unseen;
    ahead.t += kD4Group;
    if (ahead.t >= ahead.end && unseen > 0) {
      ahead.next_unit(p, lane);
      kvh_ahead = kv_head(ahead.head, &ignored);
    }
    return x;
  };
  unsigned char* ring = smem + warp * (kD4Stages * kStageBytes);
  const uint32_t ring_u32 = smem_u32(ring);
  int uncopied = left;
  auto copy_group = [&](Place x, int stage) {
    if (uncopied > 0) {
      --uncopied;
#pragma unroll
      for (int h = 0; h < (EVEN ? 2 : 1); ++h)
        if (static_cast<uint32_t>(x.page[h]) >= static_cast<uint32_t>(p.n_pages)) {
          if (p.status) atomicExch(p.status, LF_DEV_BAD_PAGE);
          x.page[h] = 0;
        }
      const uint32_t dst = ring_u32 + stage * kStageBytes + lane * R::kAlign;
      if constexpr (EVEN) {
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int64_t of_page = p.even_stride[2 * kv], of_head = p.even_stride[2 * kv + 1];
          const char* base = (kv ? p.v : p.k) + x.kvh * of_head + lane * R::kAlign;
          const char* lo = base + x.page[0] * of_page + x.slot[0] * R::kBytes;
          const char* hi = base + x.page[1] * of_page + (x.slot[1] - 16) * R::kBytes;
          const char* mid = lane < 16 ? lo : hi;  // (a half is 2.5 pieces of each lane)
#pragma unroll
          for (int i = 0; i < 5; ++i)
            cp_async_piece<R::kAlign>(dst + kv * kHalf + 32 * i * R::kAlign,
                                      (i < 2 ? lo : i == 2 ? mid : hi) + 32 * i * R::kAlign);
        }
      } else {
        const int64_t kr = x.kvh * p.k_stride[2] + x.page[0] * p.k_stride[0] + x.slot[0] * p.k_stride[1];
        const int64_t vr = x.kvh * p.v_stride[2] + x.page[0] * p.v_stride[0] + x.slot[0] * p.v_stride[1];
#pragma unroll
        for (int i = 0; i < kPieces * kD4Group / 32; ++i) {
          const int id = lane + 32 * i, row = id / kPieces, from = (id - row * kPieces) * R::kAlign;
          cp_async_piece<R::kAlign>(dst + 32 * i * R::kAlign, p.k + __shfl_sync(0xffffffffu, kr, row) + from);
          cp_async_piece<R::kAlign>(dst + kHalf + 32 * i * R::kAlign, p.v + __shfl_sync(0xffffffffu, vr, row) + from);
        }
      }
    }
    cp_async_commit();
  };

  // The query heads of a unit: columns of the first product, in the order that the codes have (in shared memory:
  // registers are what bounds the warps of an SM); and the sums of the columns, which go with the midpoints (sum_z) and,
  // times -8, with the scales (sum_s), as two or three bf16 each: as many as one more instruction has room for, 2^-17 of
  // a group's share of a score or less. Scores are in units of a power of two, of each row, until they are scaled.
  uint4* qf = reinterpret_cast<uint4*>(smem + WARPS * kD4Stages * kStageBytes) + warp * (32 * NG) + lane;
  uint32_t sum_z, sum_s;
  float row_a[2], row_c2[2];  // query heads 2c, 2c + 1: score = row_c2 x, or row_c2 tanh(row_a x)
  struct Query {
    uint4 x[NG];
  };
  auto load_q = [&] {
    int g0;
    const int kvh = kv_head(at.head, &g0);
    Query r;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      r.x[n] = make_uint4(0u, 0u, 0u, 0u);
      if (g0 + g < p.G)
        r.x[n] = *reinterpret_cast<const uint4*>(p.q + at.b * p.q_stride[0] + kvh * p.q_stride[1] +
                                                 (g0 + g) * p.q_stride[2] + 32 * n + 8 * c);
    }
    return r;
  };
  auto take_q = [&](const Query& raw) {
    // The row times 2^(14 - E), E the exponent of its largest column (0 or not a number: any). Products with even codes are
    // in units of 2^(E - 14 - 24).
    uint32_t top = 0;  // (numbers without their signs compare like whole ones)
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const uint32_t words[4] = {raw.x[n].x, raw.x[n].y, raw.x[n].z, raw.x[n].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __vmaxu2(top, words[e] & 0x7fff7fffu);
    }
#pragma unroll
    for (int d = 1; d <= 2; d <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, d));
    const int field = min(max(static_cast<int>(max(top >> 16, top & 0xffffu) >> 7), 14), 254);  // (`up` is a number)
    const float up = power(268 - field);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      // (In two factors: the unit of a row of columns past 2^117 is no fp32.)
      const int unit = __shfl_sync(0xffffffffu, field, 8 * c + 4 * r) + 10;
      const float of_row = power(min(unit, 254)), rest = power(127 + max(unit - 254, 0));
      // (Neither zero nor infinite: with a masked score, or a score of zero, either would be NaN.)
      row_a[r] = fminf(fmaxf(p.a * of_row * rest, -FLT_MAX), FLT_MAX);
      row_c2[r] = SOFTCAP ? p.c2 : fminf(fmaxf(p.c2 * of_row * rest, FLT_MIN), FLT_MAX);
    }
    float sum[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const uint4 r = raw.x[n];
      // (Exact, but for columns below 2^-24 of the largest; odd codes come times 16.)
      const float x0 = bf16lo_to_f32(r.x) * up, x1 = bf16hi_to_f32(r.x) * up, x2 = bf16lo_to_f32(r.y) * up,
                  x3 = bf16hi_to_f32(r.y) * up, x4 = bf16lo_to_f32(r.z) * up, x5 = bf16hi_to_f32(r.z) * up,
                  x6 = bf16lo_to_f32(r.w) * up, x7 = bf16hi_to_f32(r.w) * up;
      qf[32 * n] = make_uint4(pack_f16x2(x0, x4), pack_f16x2(x1 * 0.0625f, x5 * 0.0625f), pack_f16x2(x2, x6),
                              pack_f16x2(x3 * 0.0625f, x7 * 0.0625f));
      float all_q = ((x0 + x1) + (x2 + x3)) + ((x4 + x5) + (x6 + x7));
#pragma unroll
      for (int d = 1; d <= 2; d <<= 1) all_q += __shfl_xor_sync(0xffffffffu, all_q, d);
      sum[n] = all_q * 0x1p-24f;
    }
    // Inner index 2c, 2c + 1 of the product of both: a pair of column groups, and a part of the sums.
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
    if constexpr (NG == 4)
      sum_z = c == 0 ? part[0][0] : c == 1 ? part[0][1] : c == 2 ? part[1][0] : part[1][1];
    else
      sum_z = c == 0 ? part[0][0] : c == 1 ? part[1][0] : c == 2 ? part[2][0] : 0u;
    sum_s = pack_bf16x2(-8.f * bf16lo_to_f32(sum_z), -8.f * bf16hi_to_f32(sum_z));  // (exact)
  };

  // Query heads 2c, 2c + 1; this lane's keys, until the end of the unit. A pair: keys g, and g + 8, of every sixteen.
  float m_run[2];
  uint64_t l_run[2];
  float bottoms[NG][2];  // weights times what codes of 0 stand for
  // Of a column group of V: 2^11 over a power of two that no scale so far is above; those powers, as bf16.
  float factor[NG];
  uint32_t most[NG / 2];
  Acc o[2 * NG];  // rows of instruction 2n + h: columns 32 n + 4 g + 2 h, then + 1; each for both heads
  auto clear = [&] {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      m_run[r] = -INFINITY;
      l_run[r] = 0;
#pragma unroll
      for (int n = 0; n < NG; ++n) bottoms[n][r] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      factor[n] = 1.f;
      most[n / 2] = 0u;
    }
#pragma unroll
    for (int n = 0; n < 2 * NG; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n].x[e] = 0.f;
  };

  auto over_keys = [](float x) {
#pragma unroll
    for (int d = 4; d <= 16; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
  };
  // The sums of codes, which are all positive, and of the bottoms, about minus that, become one of the size of the result.
  // (Only at the end of a long run, the result would be left with what the roundings of sums many times its size leave.)
  // A sum of bottoms times its group's factor has to stay in fp32: midpoints of 8 over scales of 2^-115 would be infinite
  // with the factor that follows from these alone. A sum that is past the limit lowers the factor to what it bears; the
  // first that is not zero sets one where there was no scale yet, so that what has met is never brought up.
  auto meet = [&] {
    bool past = false;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
#pragma unroll
      for (int r = 0; r < 2; ++r) bottoms[n][r] = over_keys(bottoms[n][r]);
      const float big = fmaxf(fabsf(bottoms[n][0]), fabsf(bottoms[n][1]));
      past = past || big * 0x1p-20f * factor[n] > kLargestSum || (!(most[n / 2] & 0xffffu << (16 * (n & 1))) && big > 0.f);
    }
    if (__any_sync(0xffffffffu, past)) {
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float big = fmaxf(fabsf(bottoms[n][0]), fabsf(bottoms[n][1]));
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
        // (big < 2^(e - 126), e its exponent's field.)
        const int e = __float_as_int(big) >> 23, f = min(kLargestSumLog2 + 20 + 126 - e, kLargestFactorLog2);
        const uint32_t half = 0xffffu << (16 * (n & 1));
        if (most[n / 2] & half ? power(127 + f) < factor[n] : big > 0.f) {
          const float by = power(127 + f) * over(factor[n]);
          factor[n] = power(127 + f);
          most[n / 2] = (most[n / 2] & ~half) | (127u + kFactor - f) << (7 + 16 * (n & 1));
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[2 * n + t].x[i] *= by;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const float even = 0x1p-24f * factor[n], odd = 0x1p-20f * factor[n];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          o[2 * n + t].x[r] = fmaf(bottoms[n][r], even, o[2 * n + t].x[r]);
          o[2 * n + t].x[2 + r] = fmaf(bottoms[n][r], odd, o[2 * n + t].x[2 + r]);
        }
        bottoms[n][r] = 0.f;
      }
    }
  };

  // The products of the group at.t, which lies in `stage`. EDGE: not all of its keys are seen, but [from, at.end).
  int from = 0;
  auto compute = [&](const unsigned char* stage, auto edge) {
    constexpr bool EDGE = decltype(edge)::value;
    auto hidden = [&](int i) { return at.t + i < from || at.t + i >= at.end; };
    float sc[2][4];  // [half of the group]: key g (two heads), key g + 8
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned char* k0 = stage + (16 * h + g) * R::kBytes;
      const unsigned char* k1 = k0 + 8 * R::kBytes;
      uint32_t w0[NG], w1[NG], s0[NG / 2], s1[NG / 2];
      lds_words<NG>(k0 + 4 * NG * c, w0);
      lds_words<NG>(k1 + 4 * NG * c, w1);
      lds_words<NG / 2>(k0 + R::kScales, s0);
      lds_words<NG / 2>(k1 + R::kScales, s1);
      const int pair = NG == 4 ? 4 * (c & 1) : 0;
      auto word = [&](const unsigned char* at) { return *reinterpret_cast<const uint32_t*>(at + pair); };
      constexpr Acc kZero = {{0.f, 0.f, 0.f, 0.f}};
      Acc x = mma_bf16(word(k0 + R::kMids), word(k1 + R::kMids), word(k0 + R::kScales), word(k1 + R::kScales), sum_z,
                       sum_s, kZero);
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const uint32_t u0 = w0[n] >> 8, u1 = w1[n] >> 8;
        const uint4 q = qf[32 * n];
        Acc y = mma_f16(codes_even(w0[n]), codes_even(w1[n]), codes_odd(w0[n]), codes_odd(w1[n]), q.x, q.y, kZero);
        y = mma_f16(codes_even(u0), codes_even(u1), codes_odd(u0), codes_odd(u1), q.z, q.w, y);
        const float a = n & 1 ? bf16hi_to_f32(s0[n / 2]) : bf16lo_to_f32(s0[n / 2]);
        const float b = n & 1 ? bf16hi_to_f32(s1[n / 2]) : bf16lo_to_f32(s1[n / 2]);
        x.x[0] = fmaf(a, y.x[0], x.x[0]);
        x.x[1] = fmaf(a, y.x[1], x.x[1]);
        x.x[2] = fmaf(b, y.x[2], x.x[2]);
        x.x[3] = fmaf(b, y.x[3], x.x[3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float s = x.x[e];
        if constexpr (SOFTCAP) s = tanh_approx(s * row_a[e & 1]);  // (the unit's, within 2^-11, as in decode)
        if (EDGE && hidden(16 * h + g + 8 * (e >> 1))) s = -INFINITY;
        sc[h][e] = s;
      }
    }
    // The reference of a row moves when a score rises more than kRise above it, not with every maximum: the lanes of
    // a row look at each other's scores only then.
    float mx[2];
    mx[0] = fmaxf(max3(sc[0][0], sc[0][2], sc[1][0]), sc[1][2]) * row_c2[0];
    mx[1] = fmaxf(max3(sc[0][1], sc[0][3], sc[1][1]), sc[1][3]) * row_c2[1];
    // Likewise the factor of a column group, when a scale is above all before it.
    uint32_t top[NG / 2];
    bool moves = mx[0] > m_run[0] + kRise || mx[1] > m_run[1] + kRise;
    uint32_t meta[4][NG];  // scales, then midpoints, of keys g + 8 i
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lds_words<NG>(stage + kHalf + (g + 8 * i) * R::kBytes + R::kScales, meta[i]);
      if constexpr (EDGE) {  // (what lies in rows that are not seen may be NaN)
        const bool no = hidden(g + 8 * i);
#pragma unroll
        for (int n = 0; n < NG; ++n) meta[i][n] = no ? 0u : meta[i][n];
      }
#pragma unroll
      for (int n = 0; n < NG / 2; ++n) top[n] = __vmaxu2(i ? top[n] : most[n], meta[i][n]);
    }
#pragma unroll
    for (int n = 0; n < NG / 2; ++n) moves = moves || top[n] != most[n];
    if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
      for (int n = 0; n < NG / 2; ++n) {
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) top[n] = __vmaxu2(top[n], __shfl_xor_sync(0xffffffffu, top[n], d));
        if (top[n] == most[n]) continue;
        uint32_t now = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t of = (top[n] >> (16 * i)) & 0xffffu, before = (most[n] >> (16 * i)) & 0xffffu;
          // (Up to four times as large, none moves it again. From 2^-114 to 2^127; scales below lose bits.)
          const uint32_t wanted = min(max(((of & 0x7fffu) >> 7) + 3u, 127u + kFactor - kLargestFactorLog2), 254u);
          const uint32_t field = of > before ? max(wanted, before >> 7) : before >> 7;
          now |= (field << 7) << (16 * i);
          if (of > before) {
            const float f = power(254 + kFactor - static_cast<int>(field)), by = f * over(factor[2 * n + i]);
            factor[2 * n + i] = f;
            // (With the first scale above zero too, where o is zero or holds sums that met before it.)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[4 * n + 2 * i + t].x[e] *= by;
          }
        }
        most[n] = now;
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], d));
        mx[r] = fmaxf(mx[r], m_run[r]);
        const float alpha = mx[r] == -INFINITY ? 0.f : ex2_approx(m_run[r] - mx[r]);
        m_run[r] = mx[r];
        const uint64_t alpha2 = pack2(alpha, alpha);
        l_run[r] = mul2(l_run[r], alpha2);
#pragma unroll
        for (int n = 0; n < NG; ++n) bottoms[n][r] *= alpha;
#pragma unroll
        for (int n = 0; n < 2 * NG; ++n) {
          o[n].x[r] *= alpha;
          o[n].x[2 + r] *= alpha;
        }
      }
    }
    uint64_t up[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float x = m_run[r] == -INFINITY ? 0.f : -m_run[r];
      up[r] = pack2(x, x);
    }

#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint64_t pr[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x, y;
        unpack2(fma2(pack2(sc[h][r], sc[h][2 + r]), pack2(row_c2[r], row_c2[r]), up[r]), x, y);
        pr[r] = pack2(ex2_approx(x), ex2_approx(y));
        l_run[r] = add2(l_run[r], pr[r]);  // this lane's share; the keys are summed at the end of the unit
      }
      const unsigned char* v = stage + kHalf + 16 * h * R::kBytes;
      const uint32_t(&s0)[NG] = meta[2 * h];
      const uint32_t(&s1)[NG] = meta[2 * h + 1];
      // Codes of keys 2c, 2c + 1, 2c + 8, 2c + 9: [key][pair of column groups].
      uint32_t cv[4][NG / 2];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        lds_words<NG / 2>(v + (2 * c + (r & 1) + 8 * (r >> 1)) * R::kBytes + g * R::kValuePiece, cv[r]);
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const float a = n & 1 ? bf16hi_to_f32(s0[n / 2]) : bf16lo_to_f32(s0[n / 2]);
        const float b = n & 1 ? bf16hi_to_f32(s1[n / 2]) : bf16lo_to_f32(s1[n / 2]);
        const float za = n & 1 ? bf16hi_to_f32(s0[NG / 2 + n / 2]) : bf16lo_to_f32(s0[NG / 2 + n / 2]);
        const float zb = n & 1 ? bf16hi_to_f32(s1[NG / 2 + n / 2]) : bf16lo_to_f32(s1[NG / 2 + n / 2]);
        float x0, y0, x1, y1, bottom_a, bottom_b;  // (bottom: what a code of 0 stands for)
        unpack2(fma2(pack2(a, b), pack2(-8.f, -8.f), pack2(za, zb)), bottom_a, bottom_b);
        const uint64_t scaled = mul2(pack2(a, b), pack2(factor[n], factor[n]));
        unpack2(mul2(pr[0], scaled), x0, y0);
        unpack2(mul2(pr[1], scaled), x1, y1);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float pa, pb;
          unpack2(pr[r], pa, pb);
          bottoms[n][r] = fmaf(pa, bottom_a, fmaf(pb, bottom_b, bottoms[n][r]));
        }
        const uint32_t pb0 = transpose_8x8(pack_f16x2(x0, x1));
        const uint32_t pb1 = transpose_8x8(pack_f16x2(y0, y1));
        const uint32_t sel = n & 1 ? 0x7632u : 0x5410u;
        const uint32_t x = __byte_perm(cv[0][n / 2], cv[1][n / 2], sel);
        const uint32_t y = __byte_perm(cv[2][n / 2], cv[3][n / 2], sel);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t ux = e ? x >> 8 : x, uy = e ? y >> 8 : y;
          Acc& d = o[2 * n + e];
          d = mma_f16(codes_even(ux), codes_odd(ux), codes_even(uy), codes_odd(uy), pb0, pb1, d);
        }
      }
    }
  };

  // A group is looked up while the one before it is copied, and that while the one before that is computed.
  if constexpr (DIRECT) clear();  // (for a warp without a group)
  Query query = load_q();
  copy_group(look_up(), 0);
  Place next = look_up();
  int it = 0;
  while (left > 0) {
    // A unit, or the part of one that is this warp's.
    take_q(query);
    clear();
    const int unit = at.b * p.heads + at.head, first = p.first_token(at.end);
    if (!DIRECT && lane == 0 && at.t == first) p.warps[unit].x = static_cast<int>(w);  // where the join finds its parts
    from = p.window > 0 ? at.end - p.window : 0;
    int here = min(left, (at.end - at.t + kD4Group - 1) / kD4Group);
    left -= here;
    for (; here > 0; --here, at.t += kD4Group) {
      copy_group(next, it ^ 1);
      next = look_up();
      cp_async_wait<1>();
      __syncwarp();
      const unsigned char* stage = ring + it * kStageBytes;
      if (at.t < from || at.t + kD4Group > at.end)
        compute(stage, std::true_type{});
      else
        compute(stage, std::false_type{});
      __syncwarp();  // every lane is done with this stage before it is refilled
      it ^= 1;
      if (here % kMeet == 1) meet();
    }

    // This warp is done with the unit: its rows and their (maximum, sum) go to the join.
    int g0;
    kv_head(at.head, &g0);
    [[maybe_unused]] const bool done = at.t >= at.end;
    if (left > 0) {  // (the next one's queries come in under what is left to do: 64 requests of 1500 keys 39 -> 36 us)
      at.next_unit(p, lane);
      query = load_q();
    }
    if constexpr (DIRECT) break;  // (a warp has one unit; its sums go to the others below)
    if (lane == 0 && done) p.warps[unit].y = static_cast<int>(w);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float la, lb;
      unpack2(l_run[r], la, lb);
      const float l = over_keys(la + lb);
      if (g0 + 2 * c + r < p.G) {
        const int64_t place = (static_cast<int64_t>(w) + unit) * kD4Heads + 2 * c + r;
        float* dst = p.part_o + place * D + 4 * g;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const float back = over(factor[n]), even = 0x1p24f * back, odd = 0x1p20f * back;
          *reinterpret_cast<float4*>(dst + 32 * n) =
              make_float4(o[2 * n].x[r] * even, o[2 * n].x[2 + r] * odd, o[2 * n + 1].x[r] * even, o[2 * n + 1].x[2 + r] * odd);
        }
        if (g == 0) p.part_ml[place] = make_float2(m_run[r], l);
      }
    }
  }
  cp_async_wait<0>();
  if constexpr (DIRECT) {
    constexpr int kPart = D + 2;
    float* s_part = reinterpret_cast<float*>(smem);  // [warp][query head][D, maximum, sum], where the rings were
    static_assert(WARPS * kD4Heads * kPart * 4 <= WARPS * kD4Stages * kStageBytes, "the parts lie in the rings");
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float la, lb;
      unpack2(l_run[r], la, lb);
      const float l = over_keys(la + lb);
      float* dst = s_part + (warp * kD4Heads + 2 * c + r) * kPart;
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const float back = over(factor[n]), even = 0x1p24f * back, odd = 0x1p20f * back;
        dst[32 * n + 4 * g] = o[2 * n].x[r] * even;
        dst[32 * n + 4 * g + 1] = o[2 * n].x[2 + r] * odd;
        dst[32 * n + 4 * g + 2] = o[2 * n + 1].x[r] * even;
        dst[32 * n + 4 * g + 3] = o[2 * n + 1].x[2 + r] * odd;
      }
      if (g == 0) {
        dst[D] = m_run[r];
        dst[D + 1] = l;
      }
    }
    __syncthreads();
    int g0;
    const int kvh = kv_head(blockIdx.x - at.b * p.heads, &g0);
    for (int i = threadIdx.x; i < kD4Heads * D; i += WARPS * 32) {
      const int head = i / D, col = i - head * D;
      if (g0 + head >= p.G) break;
      const float* src = s_part + head * kPart;
      float m = -INFINITY;
#pragma unroll
      for (int x = 0; x < WARPS; ++x) m = fmaxf(m, src[x * kD4Heads * kPart + D]);
      const float m_safe = m == -INFINITY ? 0.f : m;
      float l = 0.f, y = 0.f;
#pragma unroll
      for (int x = 0; x < WARPS; ++x) {
        const float wt = ex2_approx(src[x * kD4Heads * kPart + D] - m_safe);
        l = fmaf(src[x * kD4Heads * kPart + D + 1], wt, l);
        y = fmaf(src[x * kD4Heads * kPart + col], wt, y);
      }
      p.out[at.b * p.o_stride[0] + kvh * p.o_stride[1] + (g0 + head) * p.o_stride[2] + col] =
          __float2bfloat16_rn(l == 0.f ? 0.f : y / l);
    }
  }
}

// out = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m) over the parts of a row's unit, which WARPS warps share. Bound by the
// latency of its loads: which parts there are follows from the lengths, which it adds up while the products still run
// (they are read in front of pdl_wait: the products' kernel waits for what is before it ahead of letting this one start),
// so that behind them there is one round trip to memory.
template <int D, int WARPS>
__global__ void __launch_bounds__(128) decode4_join_kernel(const Decode4Params p) {
  constexpr int EPL = D / 32;
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % WARPS;
  const uint32_t row = blockIdx.x * (4 / WARPS) + (threadIdx.x >> 5) / WARPS;
  const uint32_t kv_heads = p.heads / p.div_groups.d;
  const uint32_t bh = row / p.G, head = row - bh * p.G;
  const uint32_t b = bh / kv_heads, kvh = bh - b * kv_heads;
  const bool here = b < static_cast<uint32_t>(p.B);
  const uint32_t of_b = kvh * p.div_groups.d + head / kD4Heads;  // units of the request ahead of the row's
  const int64_t unit = static_cast<int64_t>(b) * p.heads + of_b;
  const uint32_t groups = here ? p.groups_of(p.length(b)) : 0;
  uint32_t first = 0, n = 0;
  if (p.B <= kD4Scan) {
    uint32_t all = 0, before = 0;
#pragma unroll
    for (int i = 0; i < kD4Scan; i += 32) {
      const uint32_t x = i + lane < p.B ? p.groups_of(p.length(i + lane)) : 0;
      all += x;
      before += i + lane < static_cast<int>(b) ? x : 0;
    }
    const uint32_t run = p.run(__reduce_add_sync(0xffffffffu, all) * p.heads);
    const uint32_t from = __reduce_add_sync(0xffffffffu, before) * p.heads + of_b * groups;
    first = from / run;
    n = groups > 0 ? (from + groups - 1) / run - first + 1 : 0;
  }
  pdl_wait();
  if (p.status && here && kvh == 0 && head == 0 && warp == 0 && lane == 0) {  // (what is cut is reported once)
    const int len = p.seq_lens[b];
    if (len < 0 || len > p.max_len) atomicCAS(p.status, 0, LF_DEV_BAD_LENGTHS);
  }
  if (p.B > kD4Scan && groups > 0) {
    const int2 w = p.warps[unit];
    first = w.x;
    n = w.y - w.x + 1;
  }
  if (!LF_BOUNDS(n == 0 || first + n <= p.n_warps, p.status, 77)) n = 0;
  const int64_t at = (first + unit) * kD4Heads + head % kD4Heads;  // its parts: kD4Heads rows apart
  float m_all = -INFINITY, l_all = 0.f, o[EPL] = {};
  for (uint32_t s0 = warp; s0 < n; s0 += 8 * WARPS) {  // eight parts of this warp
    float x[8][EPL];
    float2 ml = make_float2(-INFINITY, 0.f);
    if (s0 + WARPS * (lane & 7) < n) ml = p.part_ml[at + static_cast<int64_t>(s0 + WARPS * (lane & 7)) * kD4Heads];
#pragma unroll
    for (uint32_t u = 0; u < 8; ++u) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) x[u][e] = 0.f;
      if (s0 + WARPS * u < n) {
        const float* src = p.part_o + (at + static_cast<int64_t>(s0 + WARPS * u) * kD4Heads) * D + lane * EPL;
        if constexpr (EPL == 4) {
          const float4 v = *reinterpret_cast<const float4*>(src);
          x[u][0] = v.x, x[u][1] = v.y, x[u][2] = v.z, x[u][3] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(src);
          x[u][0] = v.x, x[u][1] = v.y;
        }
      }
    }
    float m_new = fmaxf(ml.x, m_all);
#pragma unroll
    for (int d = 4; d >= 1; d >>= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, d));
    const float m_safe = m_new == -INFINITY ? 0.f : m_new;
    const float back = ex2_approx(m_all - m_safe), wt = ex2_approx(ml.x - m_safe);
    float l = ml.y * wt;
#pragma unroll
    for (int d = 4; d >= 1; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    l_all = fmaf(l_all, back, l);
    m_all = m_new;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] *= back;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float wu = __shfl_sync(0xffffffffu, wt, u);
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[e] = fmaf(x[u][e], wu, o[e]);
    }
  }
  if constexpr (WARPS > 1) {  // (the whole CTA has one row)
    __shared__ float s_o[WARPS][D];
    __shared__ float2 s_ml[WARPS];
#pragma unroll
    for (int e = 0; e < EPL; ++e) s_o[warp][lane * EPL + e] = o[e];
    if (lane == 0) s_ml[warp] = make_float2(m_all, l_all);
    __syncthreads();
    if (warp > 0) return;
    m_all = -INFINITY;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) m_all = fmaxf(m_all, s_ml[i].x);
    const float m_safe = m_all == -INFINITY ? 0.f : m_all;
    l_all = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      const float wt = ex2_approx(s_ml[i].x - m_safe);
      l_all = fmaf(s_ml[i].y, wt, l_all);
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[e] = fmaf(s_o[i][lane * EPL + e], wt, o[e]);
    }
  }
  if (!here) return;
  const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
  __nv_bfloat16* dst = p.out + b * p.o_stride[0] + kvh * p.o_stride[1] + head * p.o_stride[2] + lane * EPL;
  if constexpr (EPL == 4)
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(o[0] * inv, o[1] * inv);
}

// How a call is cut, and the room for its parts.
struct Decode4Cut {
  bool direct = false;
  int ctas = 0, heads = 1;
  int64_t units = 0;
  size_t parts = 0;  // rows
  size_t bytes(int D) const { return parts * (D + 2) * sizeof(float) + units * sizeof(int2); }
};

// Groups of the longest unit.
static int64_t most_groups(int window, int max_len) {
  const int64_t seen = window > 0 ? std::min<int64_t>(max_len, static_cast<int64_t>(window) + 15) : max_len;
  return (seen + kD4Group - 1) / kD4Group;
}

static Decode4Cut cut_decode4(int B, int Hkv, int G, int D, int window, int max_len) {
  static thread_local int cached_dev = -1, cached = 148;
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev != cached_dev) {
    if (cudaDeviceGetAttribute(&cached, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) cached = 148;
    cached_dev = dev;
  }
  Decode4Cut c;
  if (max_len <= 0) return c;
  c.heads = Hkv * ((G + kD4Heads - 1) / kD4Heads);
  c.units = static_cast<int64_t>(B) * c.heads;
  // One launch, a CTA of eight warps a unit, where units have an SM each and are short (8 kv heads, D = 128): 4 requests
  // of 100 keys 4.6 us a call instead of 7.8, 4 of 500 6.6 instead of 7.8, 16 of 500 6.7 instead of 10.0, but 4 of 1000
  // 9.4 instead of 8.5. With twelve warps 5.1, 7.0 and 7.0.
  if (c.units <= cached && most_groups(window, max_len) <= kD4DirectGroups) {
    c.direct = true;
    c.ctas = static_cast<int>(c.units);
    c.units = 0;
    return c;
  }
  const int64_t runs = (c.units * most_groups(window, max_len) + kD4Run - 1) / kD4Run;
  c.ctas = static_cast<int>(std::min<int64_t>(runs, static_cast<int64_t>(d4_ctas(D)) * cached));
  c.parts = static_cast<size_t>(c.units + c.ctas * kD4Warps) * kD4Heads;
  return c;
}

template <int D, bool SOFTCAP, bool EVEN, bool DIRECT>
static int launch_decode4(const Decode4Params& p, unsigned grid, cudaStream_t st) {
  constexpr size_t smem = static_cast<size_t>(d4_warps(DIRECT)) * (kD4Stages * 2 * kD4Group * Record4<D>::kBytes + 16 * D);
  static thread_local int configured_dev = -1;
  const auto kernel = decode4_kernel<D, SOFTCAP, EVEN, DIRECT>;
  const int rc = packed_configure(kernel, smem, &configured_dev);
  if (rc != LF_OK) return rc;
  launch_pdl(kernel, dim3(grid), d4_warps(DIRECT) * 32, smem, st, p);
  return check_launch("decode4_kernel");
}

}  // namespace lf

extern "C" {

size_t lf_decode_4bit_workspace_bytes(int32_t B, int32_t Hkv, int32_t G, int32_t D, int32_t window,
                                      int32_t max_seq_len) {
  using namespace lf;
  if (B <= 0 || Hkv <= 0 || G <= 0 || G > kPackedRows || D <= 0 || window < 0 || max_seq_len < 0) return 0;
  return cut_decode4(B, Hkv, G, D, window, max_seq_len).bytes(D);
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
  const int head_groups = (a->G + kD4Heads - 1) / kD4Heads;
  const int64_t units = static_cast<int64_t>(a->B) * a->Hkv * head_groups;
  if (a->B > 65535 || units > (1 << 26) || units * most_groups(a->window, a->max_seq_len) > 0x7fffffff)
    return LF_ERR_TOO_LARGE;
  if (!aligned_16(a->q) || !aligned_16(a->out) || !record4_aligned(a->k, a->k_stride, a->D) ||
      !record4_aligned(a->v, a->v_stride, a->D))
    return LF_ERR_ALIGNMENT;
  for (int i = 0; i < 3; ++i)
    if (a->q_stride[i] % 8 || a->o_stride[i] % 4) return LF_ERR_ALIGNMENT;
  const Decode4Cut cut = cut_decode4(a->B, a->Hkv, a->G, a->D, a->window, a->max_seq_len);
  const size_t need = cut.bytes(a->D);
  if (need && (!a->workspace || a->workspace_bytes < need)) return LF_ERR_WORKSPACE;
  if (!aligned_16(a->workspace)) return LF_ERR_ALIGNMENT;

  Decode4Params p = {};
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
    p.o_stride[i] = a->o_stride[i];
  }
  p.table = a->block_table;
  p.bt_stride = a->bt_stride;
  p.seq_lens = a->seq_lens;
  p.B = a->B;
  p.G = a->G;
  p.heads = a->Hkv * head_groups;
  p.div_groups = FastDiv::make(head_groups);
  p.window = a->window;
  p.max_len = a->max_seq_len;
  p.bt_blocks = a->bt_blocks;
  p.page_size = a->page_size;
  p.page_shift = shift_of(a->page_size);
  p.n_pages = a->n_pages;
  p.a = score.a;
  p.c2 = score.c2;
  p.status = a->status;
  p.n_warps = std::max(cut.ctas, 1) * kD4Warps;
  p.out = static_cast<__nv_bfloat16*>(a->out);
  const int64_t rows = static_cast<int64_t>(a->B) * a->Hkv * a->G;
  bool even = p.page_shift >= 4 && a->k_stride[1] == LF_RECORD4_BYTES(a->D) && a->v_stride[1] == LF_RECORD4_BYTES(a->D);
  const int64_t strides[4] = {a->k_stride[0], a->k_stride[2], a->v_stride[0], a->v_stride[2]};
  for (int i = 0; i < 4; ++i) {
    even = even && strides[i] >= 0 && strides[i] <= 0x7fffffff;
    p.even_stride[i] = static_cast<int32_t>(strides[i]);
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto with_d = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (cut.ctas > 0) {
      auto pick = [&](auto direct) {
        constexpr bool DIRECT = decltype(direct)::value;
        return score.softcap ? (even ? launch_decode4<D, true, true, DIRECT> : launch_decode4<D, true, false, DIRECT>)
                             : (even ? launch_decode4<D, false, true, DIRECT> : launch_decode4<D, false, false, DIRECT>);
      };
      const auto run = cut.direct ? pick(std::true_type{}) : pick(std::false_type{});
      const int r = run(p, static_cast<unsigned>(cut.ctas), st);
      if (r != LF_OK || cut.direct) return r;
    }
    // Four warps a row where a unit has more than six warps' parts on average. Calls back to back, four / one, 8 kv heads
    // of D = 128: 1 request of 32768 keys (222 parts a unit) 19.7 / 29.4 us, 9 of 2048 (25) 13.8 / 15.5, 32 of 2048 (7)
    // 25.5 / 31.3, 64 of 2048 (3.5) 45.1 / 42.0. It does not fit everywhere: 16 of 4096 (14) 32.0 / 28.4, 37 of 2048
    // (6) 28.6 / 35.4.
    if (p.n_warps > 6 * units)
      launch_pdl(decode4_join_kernel<D, 4>, dim3(static_cast<unsigned>(rows)), 128, 0, st, p);
    else
      launch_pdl(decode4_join_kernel<D, 1>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, st, p);
    return check_launch("decode4_join_kernel");
  };
  return a->D == 128 ? with_d(std::integral_constant<int, 128>{}) : with_d(std::integral_constant<int, 64>{});
}

}  // extern "C"

// Decode attention of a batch whose requests share their first tokens: one query token per request,
// the keys below prefix_len in the same pages for all of them, the others in pages of their own.
//
//   shared part  for a kv head, the B * G query rows against the prefix are one product with M = B * G:
//                the tiles of lf_packed.cuh, each over a slice of the prefix. The prefix is read from
//                HBM once for all requests, where a paged decode reads it B times.
//   own part     a unit is the own keys of a (request, kv head), in groups of 16; all units' groups in one
//                row are dealt out to the warps in equal runs, as in decode: bound by HBM.
//   join         join_kernel: out = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m) over the parts of both.
//
// The first two are CTAs of one launch: where the slices of the prefix leave places, the own keys stream in beside
// them, and otherwise as they end. 64 requests, 2048 shared keys and up to 1024 own, 32 heads on 8: 128 prefix CTAs
// on 148 SMs, 38 us (bytes once at HBM's rate 12.6). 128 requests, 32768 shared and up to 2048 own: 288 prefix CTAs
// take nearly every place, and the own keys follow them; 136 us (53.6), where a paged decode of the same cache reads
// the prefix 128 times.
#include "lf_packed.cuh"

#include <algorithm>
#include <type_traits>

namespace lf {

constexpr int kOwnWarps = 4;
constexpr int kOwnStages = 3;
constexpr int kOwnGroup = 16;  // tokens that a warp takes at a time
constexpr int kOwnHeads = 8;   // query heads of a CTA: rows 0..7 of a 16-row MMA tile

struct OwnParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t q_stride[3], k_stride[3], v_stride[3];  // (b, kv head, g); (page, slot, kv head)
  const int32_t* table;
  int64_t bt_stride;
  const int32_t* seq_lens;
  int32_t B, G;
  int32_t heads;       // units of a request: kv heads times groups of 8 query heads
  FastDiv div_groups;  // groups of query heads
  int32_t prefix_len, max_len;
  int32_t bt_blocks, page_size, page_shift, n_pages;
  float a, c2;
  // Part of warp w for unit u: at place w + u, which no other pair has, since both only grow along the row
  // of groups; [place][8 query heads][D], (maximum, sum), and the warps that a unit's groups went to.
  float* part_o;
  float2* part_ml;
  int2* warps;
  int32_t* status;
};

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kOwnRun = 2;  // groups of a warp, at least

// Keys of request b that count, from its length: never more than the caller said or the table holds.
__device__ __forceinline__ int own_end(const int32_t* seq_lens, int b, int max_len) {
  return min(max(seq_lens[b], 0), max_len);
}

// Sixteen tokens of a unit, as a warp has them in hand.
struct OwnGroup {
  int b, head;  // request; kv head and group of query heads. b < 0: no more
  int t, end;   // first token, end of the unit
};

// The own keys, by warps 0..3 of a CTA, each for itself: all units' groups of 16 tokens in one row, of which
// warp `w` of `n_warps` has an equal run, whatever the requests' lengths. A warp's groups follow each other
// across units - the page of one is looked up while two are being copied and one is computed - so the start
// of a unit costs no round trip to memory. (128 requests of 2048 own keys, a CTA per slice of 256 keys: 3.5
// TB/s.)
//
// The layout of the products is that of decode_mma_kernel: the G query rows are rows 0..7 of the M
// dimension of m16n8k16, K and V fragments come straight from the 16-byte pieces that were copied (piece j
// of row r sits at piece j ^ (r & 7)), and P enters the second product as two bf16, its rounding in rows g
// and what that leaves in rows 8 + g, at no extra MMA.
template <int D, bool SOFTCAP>
__device__ __forceinline__ void own_part(const OwnParams& p, int w, int n_warps) {
  constexpr int KI = D / 32;  // 16-byte pieces of a K row per lane
  constexpr int VH = D / 64;
  constexpr int NT = D / 8;
  constexpr int CPR = D / 8, RPI = 32 / CPR;
  constexpr int kRowBytes = D * 2, kStageBytes = 2 * kOwnGroup * kRowBytes;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;

  // Groups of the requests [b0, b0 + 32), one per lane; those of a unit.
  int b0 = 0, groups = 0;
  auto load_groups = [&](int from) {
    b0 = from;
    const int own = b0 + lane < p.B ? own_end(p.seq_lens, b0 + lane, p.max_len) - p.prefix_len : 0;
    groups = own > 0 ? (own + kOwnGroup - 1) / kOwnGroup : 0;
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
  const long long run = max((all + n_warps - 1) / n_warps, static_cast<long long>(kOwnRun));
  long long left = min(all - w * run, run);  // groups of this warp
  if (left <= 0) return;
  OwnGroup now;
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
    now.t = p.prefix_len + static_cast<int>(into - static_cast<long long>(now.head) * n) * kOwnGroup;
    now.end = own_end(p.seq_lens, now.b, p.max_len);
  }
  // The group behind x, while this warp has any.
  auto next_group = [&](const OwnGroup& x) {
    OwnGroup y = x;
    if (--left <= 0) {
      y.b = -1;
      return y;
    }
    y.t += kOwnGroup;
    if (y.t < y.end) return y;
    y.t = p.prefix_len;
    if (++y.head < p.heads) return y;
    y.head = 0;
    for (;;) {  // the next request that has own keys
      const unsigned some = __ballot_sync(0xffffffffu, groups > 0 && b0 + lane > y.b);
      if (some) {
        y.b = b0 + __ffs(some) - 1;
        y.end = own_end(p.seq_lens, y.b, p.max_len);
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
  // Page of this lane's row of a group (rows past the end: the last token again).
  auto look_up = [&](const OwnGroup& x) {
    if (x.b < 0) return 0;
    const int at = page_of(min(x.t + (lane & 15), x.end - 1));
    if (!LF_BOUNDS(x.b < p.B && x.head < p.heads && at >= 0 && at < p.bt_blocks, p.status, 72)) return 0;
    return p.table[x.b * p.bt_stride + at];
  };
  unsigned char* ring = smem + warp * (kOwnStages * kStageBytes);
  const int r0 = lane / CPR, j0 = lane % CPR;
  const uint32_t ring_u32 = smem_u32(ring) + r0 * kRowBytes;
  auto copy_group = [&](const OwnGroup& x, int stage, int page) {
    if (x.b >= 0) {
      int g0;
      const int kvh = kv_head(x.head, &g0);
      const __nv_bfloat16* kbase = p.k + kvh * p.k_stride[2];
      const __nv_bfloat16* vbase = p.v + kvh * p.v_stride[2];
      const uint32_t dst = ring_u32 + stage * kStageBytes;
      const int t = min(x.t + (lane & 15), x.end - 1);
      if (page < 0 || page >= p.n_pages) {
        if (p.status) atomicExch(p.status, LF_DEV_BAD_PAGE);
        page = 0;
      }
      const int slot = t - page_of(t) * p.page_size;
      if (x.t + kOwnGroup <= x.end && page_of(x.t) == page_of(x.t + 15)) {
        // A group inside one page: its rows are evenly spaced.
        const int slot0 = __shfl_sync(0xffffffffu, slot, 0);
        const __nv_bfloat16* kp = kbase + static_cast<int64_t>(page) * p.k_stride[0] +
                                  (slot0 + r0) * p.k_stride[1] + 8 * j0;
        const __nv_bfloat16* vp = vbase + static_cast<int64_t>(page) * p.v_stride[0] +
                                  (slot0 + r0) * p.v_stride[1] + 8 * j0;
#pragma unroll
        for (int q = 0; q < 16 / RPI; ++q) {
          const uint32_t to = dst + q * RPI * kRowBytes + ((j0 ^ ((r0 + q * RPI) & 7)) << 4);
          cp_async_16(to, kp);
          cp_async_16(to + 16 * kRowBytes, vp);
          kp += RPI * p.k_stride[1];
          vp += RPI * p.v_stride[1];
        }
      } else {
        const int64_t off = static_cast<int64_t>(page) * (lane < 16 ? p.k_stride[0] : p.v_stride[0]) +
                            slot * (lane < 16 ? p.k_stride[1] : p.v_stride[1]);
#pragma unroll
        for (int q = 0; q < 16 / RPI; ++q) {
          const int r = r0 + q * RPI;
          const uint32_t to = dst + q * RPI * kRowBytes + ((j0 ^ (r & 7)) << 4);
          cp_async_16(to, kbase + __shfl_sync(0xffffffffu, off, r) + 8 * j0);
          cp_async_16(to + 16 * kRowBytes, vbase + __shfl_sync(0xffffffffu, off, 16 + r) + 8 * j0);
        }
      }
    }
    cp_async_commit();
  };
  uint4 qr[KI];
  auto load_q = [&](const OwnGroup& x) {
    int g0;
    const int kvh = kv_head(x.head, &g0);
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      qr[i] = make_uint4(0u, 0u, 0u, 0u);
      if (g0 + g < p.G)
        qr[i] = *reinterpret_cast<const uint4*>(p.q + x.b * p.q_stride[0] + kvh * p.q_stride[1] +
                                                (g0 + g) * p.q_stride[2] + 8 * (4 * i + c));
    }
  };

  // now: computed; then, later: being copied; ahead, last: their pages are being looked up. (One look-up
  // ahead, a warp took a group of 8 KB per round trip to the table.)
  static_assert(kOwnStages == 3, "two groups are copied while one is computed");
  OwnGroup then = next_group(now), later = next_group(then);
  load_q(now);
  {
    const int pg0 = look_up(now), pg1 = look_up(then);
    copy_group(now, 0, pg0);
    copy_group(then, 1, pg1);
  }
  OwnGroup ahead = next_group(later);
  int page = look_up(later), page_ahead = look_up(ahead);

  float m_run = -INFINITY, l_run = 0.f;
  float o[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = 0.f;

  for (int it = 0; now.b >= 0; it = it == 2 ? 0 : it + 1) {
    copy_group(later, it == 0 ? 2 : it - 1, page);
    const OwnGroup last = next_group(ahead);
    page = page_ahead;
    page_ahead = look_up(last);
    cp_async_wait<kOwnStages - 1>();
    __syncwarp();
    const unsigned char* stage = ring + it * kStageBytes;
    float sc[2][2];
#pragma unroll
    for (int s8 = 0; s8 < 2; ++s8) {
      uint4 kr[KI];
#pragma unroll
      for (int i = 0; i < KI; ++i)
        kr[i] = *reinterpret_cast<const uint4*>(stage + (8 * s8 + g) * kRowBytes + (((4 * i + c) ^ g) << 4));
      float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        mma_16816(x, qr[i].x, 0u, qr[i].y, 0u, kr[i].x, kr[i].y);
        mma_16816(y, qr[i].z, 0u, qr[i].w, 0u, kr[i].z, kr[i].w);
      }
      sc[s8][0] = x[0] + y[0];
      sc[s8][1] = x[1] + y[1];
    }
    float mx = -INFINITY;
#pragma unroll
    for (int s8 = 0; s8 < 2; ++s8)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float s = sc[s8][e];
        if constexpr (SOFTCAP) s = tanh_approx(s * p.a);  // (the unit's, within 2^-11, as in decode)
        s *= p.c2;
        if (now.t + 8 * s8 + 2 * c + e >= now.end) s = -INFINITY;
        sc[s8][e] = s;
        mx = fmaxf(mx, s);
      }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float m_new = fmaxf(m_run, mx);
    const float m_safe = m_new == -INFINITY ? 0.f : m_new;
    if (__any_sync(0xffffffffu, m_new > m_run)) {
      const float alpha = ex2_approx(m_run - m_safe);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] *= alpha;
    }
    float pr[2][2], psum = 0.f;
#pragma unroll
    for (int s8 = 0; s8 < 2; ++s8)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        pr[s8][e] = ex2_approx(sc[s8][e] - m_safe);
        psum += pr[s8][e];
      }
    l_run += psum;  // this lane's share; the quad is summed at the end of the unit
    const uint32_t pa0 = pack_bf16x2(pr[0][0], pr[0][1]);
    const uint32_t pa2 = pack_bf16x2(pr[1][0], pr[1][1]);
    const uint32_t pa1 = pack_bf16x2(pr[0][0] - bf16lo_to_f32(pa0), pr[0][1] - bf16hi_to_f32(pa0));
    const uint32_t pa3 = pack_bf16x2(pr[1][0] - bf16lo_to_f32(pa2), pr[1][1] - bf16hi_to_f32(pa2));
#pragma unroll
    for (int h = 0; h < VH; ++h) {
      uint4 vq[4];
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int r = 2 * c + (r4 & 1) + 8 * (r4 >> 1);
        vq[r4] = *reinterpret_cast<const uint4*>(stage + (16 + r) * kRowBytes +
                                                 (((8 * h + g) ^ (r & 7)) << 4));
      }
      const uint32_t w0[4] = {vq[0].x, vq[0].y, vq[0].z, vq[0].w};
      const uint32_t w1[4] = {vq[1].x, vq[1].y, vq[1].z, vq[1].w};
      const uint32_t w2[4] = {vq[2].x, vq[2].y, vq[2].z, vq[2].w};
      const uint32_t w3[4] = {vq[3].x, vq[3].y, vq[3].z, vq[3].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t sel = (e & 1) ? 0x7632u : 0x5410u;
        mma_16816(o[h * 8 + e], pa0, pa1, pa2, pa3, __byte_perm(w0[e >> 1], w1[e >> 1], sel),
                  __byte_perm(w2[e >> 1], w3[e >> 1], sel));
      }
    }
    const int unit = now.b * p.heads + now.head;
    if (lane == 0) {  // where the join finds the unit's parts
      if (now.t == p.prefix_len) p.warps[unit].x = w;
      if (now.t + kOwnGroup >= now.end) p.warps[unit].y = w;
    }
    if (then.b != now.b || then.head != now.head) {
      // This warp is done with the unit: its rows and their (maximum, sum) go to the join.
      int g0;
      kv_head(now.head, &g0);
      l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
      l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
      if (g0 + g < p.G) {
        const int64_t at = (static_cast<int64_t>(w) + unit) * kOwnHeads + g;
        float* dst = p.part_o + at * D;
#pragma unroll
        for (int h = 0; h < VH; ++h)
#pragma unroll
          for (int u = 0; u < 2; ++u) {  // output column 2c + u of MMA (h, e): d = 64 h + 16 c + 8 u + e
            uint32_t x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float y = o[h * 8 + e][u];
              x[e] = __float_as_uint(fabsf(y) != INFINITY ? y + o[h * 8 + e][2 + u] : y);
            }
            stg_32(dst + 64 * h + 16 * c + 8 * u, x);
          }
        if (c == 0) p.part_ml[at] = make_float2(m_run, l_run);
      }
      m_run = -INFINITY;
      l_run = 0.f;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
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

struct JoinParams {
  const float* prefix_o;    // [split][row][D]
  const float2* prefix_ml;  // [split][row]
  const float* own_o;       // as OwnParams has them
  const float2* own_ml;
  const int2* warps;
  __nv_bfloat16* out;
  int64_t o_stride[3];  // (b, kv head, g)
  const int32_t* seq_lens;
  int32_t prefix_len, max_len, prefix_splits;
  int64_t rows;
  int32_t Hkv, G, groups;  // groups of 8 query heads
  int32_t* status;
};

// One warp per output row. Lane s holds (reference, sum) of part s; the rows of the parts stream in with
// their weights broadcast. Parts that hold no key of the row have sum 0 and are left out (what their
// accumulators hold is of no value); a row without a key is zeros. Bound by the latency of its loads, with cold caches
// 5 us for 128 rows and 8 for 2048 and 4096.
template <int D>
__global__ void __launch_bounds__(128) join_kernel(const JoinParams p) {
  constexpr int EPL = D / 32;
  pdl_trigger();
  pdl_wait();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= p.rows) return;
  const int64_t b = row / (p.Hkv * p.G);
  const int rest = static_cast<int>(row - b * (p.Hkv * p.G));
  const int kvh = rest / p.G, g = rest - kvh * p.G;
  const int64_t unit = (b * p.Hkv + kvh) * p.groups + g / kOwnHeads;
  if (p.status && rest == 0 && lane == 0) {  // (what is cut is reported once, by the request's first row)
    const int len = p.seq_lens[b];
    if (len < 0 || len > p.max_len) atomicCAS(p.status, 0, LF_DEV_BAD_LENGTHS);
  }
  int64_t own_at = 0;
  int n = p.prefix_splits;
  if (own_end(p.seq_lens, static_cast<int>(b), p.max_len) > p.prefix_len) {
    const int2 w = p.warps[unit];
    own_at = (w.x + unit) * kOwnHeads + g % kOwnHeads;
    n += w.y - w.x + 1;
  }
  // Place of part s.
  auto place = [&](int s) {
    return s < p.prefix_splits ? s * p.rows + row
                               : own_at + static_cast<int64_t>(s - p.prefix_splits) * kOwnHeads;
  };
  float m_all = -INFINITY, l_all = 0.f;
  float o[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) o[e] = 0.f;
  for (int s0 = 0; s0 < n; s0 += 32) {
    float2 ml = make_float2(-INFINITY, 0.f);
    const int mine = s0 + lane;
    if (mine < n) ml = (mine < p.prefix_splits ? p.prefix_ml : p.own_ml)[place(mine)];
    const bool live = ml.y != 0.f;
    float m_new = live ? ml.x : -INFINITY;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, d));
    m_new = fmaxf(m_new, m_all);
    const float m_safe = m_new == -INFINITY ? 0.f : m_new;
    const float back = ex2_approx(m_all - m_safe);
    const float w = live ? ex2_approx(ml.x - m_safe) : 0.f;
    float l = ml.y * w;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    l_all = l_all * back + l;
    m_all = m_new;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] *= back;
    unsigned todo = __ballot_sync(0xffffffffu, live);
    while (todo) {
      float x[8][EPL], wt[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int s = todo ? __ffs(todo) - 1 : 0;
        const float ws = __shfl_sync(0xffffffffu, w, s);
        wt[u] = todo ? ws : 0.f;
#pragma unroll
        for (int e = 0; e < EPL; ++e) x[u][e] = 0.f;
        if (todo) {
          const float* src = (s0 + s < p.prefix_splits ? p.prefix_o : p.own_o) + place(s0 + s) * D + lane * EPL;
          if constexpr (EPL == 4) {
            const float4 v = *reinterpret_cast<const float4*>(src);
            x[u][0] = v.x; x[u][1] = v.y; x[u][2] = v.z; x[u][3] = v.w;
          } else {
            const float2 v = *reinterpret_cast<const float2*>(src);
            x[u][0] = v.x; x[u][1] = v.y;
          }
        }
        todo &= todo - 1;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[e] = fmaf(x[u][e], wt[u], o[e]);
    }
  }
  const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
  __nv_bfloat16* op = p.out + b * p.o_stride[0] + kvh * p.o_stride[1] + g * p.o_stride[2] + lane * EPL;
  if constexpr (EPL == 4)
    *reinterpret_cast<uint2*>(op) =
        make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(op) = pack_bf16x2(o[0] * inv, o[1] * inv);
}

// Both parts in one launch: the slices of the prefix, which are long, come first and take two CTAs per
// SM at most; those of the requests' own keys fill the places that are left, then the ones that get free.
template <int D, bool SOFTCAP>
__global__ void __launch_bounds__(kPackedThreads, 2)
    shared_prefix_kernel(const __grid_constant__ CUtensorMap tmap_q,
                         const __grid_constant__ CUtensorMap tmap_k,
                         const __grid_constant__ CUtensorMap tmap_v, const PackedParams p,
                         const OwnParams own, const int prefix_ctas) {
  pdl_trigger();
  const int cta = static_cast<int>(blockIdx.x);
  if (cta < prefix_ctas) {
    packed_tiles<D, kPackedPrefix, SOFTCAP>(tmap_q, tmap_k, tmap_v, p, cta);
  } else if (threadIdx.x >= kOwnWarps * 32) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    // (No tensor memory for these, but the right to ask for it has to be given up: until its CTA has done so, an
    // SM took no other one of this kernel. 128 x 2048 own keys 217 -> 175 us.)
    if (threadIdx.x < 32) tmem_relinquish();
    pdl_wait();
    // (Runs go round the CTAs first, then their warps: few of them are spread over all SMs.)
    const int ctas = static_cast<int>(gridDim.x) - prefix_ctas;
    own_part<D, SOFTCAP>(own, (threadIdx.x >> 5) * ctas + cta - prefix_ctas, ctas * kOwnWarps);
  }
}

// How a call is cut, and the room for its parts.
struct PrefixCut {
  int prefix_splits = 0, prefix_chunk = kPackedKeys;  // slices of the prefix, whole key blocks each
  int own_ctas = 0, heads = 1;
  int64_t units = 0;
  size_t prefix_parts = 0, own_parts = 0;  // rows
  size_t bytes(int D) const { return (prefix_parts + own_parts) * (D + 2) * sizeof(float) + units * sizeof(int2); }
};

static int shared_sm_count() {
  static thread_local int cached_dev = -1, cached = 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev != cached_dev) {
    cudaDeviceGetAttribute(&cached, cudaDevAttrMultiProcessorCount, dev);
    cached_dev = dev;
  }
  return cached > 0 ? cached : 148;
}

static PrefixCut cut_prefix(int B, int Hkv, int G, int prefix_len, int max_len) {
  PrefixCut c;
  const int sms = shared_sm_count();
  const int64_t rows = static_cast<int64_t>(B) * Hkv * G;
  if (prefix_len > 0) {
    const int tq = kPackedRows / G;
    const int64_t units = static_cast<int64_t>((B + tq - 1) / tq) * Hkv;
    const int blocks = (prefix_len + kPackedKeys - 1) / kPackedKeys;
    // As many slices as one wave of two CTAs per SM takes, of four key blocks or more: a slice's rows are
    // written and read again, 64 KB each way against 32 KB of K and V a block. (64 requests, 2048 shared keys: two
    // blocks 25 us, four 20.) Few rows cost less: 4 requests of 4 heads, 512 shared keys, two blocks 9.9 us, four 11.1.
    const int least = std::min(B, tq) * G > kPackedRows / 2 ? 4 : 2;
    int64_t s = std::max<int64_t>(1, 2ll * sms / units);
    s = std::min<int64_t>(s, (blocks + least - 1) / least);
    const int per = static_cast<int>((blocks + s - 1) / s);
    c.prefix_chunk = per * kPackedKeys;
    c.prefix_splits = (blocks + per - 1) / per;
    c.prefix_parts = static_cast<size_t>(c.prefix_splits) * rows;
  }
  const int own = std::max(0, max_len - prefix_len);
  if (own > 0) {
    c.heads = Hkv * ((G + kOwnHeads - 1) / kOwnHeads);
    c.units = static_cast<int64_t>(B) * c.heads;
    const int64_t runs = (c.units * ((own + kOwnGroup - 1) / kOwnGroup) + kOwnRun - 1) / kOwnRun;
    c.own_ctas = static_cast<int>(std::min<int64_t>(runs, 2ll * sms));
    c.own_parts = static_cast<size_t>(c.units + c.own_ctas * kOwnWarps) * kOwnHeads;
  }
  return c;
}

template <int D, bool SOFTCAP>
static int launch_shared(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                         const PackedParams& pp, const OwnParams& po, int prefix_ctas, unsigned grid,
                         cudaStream_t st) {
  using Shape = PackedShape<D>;
  constexpr size_t ring = static_cast<size_t>(kOwnWarps) * kOwnStages * 2 * kOwnGroup * D * 2;
  static_assert(ring <= Shape::kSmem, "the rings of the own part");
  static thread_local int configured_dev = -1;
  const auto kernel = shared_prefix_kernel<D, SOFTCAP>;
  const int rc = packed_configure(kernel, Shape::kSmem, &configured_dev);
  if (rc != LF_OK) return rc;
  launch_pdl(kernel, dim3(grid), kPackedThreads, Shape::kSmem, st, mq, mk, mv, pp, po, prefix_ctas);
  return check_launch("shared_prefix_kernel");
}

}  // namespace lf

extern "C" {

size_t lf_shared_prefix_workspace_bytes(int32_t B, int32_t Hkv, int32_t G, int32_t D, int32_t prefix_len,
                                        int32_t max_seq_len) {
  using namespace lf;
  if (B <= 0 || Hkv <= 0 || G <= 0 || G > kPackedRows || D <= 0 || prefix_len < 0) return 0;
  return cut_prefix(B, Hkv, G, std::min(prefix_len, max_seq_len), max_seq_len).bytes(D);
}

int lf_shared_prefix_decode_bf16(const LfSharedPrefixArgs* a, void* stream) {
  using namespace lf;
  if (!a || !a->q || !a->k || !a->v || !a->out || !a->block_table || !a->seq_lens) return LF_ERR_INVALID_ARG;
  if (a->B <= 0 || a->Hkv <= 0 || a->G <= 0 || a->page_size <= 0 || a->n_pages <= 0 || a->bt_blocks <= 0 ||
      a->prefix_len < 0 || a->max_seq_len < 0)
    return LF_ERR_INVALID_ARG;
  if (a->D != 64 && a->D != 128) return LF_ERR_UNSUPPORTED;
  if (a->G > kPackedRows) return LF_ERR_UNSUPPORTED;
  const int64_t held = static_cast<int64_t>(a->bt_blocks) * a->page_size;
  if (a->prefix_len > held || a->max_seq_len > held) return LF_ERR_INVALID_ARG;
  if (a->max_seq_len > kMostKeys) return LF_ERR_TOO_LARGE;
  PackedScore score;
  int rc = packed_score(a->scale, a->n_mod, a->mod_op, a->mod_arg, &score);
  if (rc != LF_OK) return rc;
  const int head_groups = (a->G + kOwnHeads - 1) / kOwnHeads;
  if (a->B > 65535 || static_cast<int64_t>(a->B) * a->Hkv * head_groups > (1 << 26)) return LF_ERR_TOO_LARGE;
  if (!packed_aligned(a->q) || !packed_aligned(a->k) || !packed_aligned(a->v) || !packed_aligned(a->out))
    return LF_ERR_ALIGNMENT;
  for (int i = 0; i < 3; ++i)
    if (a->q_stride[i] % 8 || a->k_stride[i] % 8 || a->v_stride[i] % 8 || a->o_stride[i] % 4)
      return LF_ERR_ALIGNMENT;
  const int64_t rows = static_cast<int64_t>(a->B) * a->Hkv * a->G;
  const int prefix_len = std::min(a->prefix_len, a->max_seq_len);
  const PrefixCut cut = cut_prefix(a->B, a->Hkv, a->G, prefix_len, a->max_seq_len);
  const size_t need = cut.bytes(a->D);
  if (need && (!a->workspace || a->workspace_bytes < need)) return LF_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) & 31u) return LF_ERR_ALIGNMENT;  // (32-byte stores)
  float* part_o = static_cast<float*>(a->workspace);
  float* own_o = part_o + cut.prefix_parts * a->D;
  float2* part_ml = reinterpret_cast<float2*>(own_o + cut.own_parts * a->D);
  float2* own_ml = part_ml + cut.prefix_parts;
  int2* warps = reinterpret_cast<int2*>(own_ml + cut.own_parts);

  PackedParams pp = {};
  OwnParams po = {};
  CUtensorMap mq = {}, mk = {}, mv = {};
  int64_t prefix_ctas = 0;
  const int page_shift = packed_page_shift(a->page_size);
  if (cut.prefix_splits > 0) {
    pp.kv_lens = a->seq_lens;
    pp.table = a->block_table;
    pp.bt_stride = a->bt_stride;
    pp.B = a->B;
    pp.Hkv = a->Hkv;
    pp.G = a->G;
    pp.tq = kPackedRows / a->G;
    pp.a = score.a;
    pp.c2 = score.c2;
    pp.m_first = score.m_first;
    pp.bt_blocks = a->bt_blocks;
    pp.page_size = a->page_size;
    pp.page_shift = page_shift;
    pp.n_pages = a->n_pages;
    pp.prefix_len = prefix_len;
    pp.chunk = cut.prefix_chunk;
    pp.part_o = part_o;
    pp.part_ml = part_ml;
    pp.status = a->status;
    pp.n_tiles = (a->B + pp.tq - 1) / pp.tq;
    pp.div_tiles = FastDiv::make(pp.n_tiles);
    pp.div_chunk = FastDiv::make(a->Hkv);
    pp.div_g = FastDiv::make(a->G);
    prefix_ctas = static_cast<int64_t>(pp.n_tiles) * a->Hkv * cut.prefix_splits;
    rc = make_map_5d(&mq, TileMapSpec{a->q, {a->D, a->G, a->Hkv, a->B, 1},
                                      {a->q_stride[2], a->q_stride[1], a->q_stride[0], 0}, {a->G, 1, pp.tq, 1}});
    if (rc == LF_OK)
      rc = packed_pool_maps(&mk, &mv, a->k, a->v, a->k_stride, a->v_stride, a->n_pages, a->page_size, a->Hkv,
                            a->D, &pp);
    if (rc != LF_OK) return rc;
  }
  po.q = static_cast<const __nv_bfloat16*>(a->q);
  po.k = static_cast<const __nv_bfloat16*>(a->k);
  po.v = static_cast<const __nv_bfloat16*>(a->v);
  JoinParams pj = {};
  for (int i = 0; i < 3; ++i) {
    po.q_stride[i] = a->q_stride[i];
    po.k_stride[i] = a->k_stride[i];
    po.v_stride[i] = a->v_stride[i];
    pj.o_stride[i] = a->o_stride[i];
  }
  po.table = a->block_table;
  po.bt_stride = a->bt_stride;
  po.seq_lens = pj.seq_lens = a->seq_lens;
  po.B = a->B;
  po.G = pj.G = a->G;
  po.heads = a->Hkv * head_groups;
  po.div_groups = FastDiv::make(head_groups);
  po.prefix_len = pj.prefix_len = prefix_len;
  po.max_len = pj.max_len = a->max_seq_len;
  po.bt_blocks = a->bt_blocks;
  po.page_size = a->page_size;
  po.page_shift = page_shift;
  po.n_pages = a->n_pages;
  po.a = score.a;
  po.c2 = score.c2;
  po.part_o = own_o;
  po.part_ml = own_ml;
  po.warps = warps;
  po.status = a->status;
  pj.prefix_o = part_o;
  pj.prefix_ml = part_ml;
  pj.own_o = own_o;
  pj.own_ml = own_ml;
  pj.warps = warps;
  pj.prefix_splits = cut.prefix_splits;
  pj.Hkv = a->Hkv;
  pj.groups = head_groups;
  pj.out = static_cast<__nv_bfloat16*>(a->out);
  pj.rows = rows;
  pj.status = a->status;

  const int64_t grid = prefix_ctas + cut.own_ctas;
  if (grid > 0x7fffffff) return LF_ERR_TOO_LARGE;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto with_d = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (grid > 0) {
      const auto launch = score.softcap ? launch_shared<D, true> : launch_shared<D, false>;
      const int r = launch(mq, mk, mv, pp, po, static_cast<int>(prefix_ctas), static_cast<unsigned>(grid), st);
      if (r != LF_OK) return r;
    }
    launch_pdl(join_kernel<D>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, st, pj);
    return check_launch("join_kernel");
  };
  return a->D == 128 ? with_d(std::integral_constant<int, 128>{}) : with_d(std::integral_constant<int, 64>{});
}

}  // extern "C"

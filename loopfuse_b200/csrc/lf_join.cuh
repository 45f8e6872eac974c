// The join of attention partials of requests of different lengths, and what the kernels that write them share.
#pragma once

#include "lf_common.cuh"

namespace lf {

constexpr int kOwnHeads = 8;  // query heads that a warp computes together: 8 rows of a matrix instruction

// Keys of request b that count, from its length: never more than the caller said or the table holds.
__device__ __forceinline__ int own_end(const int32_t* seq_lens, int b, int max_len) {
  return min(max(seq_lens[b], 0), max_len);
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
static __global__ void __launch_bounds__(128) join_kernel(const JoinParams p) {
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

}  // namespace lf

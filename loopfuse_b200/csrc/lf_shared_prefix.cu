// Decode attention of a batch whose requests share their first tokens: one query token per request,
// the keys below prefix_len in the same pages for all of them, the others in pages of their own.
//
//   shared part  for a kv head, the B * G query rows against the prefix are one product with M = B * G:
//                the tiles of lf_packed.cuh, each over a slice of the prefix. The prefix is read from
//                HBM once for all requests, where a paged decode reads it B times.
//   own part     own_kernel: a CTA per (request, kv head, slice of its own keys), as in decode: bound by
//                HBM.
//   join         join_kernel: out = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m) over the slices of both.
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
  int32_t B, Hkv, G, head_groups;
  int32_t prefix_len, max_len, chunk, first_split;  // first_split: slices of the prefix
  int32_t page_size, page_shift, n_pages;
  float a, c2;
  float* part_o;
  float2* part_ml;
  int32_t* status;
};

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Keys of request b that count, from its length: never more than the caller said or the table holds.
__device__ __forceinline__ int own_end(const int32_t* seq_lens, int b, int max_len) {
  return min(max(seq_lens[b], 0), max_len);
}

// The layout of the products is that of decode_mma_kernel: the G query rows are rows 0..7 of the M
// dimension of m16n8k16, K and V fragments come straight from the 16-byte pieces that were copied
// (piece j of row r sits at piece j ^ (r & 7)), and P enters the second product as two bf16, its
// rounding in rows g and what that leaves in rows 8 + g, at no extra MMA.
template <int D, bool SOFTCAP>
__global__ void __launch_bounds__(kOwnWarps * 32, 2) own_kernel(const OwnParams p) {
  constexpr int KI = D / 32;  // 16-byte pieces of a K row per lane
  constexpr int VH = D / 64;
  constexpr int NT = D / 8;
  constexpr int CPR = D / 8, RPI = 32 / CPR;
  constexpr int kRowBytes = D * 2, kStageBytes = 2 * kOwnGroup * kRowBytes;
  extern __shared__ __align__(1024) unsigned char smem[];
  pdl_trigger();
  pdl_wait();
  const int split = blockIdx.x;
  const int kvh = blockIdx.y / p.head_groups;
  const int g0 = (blockIdx.y - kvh * p.head_groups) * kOwnHeads;
  const int b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int n_heads = min(kOwnHeads, p.G - g0);
  const int end = own_end(p.seq_lens, b, p.max_len);
  const int t0 = p.prefix_len + split * p.chunk;
  const int t1 = min(end, t0 + p.chunk);
  if (t0 >= t1) return;

  uint4 qr[KI];
#pragma unroll
  for (int i = 0; i < KI; ++i) {
    qr[i] = make_uint4(0u, 0u, 0u, 0u);
    if (g < n_heads)
      qr[i] = *reinterpret_cast<const uint4*>(p.q + b * p.q_stride[0] + kvh * p.q_stride[1] +
                                              (g0 + g) * p.q_stride[2] + 8 * (4 * i + c));
  }
  const __nv_bfloat16* kbase = p.k + kvh * p.k_stride[2];
  const __nv_bfloat16* vbase = p.v + kvh * p.v_stride[2];
  const int32_t* table = p.table + b * p.bt_stride;
  auto page_of = [&](int t) { return p.page_shift >= 0 ? (t >> p.page_shift) : (t / p.page_size); };
  const int t_last = t1 - 1;
  // Page of this lane's row of the group at tg (rows past the end: the last token again), requested a
  // group ahead of its use.
  auto request = [&](int tg) {
    return tg < t1 ? table[page_of(min(tg + (lane & 15), t_last))] : 0;
  };
  unsigned char* ring = smem + warp * (kOwnStages * kStageBytes);
  const int r0 = lane / CPR, j0 = lane % CPR;
  const uint32_t ring_u32 = smem_u32(ring) + r0 * kRowBytes;
  auto copy_group = [&](int tg, int stage, int page) {
    if (tg < t1) {
      const uint32_t dst = ring_u32 + stage * kStageBytes;
      const int t = min(tg + (lane & 15), t_last);
      const int pg = page_of(t);
      if (page < 0 || page >= p.n_pages) {
        if (p.status) atomicExch(p.status, LF_DEV_BAD_PAGE);
        page = 0;
      }
      const int slot = t - pg * p.page_size;
      if (tg + 15 <= t_last && page_of(tg) == page_of(tg + 15)) {
        // A group inside one page: its rows are evenly spaced.
        const __nv_bfloat16* kp = kbase + static_cast<int64_t>(page) * p.k_stride[0] +
                                  __shfl_sync(0xffffffffu, slot, 0) * p.k_stride[1] +
                                  r0 * p.k_stride[1] + 8 * j0;
        const __nv_bfloat16* vp = vbase + static_cast<int64_t>(page) * p.v_stride[0] +
                                  __shfl_sync(0xffffffffu, slot, 0) * p.v_stride[1] +
                                  r0 * p.v_stride[1] + 8 * j0;
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

  float m_run = -INFINITY, l_run = 0.f;
  float o[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = 0.f;

  constexpr int kStep = kOwnGroup * kOwnWarps;
  const int tg0 = t0 + warp * kOwnGroup;
  int page = request(tg0);
#pragma unroll
  for (int st = 0; st < kOwnStages - 1; ++st) {
    const int next = request(tg0 + (st + 1) * kStep);
    copy_group(tg0 + st * kStep, st, page);
    page = next;
  }
  int it = 0;
  for (int tg = tg0; tg < t1; tg += kStep, ++it) {
    const int next = request(tg + kOwnStages * kStep);
    copy_group(tg + (kOwnStages - 1) * kStep, (it + kOwnStages - 1) % kOwnStages, page);
    page = next;
    cp_async_wait<kOwnStages - 1>();
    __syncwarp();
    const unsigned char* stage = ring + (it % kOwnStages) * kStageBytes;
    uint4 kr[2][KI];
#pragma unroll
    for (int s8 = 0; s8 < 2; ++s8)
#pragma unroll
      for (int i = 0; i < KI; ++i)
        kr[s8][i] =
            *reinterpret_cast<const uint4*>(stage + (8 * s8 + g) * kRowBytes + (((4 * i + c) ^ g) << 4));
    float sc[2][2];
#pragma unroll
    for (int s8 = 0; s8 < 2; ++s8) {
      float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        mma_16816(x, qr[i].x, 0u, qr[i].y, 0u, kr[s8][i].x, kr[s8][i].y);
        mma_16816(y, qr[i].z, 0u, qr[i].w, 0u, kr[s8][i].z, kr[s8][i].w);
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
        if constexpr (SOFTCAP) s = tanh_approx(s * p.a);
        s *= p.c2;
        if (tg + 8 * s8 + 2 * c + e >= t1) s = -INFINITY;
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
    l_run += psum;  // this lane's share; the quad is summed after the loop
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
    __syncwarp();
  }
  cp_async_wait<0>();
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (fabsf(o[j][e]) != INFINITY) o[j][e] += o[j][2 + e];
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);

  // The warps' parts meet in shared memory (in the rings), [warp][head][D + 2].
  constexpr int kStride = D + 2;
  float* merge = reinterpret_cast<float*>(smem);
  __syncthreads();
  if (g < n_heads) {
    float* dst = merge + (warp * n_heads + g) * kStride;
#pragma unroll
    for (int h = 0; h < VH; ++h)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dst[64 * h + 16 * c + e] = o[h * 8 + e][0];
        dst[64 * h + 16 * c + 8 + e] = o[h * 8 + e][1];
      }
    if (c == 0) {
      dst[D] = m_run;
      dst[D + 1] = l_run;
    }
  }
  __syncthreads();
  const int64_t row0 = (static_cast<int64_t>(b) * p.Hkv + kvh) * p.G + g0;
  const int64_t rows = static_cast<int64_t>(p.B) * p.Hkv * p.G;
  for (int idx = threadIdx.x; idx < n_heads * D; idx += kOwnWarps * 32) {
    const int gg = idx / D, cc = idx - gg * D;
    float m_all = -INFINITY;
#pragma unroll
    for (int w = 0; w < kOwnWarps; ++w) m_all = fmaxf(m_all, merge[(w * n_heads + gg) * kStride + D]);
    const float m_safe = m_all == -INFINITY ? 0.f : m_all;
    float l_all = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kOwnWarps; ++w) {
      const float* src = merge + (w * n_heads + gg) * kStride;
      const float wt = ex2_approx(src[D] - m_safe);
      l_all += src[D + 1] * wt;
      acc += src[cc] * wt;
    }
    const int64_t at = (p.first_split + split) * rows + row0 + gg;
    p.part_o[at * D + cc] = acc;
    if (cc == 0) p.part_ml[at] = make_float2(m_all, l_all);
  }
}

struct JoinParams {
  const float* part_o;
  const float2* part_ml;
  __nv_bfloat16* out;
  int64_t o_stride[3];  // (b, kv head, g)
  const int32_t* seq_lens;
  int32_t prefix_len, max_len, chunk, prefix_splits;
  int64_t rows;
  int32_t Hkv, G;
};

// One warp per output row. Lane s holds (reference, sum) of slice s; the rows of the slices stream in with
// their weights broadcast. Slices that hold no key of the row have sum 0 and are left out (what their
// accumulators hold is of no value); a row without a key is zeros.
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
  const int own = own_end(p.seq_lens, static_cast<int>(b), p.max_len) - p.prefix_len;
  const int n = p.prefix_splits + (own > 0 ? (own + p.chunk - 1) / p.chunk : 0);
  float m_all = -INFINITY, l_all = 0.f;
  float o[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) o[e] = 0.f;
  for (int s0 = 0; s0 < n; s0 += 32) {
    float2 ml = make_float2(-INFINITY, 0.f);
    if (s0 + lane < n) ml = p.part_ml[(s0 + lane) * p.rows + row];
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
      float x[4][EPL], wt[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = todo ? __ffs(todo) - 1 : 0;
        const float ws = __shfl_sync(0xffffffffu, w, s);
        wt[u] = todo ? ws : 0.f;
#pragma unroll
        for (int e = 0; e < EPL; ++e) x[u][e] = 0.f;
        if (todo) {
          const float* src = p.part_o + ((s0 + s) * p.rows + row) * D + lane * EPL;
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
      for (int u = 0; u < 4; ++u)
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

template <int D, bool SOFTCAP>
__global__ void __launch_bounds__(kPackedThreads, 2)
    prefix_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                  const __grid_constant__ CUtensorMap tmap_v, const PackedParams p) {
  pdl_trigger();
  packed_tiles<D, kPackedPrefix, SOFTCAP>(tmap_q, tmap_k, tmap_v, p, blockIdx.x);
}

// How a call is cut: slices of the prefix (a multiple of a key block each), and of the requests' own keys.
struct PrefixCut {
  int prefix_splits, prefix_chunk, own_splits, own_chunk;
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
  PrefixCut c = {0, kPackedKeys, 0, 256};
  const int sms = shared_sm_count();
  if (prefix_len > 0) {
    const int tq = kPackedRows / G;
    const int64_t units = static_cast<int64_t>((B + tq - 1) / tq) * Hkv;
    const int blocks = (prefix_len + kPackedKeys - 1) / kPackedKeys;
    // As many slices as one wave of two CTAs per SM takes, of four key blocks or more.
    int64_t s = std::max<int64_t>(1, 2ll * sms / units);
    s = std::min<int64_t>(s, (blocks + 3) / 4);
    const int per = static_cast<int>((blocks + s - 1) / s);
    c.prefix_chunk = per * kPackedKeys;
    c.prefix_splits = (blocks + per - 1) / per;
  }
  const int own = std::max(0, max_len - prefix_len);
  if (own > 0) {
    const int64_t units = static_cast<int64_t>(B) * Hkv * ((G + kOwnHeads - 1) / kOwnHeads);
    if (units * ((own + 255) / 256) < 2 * sms) c.own_chunk = 128;
    // (Slices of very long requests grow, so that there are never more than 256 of them.)
    c.own_chunk = std::max(c.own_chunk, ((own + 255) / 256 + kOwnGroup - 1) / kOwnGroup * kOwnGroup);
    c.own_splits = (own + c.own_chunk - 1) / c.own_chunk;
  }
  return c;
}

static size_t shared_workspace(const PrefixCut& c, int64_t rows, int D) {
  return static_cast<size_t>(c.prefix_splits + c.own_splits) * rows * (D + 2) * sizeof(float);
}

template <int D, bool SOFTCAP>
static int launch_shared(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                         const PackedParams& pp, unsigned grid, const OwnParams& po, const PrefixCut& cut,
                         cudaStream_t st) {
  using Shape = PackedShape<D>;
  if (cut.prefix_splits > 0) {
    static thread_local int configured_dev = -1;
    const auto kernel = prefix_kernel<D, SOFTCAP>;
    int rc = packed_configure(kernel, Shape::kSmem, &configured_dev);
    if (rc != LF_OK) return rc;
    launch_pdl(kernel, dim3(grid), kPackedThreads, Shape::kSmem, st, mq, mk, mv, pp);
    rc = check_launch("prefix_kernel");
    if (rc != LF_OK) return rc;
  }
  if (cut.own_splits > 0) {
    constexpr size_t smem = static_cast<size_t>(kOwnWarps) * kOwnStages * 2 * kOwnGroup * D * 2;
    static_assert(static_cast<size_t>(kOwnWarps) * kOwnHeads * (D + 2) * 4 <= smem, "merge area in the rings");
    static thread_local int configured_dev = -1;
    const auto kernel = own_kernel<D, SOFTCAP>;
    int rc = packed_configure(kernel, smem, &configured_dev);
    if (rc != LF_OK) return rc;
    launch_pdl(kernel, dim3(cut.own_splits, po.Hkv * po.head_groups, po.B), kOwnWarps * 32, smem, st, po);
    rc = check_launch("own_kernel");
    if (rc != LF_OK) return rc;
  }
  return LF_OK;
}

}  // namespace lf

extern "C" {

size_t lf_shared_prefix_workspace_bytes(int32_t B, int32_t Hkv, int32_t G, int32_t D, int32_t prefix_len,
                                        int32_t max_seq_len) {
  using namespace lf;
  if (B <= 0 || Hkv <= 0 || G <= 0 || G > kPackedRows || D <= 0 || prefix_len < 0) return 0;
  return shared_workspace(cut_prefix(B, Hkv, G, std::min(prefix_len, max_seq_len), max_seq_len),
                          static_cast<int64_t>(B) * Hkv * G, D);
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
  PackedScore score;
  int rc = packed_score(a->scale, a->n_mod, a->mod_op, a->mod_arg, &score);
  if (rc != LF_OK) return rc;
  const int head_groups = (a->G + kOwnHeads - 1) / kOwnHeads;
  if (a->B > 65535 || static_cast<int64_t>(a->Hkv) * head_groups > 65535) return LF_ERR_TOO_LARGE;
  if (!packed_aligned(a->q) || !packed_aligned(a->k) || !packed_aligned(a->v) || !packed_aligned(a->out))
    return LF_ERR_ALIGNMENT;
  for (int i = 0; i < 3; ++i)
    if (a->q_stride[i] % 8 || a->k_stride[i] % 8 || a->v_stride[i] % 8 || a->o_stride[i] % 4)
      return LF_ERR_ALIGNMENT;
  const int64_t rows = static_cast<int64_t>(a->B) * a->Hkv * a->G;
  const int prefix_len = std::min(a->prefix_len, a->max_seq_len);
  const PrefixCut cut = cut_prefix(a->B, a->Hkv, a->G, prefix_len, a->max_seq_len);
  const size_t need = shared_workspace(cut, rows, a->D);
  if (need && (!a->workspace || a->workspace_bytes < need)) return LF_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) & 31u) return LF_ERR_ALIGNMENT;  // (32-byte stores)
  float* part_o = static_cast<float*>(a->workspace);
  float2* part_ml =
      reinterpret_cast<float2*>(part_o + static_cast<size_t>(cut.prefix_splits + cut.own_splits) * rows * a->D);

  PackedParams pp = {};
  OwnParams po = {};
  CUtensorMap mq = {}, mk = {}, mv = {};
  unsigned grid = 0;
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
    pp.box = packed_box(a->page_size);
    pp.prefix_len = prefix_len;
    pp.chunk = cut.prefix_chunk;
    pp.part_o = part_o;
    pp.part_ml = part_ml;
    pp.status = a->status;
    pp.n_tiles = (a->B + pp.tq - 1) / pp.tq;
    pp.div_tiles = FastDiv::make(pp.n_tiles);
    pp.div_chunk = FastDiv::make(a->Hkv);
    pp.div_g = FastDiv::make(a->G);
    const int64_t ctas = static_cast<int64_t>(pp.n_tiles) * a->Hkv * cut.prefix_splits;
    if (ctas > 0x7fffffff) return LF_ERR_TOO_LARGE;
    grid = static_cast<unsigned>(ctas);
    rc = make_map_4d(&mq, TileMapSpec{a->q, {a->D, a->G, a->Hkv, a->B},
                                      {a->q_stride[2], a->q_stride[1], a->q_stride[0]}, {a->G, 1, pp.tq}});
    if (rc == LF_OK)
      rc = packed_pool_map(&mk, a->k, a->k_stride, a->n_pages, a->page_size, a->Hkv, a->D, pp.box);
    if (rc == LF_OK)
      rc = packed_pool_map(&mv, a->v, a->v_stride, a->n_pages, a->page_size, a->Hkv, a->D, pp.box);
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
  po.Hkv = pj.Hkv = a->Hkv;
  po.G = pj.G = a->G;
  po.head_groups = head_groups;
  po.prefix_len = pj.prefix_len = prefix_len;
  po.max_len = pj.max_len = a->max_seq_len;
  po.chunk = pj.chunk = cut.own_chunk;
  po.first_split = pj.prefix_splits = cut.prefix_splits;
  po.page_size = a->page_size;
  po.page_shift = page_shift;
  po.n_pages = a->n_pages;
  po.a = score.a;
  po.c2 = score.c2;
  po.part_o = part_o;
  po.part_ml = part_ml;
  po.status = a->status;
  pj.part_o = part_o;
  pj.part_ml = part_ml;
  pj.out = static_cast<__nv_bfloat16*>(a->out);
  pj.rows = rows;

  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto with_d = [&](auto d) {
    constexpr int D = decltype(d)::value;
    const int r = score.softcap ? launch_shared<D, true>(mq, mk, mv, pp, grid, po, cut, st)
                                : launch_shared<D, false>(mq, mk, mv, pp, grid, po, cut, st);
    if (r != LF_OK) return r;
    launch_pdl(join_kernel<D>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, st, pj);
    return check_launch("join_kernel");
  };
  return a->D == 128 ? with_d(std::integral_constant<int, 128>{}) : with_d(std::integral_constant<int, 64>{});
}

}  // extern "C"

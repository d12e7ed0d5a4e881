// decode_maps.hip -- decode steps whose attention maps are used beyond softmax(q
// K^T) V (sched_decode_maps): each token's weight added up, or the difference of
// two maps. Two launches: a kernel that streams the cache once (chunks of tasks
// over the card), and one that joins the chunks and writes what the operator
// hands on (maps.h has the mathematics).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "maps_mfma.h"
#include "rt_internal.h"

using namespace schedpd;

namespace {

constexpr int kBlock = 256;
constexpr uint32_t kMostRows = 16;

template <typename T> __device__ __forceinline__ float val(const T *p);
template <> __device__ __forceinline__ float val(const float *p) { return *p; }
template <> __device__ __forceinline__ float val(const uint16_t *p) {
  return bf16_bits_to_f32(*p);
}
template <> __device__ __forceinline__ float val(const _Float16 *p) { return (float)*p; }
template <> __device__ __forceinline__ float val(const uint8_t *p) { return fp8e4m3_to_f32(*p); }

// The general stream: any cache type, layout and strides. A workgroup reads one chunk
// of one task in tiles of 32 tokens: keys and values go to LDS as fp32; each of the
// eight 32-lane groups scores the tile's tokens for two rows, in the lanes; then each
// lane adds the tile's values into one dim of some rows.
template <typename T, int D, bool DIFF>
__global__ void __launch_bounds__(kBlock) maps_valu(MapParams P) {
  constexpr uint32_t TT = 32;                   // tokens of a tile
  constexpr uint32_t RG = kBlock / (D < kBlock ? D : kBlock); // row groups of the products
  constexpr uint32_t RPL = kMostRows / RG;      // rows of a lane
  __shared__ float s_q[kMostRows][D];
  __shared__ float s_k[TT][D + 1];
  __shared__ float s_v[TT][D];
  __shared__ float s_p[kMostRows][TT + 1];
  __shared__ float s_c[kMostRows];
  __shared__ int32_t s_page[TT / 4];
  const uint32_t tid = threadIdx.x, lane32 = tid & 31u, grp = tid >> 5;
  const uint32_t task = blockIdx.x, chunk = blockIdx.y;
  const uint64_t item = (uint64_t)task * P.nsplit + chunk;
  const uint32_t r = task / P.Hkv, h = task % P.Hkv;
  const uint32_t n = map_tokens(P, r), len = map_chunk(P, n);
  const uint64_t first = (uint64_t)chunk * len;
  if (first >= n && chunk > 0u)
    return;
  const uint32_t t0 = (uint32_t)first, t1 = (uint32_t)(first + len < n ? first + len : n);
  const int64_t row = map_row(P, r);
  const uint64_t b0 = DIFF ? 0 : blocks_before(P, r);

  // map row 2g + a of the difference holds q-head g's half a, the other half zero
  for (uint32_t i = tid; i < P.rows * D; i += kBlock) {
    const uint32_t g = i / D, j = i % D;
    const uint32_t hq = h * P.G + (DIFF ? g >> 1 : g);
    const bool in = !DIFF || (j >= D / 2) == (g & 1u);
    s_q[g][j] = in ? map_load_q(P, ((int64_t)r * P.Hq + hq) * D + j) * P.scale_log2 : 0.f;
  }
  float m[2] = {kMInit, kMInit}, l[2] = {0.f, 0.f};
  float acc[RPL];
#pragma unroll
  for (uint32_t i = 0; i < RPL; ++i)
    acc[i] = 0.f;
  const uint32_t j0 = tid % (D < kBlock ? D : kBlock), rg = tid / D;

  const T *kp = static_cast<const T *>(P.k_pool) + (int64_t)h * P.khs;
  const T *vp = static_cast<const T *>(P.v_pool) + (int64_t)h * P.vhs;
  for (uint32_t tb = t0; tb < t1; tb += TT) {
    const uint32_t cnt = t1 - tb < TT ? t1 - tb : TT;
    __syncthreads();
    // page ids of the tile: at most TT / 16 + 1 pages, pages hold 16 tokens or more
    const uint32_t pg0 = tb / P.ps, pg1 = (tb + cnt - 1u) / P.ps;
    if (tid <= pg1 - pg0)
      s_page[tid] = P.bt[row + pg0 + tid];
    __syncthreads();
    for (uint32_t i = tid; i < TT * D; i += kBlock) {
      const uint32_t t = i / D, j = i % D;
      float x = 0.f;
      if (t < cnt) {
        const uint32_t page = (uint32_t)s_page[(tb + t) / P.ps - pg0], slot = (tb + t) % P.ps;
        if (page < P.num_pages) {
          x = val(kp + (int64_t)page * P.kps + (int64_t)slot * P.kts + j);
          if (sizeof(T) == 1 && P.k_scale)
            x *= P.k_scale[((int64_t)page * P.Hkv + h) * P.scale_stride];
        }
      }
      s_k[t][j] = x;
    }
    // the order of the values' loads follows their layout
    for (uint32_t i = tid; i < TT * D; i += kBlock) {
      const uint32_t t = P.vds == 1 ? i / D : i % TT, j = P.vds == 1 ? i % D : i / TT;
      float x = 0.f;
      if (t < cnt) {
        const uint32_t page = (uint32_t)s_page[(tb + t) / P.ps - pg0], slot = (tb + t) % P.ps;
        if (page < P.num_pages) {
          x = val(vp + (int64_t)page * P.vps + (int64_t)slot * P.vts + (int64_t)j * P.vds);
          if (sizeof(T) == 1 && P.v_scale)
            x *= P.v_scale[((int64_t)page * P.Hkv + h) * P.scale_stride];
        }
      }
      s_v[t][j] = x;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k) {
      const uint32_t g = grp + 8u * k;
      if (g >= P.rows)
        continue;
      float a = 0.f;
      const uint32_t j_lo = DIFF && (g & 1u) ? D / 2 : 0u, j_hi = DIFF && !(g & 1u) ? D / 2 : D;
      for (uint32_t j = j_lo; j < j_hi; ++j)
        a += s_q[g][j] * s_k[lane32][j];
      const bool in = lane32 < cnt;
      const float s = in ? a : kNegInf;
      if (!DIFF && in) {
        const uint32_t t = tb + lane32;
        if (b0 + t / 16u < P.score_blocks)
          score_block(P, b0, t / 16u, h)[g * 16u + (t & 15u)] = s;
      }
      float mx = s;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        mx = fmaxf(mx, __shfl_xor(mx, o, 32));
      const float mn = fmaxf(m[k], mx), c = __builtin_amdgcn_exp2f(m[k] - mn);
      const float p = in ? __builtin_amdgcn_exp2f(s - mn) : 0.f;
      float sum = p;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        sum += __shfl_xor(sum, o, 32);
      m[k] = mn;
      l[k] = l[k] * c + sum;
      s_p[g][lane32] = p;
      if (lane32 == 0)
        s_c[g] = c;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < RPL; ++i) {
      const uint32_t g = rg + RG * i;
      if (g >= P.rows)
        continue;
      float a = acc[i] * s_c[g];
      for (uint32_t t = 0; t < cnt; ++t)
        a += s_p[g][t] * s_v[t][j0];
      acc[i] = a;
    }
  }
#pragma unroll
  for (uint32_t k = 0; k < 2; ++k) {
    const uint32_t g = grp + 8u * k;
    if (g < P.rows && lane32 == 0) {
      float *ml = P.ml + (item * P.rows + g) * 2u;
      ml[0] = m[k];
      ml[1] = l[k];
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < RPL; ++i) {
    const uint32_t g = rg + RG * i;
    if (g < P.rows)
      P.acc[(item * P.rows + g) * D + j0] = acc[i];
  }
}

constexpr int kJoin = 512;

// Rows [g0, g1) of a task joined over its chunks: M and 1 / L into s_M, s_Li. A wave
// takes a row at a time, its lanes the chunks.
__device__ __forceinline__ void join_rows(const MapParams &P, uint64_t item0, uint32_t nch,
                                          uint32_t g0, uint32_t g1, float *s_M, float *s_Li) {
  const uint32_t lane = threadIdx.x & 63u;
  for (uint32_t g = g0 + (threadIdx.x >> 6); g < g1; g += kJoin / 64) {
    float m = kMInit, l = 0.f;
    for (uint32_t c = lane; c < nch; c += 64u) {
      const float *e = P.ml + ((item0 + c) * P.rows + g) * 2u;
      const float mc = e[0], lc = e[1], mn = fmaxf(m, mc);
      l = l * __builtin_amdgcn_exp2f(m - mn) + lc * __builtin_amdgcn_exp2f(mc - mn);
      m = mn;
    }
    float M = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
      M = fmaxf(M, __shfl_xor(M, o));
    float L = l * __builtin_amdgcn_exp2f(m - M);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
      L += __shfl_xor(L, o);
    if (lane == 0) {
      s_M[g] = M;
      s_Li[g] = 1.f / L;
    }
  }
}

// The join of what `maps_valu` and, for tasks of several chunks, maps_mfma left:
// workgroup (task, y). y < outs: the output of q-head y (FEW: of all of them); from there on the
// weights, kTokens tokens a workgroup and round. A dim's chunks are summed by kJoin / D lanes,
// 8 loads in flight each, and their sums in order.
constexpr uint32_t kTokens = 4 * kJoin;

constexpr uint32_t FEWCH = 16; // chunks of a task up to which one workgroup has its outputs

template <int D, bool DIFF, bool FEW>
__global__ void __launch_bounds__(kJoin) maps_join(MapParams P, uint32_t outs) {
  constexpr uint32_t LANES = kJoin / D, NR = DIFF ? 2 : 1, CH = 64;
  __shared__ float s_M[kMostRows], s_Li[kMostRows];
  __shared__ float s_f[NR][CH], s_o[NR][LANES][D], s_sum[kJoin / 64];
  __shared__ float s_w[kMostRows][FEWCH];
  const uint32_t tid = threadIdx.x, task = blockIdx.x;
  const uint32_t r = task / P.Hkv, h = task % P.Hkv;
  const uint32_t n = map_tokens(P, r), len = map_chunk(P, n);
  const uint32_t nch = n == 0u ? 1u : (n + len - 1u) / len;
  if (nch <= P.join_from)
    return; // the stream has finished this task
  const uint64_t item0 = (uint64_t)task * P.nsplit;
  if (FEW && blockIdx.y == 0u) {
    // a lane sums an element's few chunks: no workgroup-wide steps between the rows
    join_rows(P, item0, nch, 0u, P.rows, s_M, s_Li);
    __syncthreads();
    if (tid < P.rows * FEWCH) {
      const uint32_t g = tid / FEWCH, c = tid % FEWCH;
      s_w[g][c] = c < nch ? __builtin_amdgcn_exp2f(P.ml[((item0 + c) * P.rows + g) * 2u] - s_M[g]) *
                                s_Li[g]
                          : 0.f;
    }
    __syncthreads();
    const float *acc = P.acc + item0 * P.rows * D;
    const uint32_t hop = P.rows * D;
    auto joined = [&](uint32_t g, uint32_t j) __attribute__((always_inline)) {
      float o = 0.f;
      for (uint32_t c0 = 0; c0 < nch; c0 += 4u) {
        float v[4];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
          v[u] = acc[(uint64_t)min(c0 + u, nch - 1u) * hop + g * D + j];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
          o += c0 + u < nch ? v[u] * s_w[g][c0 + u] : 0.f;
      }
      return o;
    };
    const float nan = __builtin_nanf("");
    if constexpr (!DIFF) {
      for (uint32_t i = tid; i < P.rows * D; i += kJoin) {
        const uint32_t g = i / D, j = i % D;
        const float o = joined(g, j);
        map_store(P, ((int64_t)r * P.Hq + h * P.G + g) * D + j, n ? o : nan);
      }
    } else {
      const uint32_t lane = tid & 63u;
      for (uint32_t g = tid >> 6; g < P.G; g += kJoin / 64) {
        const uint32_t hq = h * P.G + g;
        const float la = P.lam[hq];
        float o[D / 64], ss = 0.f;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const uint32_t j = lane + 64u * i;
          o[i] = joined(2u * g, j) - la * joined(2u * g + 1u, j);
          ss += o[i] * o[i];
        }
        float inv = P.mul;
        if (P.nw) {
#pragma unroll
          for (int k = 32; k > 0; k >>= 1)
            ss += __shfl_xor(ss, k);
          inv *= rsqrtf(ss / (float)D + P.eps);
        }
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const uint32_t j = lane + 64u * i;
          map_store(P, ((int64_t)r * P.Hq + hq) * D + j,
                    n ? o[i] * inv * (P.nw ? P.nw[j] : 1.f) : nan);
        }
      }
    }
    return;
  }
  if (!FEW && blockIdx.y < outs) {
    join_rows(P, item0, nch, blockIdx.y * NR, blockIdx.y * NR + NR, s_M, s_Li);
    const uint32_t j = tid % D, part = tid / D;
    {
      const uint32_t g = blockIdx.y, g0 = g * NR, hq = h * P.G + g;
      float o[NR] = {};
      for (uint32_t c0 = 0; c0 < nch; c0 += CH) {
        const uint32_t cnt = min(CH, nch - c0);
        __syncthreads(); // the rows are joined; the previous shares have been used
        if (tid < NR * CH) {
          const uint32_t k = tid / CH, c = tid % CH;
          s_f[k][c] = c < cnt ? __builtin_amdgcn_exp2f(
                                    P.ml[((item0 + c0 + c) * P.rows + g0 + k) * 2u] - s_M[g0 + k]) *
                                    s_Li[g0 + k]
                              : 0.f;
        }
        __syncthreads();
        for (uint32_t c = part; c < cnt; c += 8u * LANES) {
          float v[8][NR];
#pragma unroll
          for (uint32_t u = 0; u < 8; ++u) {
            const uint32_t cc = min(c + u * LANES, cnt - 1u);
#pragma unroll
            for (uint32_t k = 0; k < NR; ++k)
              v[u][k] = P.acc[((item0 + c0 + cc) * P.rows + g0 + k) * D + j];
          }
#pragma unroll
          for (uint32_t u = 0; u < 8; ++u)
#pragma unroll
            for (uint32_t k = 0; k < NR; ++k)
              if (c + u * LANES < cnt)
                o[k] += v[u][k] * s_f[k][c + u * LANES];
        }
      }
#pragma unroll
      for (uint32_t k = 0; k < NR; ++k)
        s_o[k][part][j] = o[k];
      __syncthreads();
      float x = 0.f;
      if (tid < D) {
        float t[NR];
#pragma unroll
        for (uint32_t k = 0; k < NR; ++k) {
          t[k] = s_o[k][0][tid];
#pragma unroll
          for (uint32_t q = 1; q < LANES; ++q)
            t[k] += s_o[k][q][tid];
        }
        x = t[0];
        if constexpr (DIFF)
          x -= P.lam[hq] * t[NR - 1];
      }
      if constexpr (DIFF) {
        float inv = P.mul;
        if (P.nw) {
          float ss = x * x;
#pragma unroll
          for (int k = 32; k > 0; k >>= 1)
            ss += __shfl_xor(ss, k);
          if ((tid & 63u) == 0u)
            s_sum[tid >> 6] = ss;
          __syncthreads();
          ss = s_sum[0];
#pragma unroll
          for (int k = 1; k < D / 64; ++k)
            ss += s_sum[k];
          inv *= rsqrtf(ss / (float)D + P.eps);
          if (tid < D)
            inv *= P.nw[tid];
        }
        x *= inv;
      }
      if (tid < D)
        map_store(P, ((int64_t)r * P.Hq + hq) * D + tid, n ? x : __builtin_nanf(""));
    }
    return;
  }
  if constexpr (!DIFF) {
    const uint32_t first = (blockIdx.y - outs) * kTokens, stride = (gridDim.y - outs) * kTokens;
    if (first >= n)
      return;
    join_rows(P, item0, nch, 0u, P.rows, s_M, s_Li);
    const uint64_t b0 = blocks_before(P, r);
    const int64_t row = map_row(P, r);
    const int64_t have = P.counted ? (int64_t)P.counted[r] : (int64_t)n;
    __syncthreads();
    for (uint32_t t = first + tid * 4u; t < n; t += stride) {
      const uint32_t page = (uint32_t)P.bt[row + t / P.ps];
      if (page < P.num_pages && b0 + t / 16u < P.score_blocks)
        map_weights4(P, h, page, t, n, have, score_block(P, b0, t / 16u, h) + (t & 15u), s_M, s_Li);
    }
  }
}

template <bool DIFF, bool FEW> auto join_of(uint32_t d) {
  return d == 32    ? maps_join<DIFF ? 64 : 32, DIFF, FEW>
         : d == 64  ? maps_join<64, DIFF, FEW>
         : d == 128 ? maps_join<128, DIFF, FEW>
                    : maps_join<256, DIFF, FEW>;
}

uint64_t up256(uint64_t x) { return (x + 255u) & ~uint64_t(255); }

uint64_t elem_bytes(uint32_t dt) {
  return dt == SCHED_PD_F32 ? 4u : dt == SCHED_PD_FP8_E4M3 ? 1u : 2u;
}

// What a call's shape decides: how far tasks are split, and the workspace.
struct Plan {
  bool mfma;
  uint32_t rows, nsplit, chunk;
  uint64_t score_blocks, ml_off, acc_off, total;
};

int check_shape(const SchedMapsArgs *a) {
  if (!a)
    return set_error(hipErrorInvalidValue, "sched_decode_maps: args is NULL");
  if (a->abi_version != SCHED_MAPS_ABI_VERSION)
    return set_error(hipErrorInvalidValue, "sched_decode_maps: abi_version %u, library has %u",
                     a->abi_version, SCHED_MAPS_ABI_VERSION);
  if (a->op > SCHED_MAPS_DIFF)
    return set_error(hipErrorInvalidValue, "sched_decode_maps: op %u", a->op);
  auto float_dt = [](uint32_t dt) {
    return dt == SCHED_PD_F32 || dt == SCHED_PD_BF16 || dt == SCHED_PD_F16;
  };
  if (a->kv_dtype > SCHED_PD_F16 || !float_dt(a->q_dtype) || !float_dt(a->o_dtype))
    return set_error(hipErrorInvalidValue, "sched_decode_maps: dtypes (kv %u, q %u, out %u)",
                     a->kv_dtype, a->q_dtype, a->o_dtype);
  if (a->num_kv_heads == 0 || a->num_q_heads == 0 || a->num_q_heads % a->num_kv_heads)
    return set_error(hipErrorInvalidValue,
                     "sched_decode_maps: num_q_heads %u is not a multiple of num_kv_heads %u",
                     a->num_q_heads, a->num_kv_heads);
  const bool diff = a->op == SCHED_MAPS_DIFF;
  const uint32_t G = a->num_q_heads / a->num_kv_heads;
  if (G > (diff ? kMostRows / 2 : kMostRows))
    return set_error(hipErrorInvalidValue,
                     "sched_decode_maps: %u q-heads per kv-head, at most %u supported", G,
                     diff ? kMostRows / 2 : kMostRows);
  const uint32_t d = a->head_dim;
  if (!(d == 64 || d == 128 || d == 256 || (d == 32 && !diff)))
    return set_error(hipErrorInvalidValue, "sched_decode_maps: head_dim %u (supported: %s64, 128, "
                                           "256)", d, diff ? "" : "32, ");
  if (a->page_size == 0 || a->page_size % 16 || a->page_size > 256)
    return set_error(hipErrorInvalidValue,
                     "sched_decode_maps: page_size %u (multiple of 16, at most 256)",
                     a->page_size);
  if (a->flags & ~SCHED_PD_FLAG_FORCE_VALU)
    return set_error(hipErrorInvalidValue, "sched_decode_maps: flags 0x%x (FORCE_VALU or 0)",
                     a->flags);
  if (a->num_pages == 0 || a->num_pages > 0x7fffffffull)
    return set_error(hipErrorInvalidValue, "sched_decode_maps: num_pages %llu",
                     (unsigned long long)a->num_pages);
  if ((uint64_t)a->num_requests * a->num_kv_heads > (1u << 24) ||
      (uint64_t)a->max_pages * a->page_size > (1u << 24))
    return set_error(hipErrorInvalidValue, "sched_decode_maps: %u requests x %u kv-heads, tables "
                                           "of %u pages", a->num_requests, a->num_kv_heads,
                     a->max_pages);
  return 0;
}

// The matrix cores: fp32 and 16-bit caches with queries of their type, fp8 ones with bf16
// queries, rows that 16-byte loads reach, and lane offsets within 32 bits.
bool mfma_applies(const SchedMapsArgs *a) {
  if ((a->flags & SCHED_PD_FLAG_FORCE_VALU) || a->head_dim == 32)
    return false;
  const bool fp8 = a->kv_dtype == SCHED_PD_FP8_E4M3;
  if (a->q_dtype != (fp8 ? SCHED_PD_BF16 : a->kv_dtype))
    return false;
  const int64_t eb = elem_bytes(a->kv_dtype);
  const bool vt = a->v_dim_stride == 1;
  const int64_t vrow = (vt ? a->v_tok_stride : a->v_dim_stride) * eb, krow = a->k_tok_stride * eb;
  for (int64_t s : {a->k_page_stride * eb, a->k_head_stride * eb, krow, a->v_page_stride * eb,
                    a->v_head_stride * eb, vrow})
    if (s % 16)
      return false;
  return krow > 0 && vrow > 0 && krow < (1 << 26) && vrow < (1 << 25) &&
         ((uintptr_t)a->k_pool & 15u) == 0 && ((uintptr_t)a->v_pool & 15u) == 0 &&
         ((uintptr_t)a->q & 15u) == 0;
}

// How tasks are cut (map_chunk): into chunks of 8 tokens for each task of the call, between
// kLeastChunk and kMostChunk, so that a few long tasks fill the card and many tasks stay
// whole, but for the longest (a split task costs its partials and the join). In us, bf16,
// 32 / 8 heads of 128, at 4, 8 and 16 tokens a task: 16 x 2048 tokens 33.0 / 31.0 / 34.0, 32
// x 2048 56.9 / 47.7 / 47.5, differential 48 requests of 200..2900 71.4 / 65.0 / 65.3; one
// request of 1000 with kLeastChunk 256 13.6, with 512 15.5. Longer chunks where a table would
// make more than kMostSplit of a task (one request of 100003 tokens: 64 of them 79.3, 96 82.2,
// 128 84.4: more than one round of workgroups) or kMostItems of the call. On the matrix
// cores a weighted chunk's scores fit kScoreBytes of LDS (64 lognormal contexts up to 4000:
// 32 KB 81.7, 40 77.5, 48 83.5; 64 x 2048: 32 KB cut in two, 107, 40 90.3).
// Rows of 512 bytes and more: at least 128 tokens (two requests of 1000, 256 dims of bf16:
// 256 tokens 14.6, 128 12.6), fp32 ones at 4 tokens a task (8, 4 and 2: 16 fp32 requests up
// to 2000 43.1 / 29.5 / 32.9, 40 differential ones up to 1500 of 256 dims 90 / 75 / 78, 64 x
// 1000 36.2 / 36.2 / 44.1).
constexpr uint64_t kChunkPerTask = 8, kLeastChunk = 256, kMostChunk = 2048;
constexpr uint64_t kWideRow = 512, kWideLeast = 128, kWidePerTask = 4;
constexpr uint64_t kMostSplit = 64, kMostItems = 4096;
constexpr uint32_t kScoreBytes = 40u << 10;

Plan plan_of(const SchedMapsArgs *a) {
  Plan p{};
  const uint64_t tasks = std::max<uint64_t>(1, (uint64_t)a->num_requests * a->num_kv_heads);
  const uint64_t longest = (uint64_t)a->max_pages * a->page_size;
  const bool weighted = a->op == SCHED_MAPS_WEIGHTED;
  p.mfma = mfma_applies(a);
  p.rows = a->num_q_heads / a->num_kv_heads * (weighted ? 1u : 2u);
  const bool wide = (uint64_t)a->head_dim * elem_bytes(a->kv_dtype) >= kWideRow;
  const uint64_t per = wide && a->kv_dtype == SCHED_PD_F32 ? kWidePerTask : kChunkPerTask;
  uint64_t chunk = std::max(per * tasks, wide ? kWideLeast : kLeastChunk);
  chunk = std::min(chunk, kMostChunk);
  chunk = std::max({chunk, longest / kMostSplit, longest * tasks / kMostItems});
  if (weighted && p.mfma) // a whole task may have 3/2 of it
    chunk = std::min<uint64_t>(chunk, kScoreBytes / (p.rows * 4u) * 2u / 3u);
  chunk = (chunk + 63u) & ~uint64_t(63);
  if (weighted && p.mfma && (chunk + chunk / 2u + 63u) / 64u * 64u * p.rows * 4u > kScoreBytes)
    chunk -= 64u;
  p.chunk = (uint32_t)chunk;
  p.nsplit = longest <= chunk + chunk / 2u ? 1u : (uint32_t)((longest + chunk - 1u) / chunk);
  if (weighted) {
    // a call's pages are distinct: never more of them than the pool has
    uint64_t pages = a->page_indptr ? a->max_pages : (uint64_t)a->num_requests * a->max_pages;
    pages = std::min<uint64_t>(pages, a->num_pages);
    p.score_blocks = pages * (a->page_size / 16u);
  }
  p.ml_off = up256(p.score_blocks * a->num_kv_heads * p.rows * 64u);
  p.acc_off = p.ml_off + up256(tasks * p.nsplit * p.rows * 8u);
  p.total = p.acc_off + tasks * p.nsplit * p.rows * a->head_dim * 4u;
  return p;
}

typedef void (*StreamFn)(MapParams);

template <typename T> StreamFn valu_of(uint32_t d, bool diff) {
  switch (d) {
  case 32: return maps_valu<T, 32, false>;
  case 64: return diff ? maps_valu<T, 64, true> : maps_valu<T, 64, false>;
  case 128: return diff ? maps_valu<T, 128, true> : maps_valu<T, 128, false>;
  default: return diff ? maps_valu<T, 256, true> : maps_valu<T, 256, false>;
  }
}

// Blocks in flight per wave and the waves per SIMD they leave room for. Head dim 128 of 16
// bits at three waves spills 4 registers (64 lognormal contexts 87 us, at two 77.5); two
// blocks of 256 dims spill 44 at two waves, and at one wave without spills take 52.3 us
// where one block at two waves takes 48.4 (32771 tokens, the keys of the next block
// under way while a block's values are multiplied). Blocks of fp32 are as many bytes as that
// and go one by one: 64 dims at four waves 14.5 us, two blocks at three 16.7, four at two
// 18.8 (96 x 30..300 tokens); 128 dims at two waves 36.2, two blocks at one 38.0 (64 x 1000).
template <int KV, int D, bool VT, bool DIFF> StreamFn mfma_rows(uint32_t rows) {
  constexpr bool FP8 = KV == kMapFp8, F32 = KV == kMapF32;
  constexpr int DEPTH = F32 ? 1 : D == 256 ? (FP8 ? 2 : 1) : D == 128 ? (FP8 ? 3 : 2) : 4;
  constexpr int WPE = F32 ? 256 / D : D == 256 || (D == 128 && !FP8) ? 2 : 3;
  return rows <= 4   ? maps_mfma<KV, D, VT, 4, DIFF, 4, DEPTH, WPE>
         : rows <= 8 ? maps_mfma<KV, D, VT, 8, DIFF, 4, DEPTH, WPE>
                     : maps_mfma<KV, D, VT, 16, DIFF, 4, DEPTH, WPE>;
}

template <int KV, bool VT> StreamFn mfma_of(uint32_t d, bool diff, uint32_t rows) {
  if (d == 64)
    return diff ? mfma_rows<KV, 64, VT, true>(rows) : mfma_rows<KV, 64, VT, false>(rows);
  if (d == 128)
    return diff ? mfma_rows<KV, 128, VT, true>(rows) : mfma_rows<KV, 128, VT, false>(rows);
  return diff ? mfma_rows<KV, 256, VT, true>(rows) : mfma_rows<KV, 256, VT, false>(rows);
}

template <int KV> StreamFn mfma_of(uint32_t d, bool vt, bool diff, uint32_t rows) {
  return vt ? mfma_of<KV, true>(d, diff, rows) : mfma_of<KV, false>(d, diff, rows);
}

} // namespace

extern "C" {

void sched_maps_default_args(SchedMapsArgs *a) {
  if (!a)
    return;
  *a = SchedMapsArgs{};
  a->abi_version = SCHED_MAPS_ABI_VERSION;
  a->kv_dtype = a->q_dtype = a->o_dtype = SCHED_PD_BF16;
  a->decay = 1.f;
  a->eps = 1e-5f;
  a->out_scale = 1.f;
}

int64_t sched_decode_maps_workspace_bytes(const SchedMapsArgs *a) {
  if (check_shape(a))
    return -1;
  return (int64_t)plan_of(a).total;
}

int sched_decode_maps_kernel_kind(const SchedMapsArgs *a) {
  if (check_shape(a))
    return -1;
  return mfma_applies(a) ? 1 : 0;
}

int sched_decode_maps(const SchedMapsArgs *a, void *stream) {
  if (int rc = check_shape(a))
    return rc;
  if (a->num_requests == 0)
    return 0;
  const bool diff = a->op == SCHED_MAPS_DIFF;
  if (!a->q || !a->out || !a->k_pool || !a->v_pool || !a->block_table || !a->ctx_lens)
    return set_error(hipErrorInvalidValue, "sched_decode_maps: a required pointer is NULL");
  if (diff ? a->lam == nullptr : a->weights == nullptr)
    return set_error(hipErrorInvalidValue, "sched_decode_maps: %s is required",
                     diff ? "lam" : "weights");
  if (a->kv_dtype == SCHED_PD_FP8_E4M3 && (!a->k_scale || !a->v_scale))
    return set_error(hipErrorInvalidValue, "sched_decode_maps: an fp8 cache needs k_scale and "
                                           "v_scale");
  if (!a->page_indptr && a->bt_stride < a->max_pages)
    return set_error(hipErrorInvalidValue, "sched_decode_maps: bt_stride %u below max_pages %u",
                     a->bt_stride, a->max_pages);
  if (a->v_tok_stride != 1 && a->v_dim_stride != 1)
    return set_error(hipErrorInvalidValue, "sched_decode_maps: V needs v_tok_stride == 1 "
                                           "(d-major) or v_dim_stride == 1 (token-major)");
  const uintptr_t eb = elem_bytes(a->kv_dtype);
  if ((uintptr_t)a->k_pool % eb || (uintptr_t)a->v_pool % eb ||
      (uintptr_t)a->q % elem_bytes(a->q_dtype) || (uintptr_t)a->out % elem_bytes(a->o_dtype))
    return set_error(hipErrorInvalidValue,
                     "sched_decode_maps: a tensor is not aligned to its elements");
  const Plan plan = plan_of(a);
  if (!a->workspace || a->workspace_bytes < plan.total || ((uintptr_t)a->workspace & 255u))
    return set_error(hipErrorInvalidValue, "sched_decode_maps: needs a 256-byte aligned workspace "
                                           "of %llu bytes (got %llu)",
                     (unsigned long long)plan.total, (unsigned long long)a->workspace_bytes);
  MapParams P{};
  P.q = a->q, P.out = a->out, P.k_pool = a->k_pool, P.v_pool = a->v_pool;
  P.kps = a->k_page_stride, P.khs = a->k_head_stride, P.kts = a->k_tok_stride;
  P.vps = a->v_page_stride, P.vhs = a->v_head_stride, P.vts = a->v_tok_stride;
  P.vds = a->v_dim_stride;
  P.k_scale = a->k_scale, P.v_scale = a->v_scale;
  P.scale_stride = (a->k_scale != nullptr && a->v_scale == a->k_scale + 1) ? 2u : 1u;
  P.bt = a->block_table, P.indptr = a->page_indptr, P.ctx = a->ctx_lens;
  P.R = a->num_requests, P.Hq = a->num_q_heads, P.Hkv = a->num_kv_heads;
  P.G = a->num_q_heads / a->num_kv_heads, P.rows = plan.rows;
  P.D = a->head_dim, P.ps = a->page_size, P.bt_stride = a->bt_stride;
  P.max_pages = a->max_pages, P.num_pages = (uint32_t)a->num_pages;
  P.q_dtype = a->q_dtype, P.o_dtype = a->o_dtype;
  P.nsplit = plan.nsplit, P.chunk = plan.chunk;
  const float dims = (float)(diff ? a->head_dim / 2u : a->head_dim);
  P.scale_log2 = (a->sm_scale != 0.f ? a->sm_scale : 1.0f / std::sqrt(dims)) *
                 1.4426950408889634f;
  P.w = a->weights, P.w_ps = a->w_page_stride, P.w_hs = a->w_head_stride;
  P.counted = a->counted, P.decay = a->decay;
  P.w_vec = ((uintptr_t)a->weights & 15u) == 0 && a->w_page_stride % 4 == 0 &&
            a->w_head_stride % 4 == 0;
  P.lam = a->lam, P.nw = a->norm_weight, P.eps = a->eps, P.mul = a->out_scale;
  uint8_t *ws = static_cast<uint8_t *>(a->workspace);
  P.scores = reinterpret_cast<float *>(ws), P.score_blocks = plan.score_blocks;
  P.ml = reinterpret_cast<float *>(ws + plan.ml_off);
  P.acc = reinterpret_cast<float *>(ws + plan.acc_off);

  P.join_from = plan.mfma ? 1u : 0u;
  const uint32_t tasks = P.R * P.Hkv;
  StreamFn fn;
  if (plan.mfma)
    fn = a->kv_dtype == SCHED_PD_F32   ? mfma_of<kMapF32>(P.D, P.vds == 1, diff, P.rows)
         : a->kv_dtype == SCHED_PD_BF16 ? mfma_of<kMapBf16>(P.D, P.vds == 1, diff, P.rows)
         : a->kv_dtype == SCHED_PD_F16 ? mfma_of<kMapF16>(P.D, P.vds == 1, diff, P.rows)
                                       : mfma_of<kMapFp8>(P.D, P.vds == 1, diff, P.rows);
  else
    fn = a->kv_dtype == SCHED_PD_F32    ? valu_of<float>(P.D, diff)
         : a->kv_dtype == SCHED_PD_BF16 ? valu_of<uint16_t>(P.D, diff)
         : a->kv_dtype == SCHED_PD_F16  ? valu_of<_Float16>(P.D, diff)
                                        : valu_of<uint8_t>(P.D, diff);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint64_t longest = (uint64_t)P.max_pages * P.ps;
  uint32_t lds = 0;
  if (plan.mfma && !diff) {
    // the longest chunk's scores
    const uint64_t most = (std::min<uint64_t>(longest, P.chunk + P.chunk / 2u) + 63u) & ~uint64_t(63);
    lds = (uint32_t)(most * P.rows * 4u);
  }
  hipLaunchKernelGGL(fn, dim3(tasks, P.nsplit), dim3(kBlock), lds, s, P);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && P.nsplit > P.join_from) {
    // few chunks: one workgroup has all of a task's outputs
    const bool few = P.nsplit <= FEWCH;
    const uint32_t outs = few ? 1u : P.G;
    uint32_t by = outs;
    if (!diff)
      by += (uint32_t)std::max<uint64_t>(
          1, std::min<uint64_t>((longest + kTokens - 1) / kTokens, 4096u / tasks + 1u));
    auto join = few ? (diff ? join_of<true, true>(P.D) : join_of<false, true>(P.D))
                    : (diff ? join_of<true, false>(P.D) : join_of<false, false>(P.D));
    hipLaunchKernelGGL(join, dim3(tasks, by), dim3(kJoin), 0, s, P, outs);
    e = hipGetLastError();
  }
  if (e != hipSuccess)
    return set_error(e, "sched_decode_maps: launch failed: %s", hipGetErrorString(e));
  return 0;
}

} // extern "C"

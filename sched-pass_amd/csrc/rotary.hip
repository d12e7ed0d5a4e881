// rotary.hip -- norm of queries and keys per head with the position rotation in the
// same pass (sched_qk_norm_rope), the key and value rows straight into the paged
// cache if there is one.
//
// Per row x of d dims (one token, one head), in fp32:
//   x' = x * w * rsqrt(mean(x^2) + eps),
//   (y_a, y_b) = (x'_a c - x'_b s, x'_b c + x'_a s) for the rotated pairs,
// rounded once. Bound by its bytes: each row is read once and written once, the
// token's angles are read once per workgroup and shared by its heads through the
// cache. Measured: 15600 new tokens of 32 / 8 heads of 128, bf16, into a cache, 104 us (3.7
// TB/s of 5.2 that a copy reaches); a step of 256 tokens 5.6 us, of one 4.6 us (launch, then
// position, table and row one behind the other).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.h"
#include "rt_internal.h"
#include "sched_kv.h"

using namespace schedpd;

namespace {

constexpr int kBlock = 256;
// Workgroups of one token per lane group, W: below kOneToken of them each lane group takes one
// token (a step of 256 tokens: 5.4 us, with two 6.6), from there on W / kFill of them, 4 to
// 16. 4097 tokens of 18 rows of 64 dims (W 2341): one token 13.4 us, two 8.2, four 8.4,
// eight 11.0, sixteen 15.7; 9 prompts of 301..2900 tokens, 48 rows of 128 dims (W 44000):
// four 115, eight 108, sixteen 105. Non-temporal loads of the rows: 105 -> 99, but rows
// that the projection has just written, as they come, 20.8 -> 25.2 (5000 tokens, 24 rows).
constexpr uint32_t kOneToken = 2048, kFill = 1024, kLeastPer = 4, kMostPer = 16;

struct RParams {
  const void *q, *k, *v;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  void *qo, *ko;
  int64_t qo_ts, qo_hs, ko_ts, ko_hs;
  const void *qw, *kw;
  const void *pos;
  const float *cs;
  int64_t cs_stride;
  uint32_t *errors;
  uint32_t T, Hq, Hkv, d, rot, max_pos;
  uint32_t v_rows; // value rows that go along with a token's keys
  uint32_t w_dtype, inter, pos64;
  float eps;
  // the cache (kp == nullptr: none)
  void *kp, *vp;
  int64_t kps, khs, kts, vps, vhs, vts, vds;
  const int32_t *app, *ctx, *table, *pind;
  uint32_t ps, bt_stride;
  uint64_t num_pages;
};

template <int DT> __device__ __forceinline__ float ld(const void *p, int64_t i) {
  if constexpr (DT == SCHED_PD_F32)
    return static_cast<const float *>(p)[i];
  else if constexpr (DT == SCHED_PD_BF16)
    return bf16_bits_to_f32(static_cast<const uint16_t *>(p)[i]);
  else
    return (float)static_cast<const _Float16 *>(p)[i];
}

template <int DT> __device__ __forceinline__ void st(void *p, int64_t i, float v) {
  if constexpr (DT == SCHED_PD_F32)
    static_cast<float *>(p)[i] = v;
  else if constexpr (DT == SCHED_PD_BF16)
    static_cast<uint16_t *>(p)[i] = f32_to_bf16_rne(v);
  else
    static_cast<_Float16 *>(p)[i] = (_Float16)v;
}

// 16 bits as a bf16 or an fp16, by a select: as one of three branches per element, under a
// lane's condition, hipcc 7.2 left a register of the fp16 branch unset (the row's
// address was built from it).
__device__ __forceinline__ float half_w(uint32_t w_dtype, uint32_t b) {
  const float x = bf16_bits_to_f32(b), y = (float)__builtin_bit_cast(_Float16, (uint16_t)b);
  return w_dtype == SCHED_PD_BF16 ? x : y;
}

__device__ __forceinline__ float load_w(const RParams &P, const void *w, uint32_t j) {
  if (P.w_dtype == SCHED_PD_F32)
    return static_cast<const float *>(w)[j];
  return half_w(P.w_dtype, static_cast<const uint16_t *>(w)[j]);
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    x += __shfl_xor(x, o);
  return x;
}

// Where a token's cache rows go: the page, and the slot in it; page -1 = nowhere.
struct Place {
  int64_t page;
  uint32_t slot;
};

// The tokens [a0, a0 + n) of one request (the whole batch without a cache).
struct Span {
  int64_t a0, n, ctx, row, cap;
};

__device__ __forceinline__ Span span_of(const RParams &P, uint32_t r) {
  Span s{0, P.T, 0, 0, 0};
  if (P.kp == nullptr)
    return s;
  const int64_t a0 = P.app[r], a1 = P.app[r + 1];
  s.a0 = a0 < 0 ? 0 : a0;
  s.n = (a1 < (int64_t)P.T ? a1 : (int64_t)P.T) - s.a0; // rows outside the sources: skipped
  s.ctx = P.ctx[r];
  s.row = P.pind ? (int64_t)P.pind[r] : (int64_t)r * P.bt_stride;
  s.cap = P.pind ? (int64_t)P.pind[r + 1] - P.pind[r] : (int64_t)P.bt_stride;
  return s;
}

__device__ __forceinline__ Place place_of(const RParams &P, const Span &s, int64_t i) {
  const int64_t at = s.ctx - s.n + i;
  if (at < 0)
    return {-1, 0};
  const int64_t b = at / P.ps;
  if (b >= s.cap)
    return {-1, 0};
  const int32_t page = P.table[s.row + b];
  if (page < 0 || (uint64_t)page >= P.num_pages)
    return {-1, 0};
  return {page, (uint32_t)(at % P.ps)};
}

__device__ __forceinline__ int64_t position_of(const RParams &P, int64_t tok) {
  return P.pos64 ? static_cast<const int64_t *>(P.pos)[tok]
                 : (int64_t) static_cast<const int32_t *>(P.pos)[tok];
}

// Every shape: one wave per row, element e = lane + 64 i of it in each lane. The
// rotated partner of an element is read from the row itself.
template <int DT> __global__ void __launch_bounds__(kBlock) rotary_rows(RParams P) {
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Span S = span_of(P, blockIdx.x);
  const uint32_t rows = P.Hq + P.Hkv + P.v_rows, half = P.rot / 2u;
  for (int64_t i = blockIdx.y; i < S.n; i += gridDim.y) {
    const int64_t tok = S.a0 + i;
    const int64_t pos = position_of(P, tok);
    if (pos < 0 || pos >= (int64_t)P.max_pos) {
      if (threadIdx.x == 0 && P.errors)
        atomicAdd(P.errors, 1u);
      continue;
    }
    const float *cs = P.cs + pos * P.cs_stride;
    Place at{-1, 0};
    if (P.kp) {
      at = place_of(P, S, i);
      if (at.page < 0 && threadIdx.x == 0 && P.errors)
        atomicAdd(P.errors, P.Hkv);
    }
    for (uint32_t row = wave; row < rows; row += kBlock / 64) {
      const bool isq = row < P.Hq, isv = row >= P.Hq + P.Hkv;
      const uint32_t h = isq ? row : isv ? row - P.Hq - P.Hkv : row - P.Hq;
      const void *src = isq ? P.q : isv ? P.v : P.k;
      const int64_t s0 = isq   ? tok * P.q_ts + h * P.q_hs
                         : isv ? tok * P.v_ts + h * P.v_hs
                               : tok * P.k_ts + h * P.k_hs;
      void *dst;
      int64_t d0, ds = 1;
      if (isq) {
        dst = P.qo, d0 = tok * P.qo_ts + h * P.qo_hs;
      } else if (P.kp == nullptr) {
        dst = P.ko, d0 = tok * P.ko_ts + h * P.ko_hs;
      } else if (at.page < 0) {
        continue;
      } else if (isv) {
        dst = P.vp, d0 = at.page * P.vps + h * P.vhs + at.slot * P.vts, ds = P.vds;
      } else {
        dst = P.kp, d0 = at.page * P.kps + h * P.khs + at.slot * P.kts;
      }
      const void *w = isv ? nullptr : isq ? P.qw : P.kw;
      float x[4], y[4];
      float ss = 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t e = lane + 64u * u;
        x[u] = e < P.d ? ld<DT>(src, s0 + e) : 0.f;
        // the partner in the rotated pair
        const uint32_t p = P.inter ? e ^ 1u : e < half ? e + half : e - half;
        y[u] = !isv && e < P.rot ? ld<DT>(src, s0 + p) : 0.f;
        ss += x[u] * x[u];
      }
      float inv = 1.f;
      if (w != nullptr)
        inv = rsqrtf(wave_sum(ss) / (float)P.d + P.eps);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t e = lane + 64u * u;
        if (e >= P.d)
          continue;
        float o = x[u];
        if (w != nullptr)
          o *= inv * load_w(P, w, e);
        if (!isv && e < P.rot) {
          const uint32_t p = P.inter ? e ^ 1u : e < half ? e + half : e - half;
          const uint32_t j = P.inter ? e >> 1 : e < half ? e : e - half;
          const bool first = P.inter ? (e & 1u) == 0u : e < half;
          const float c = cs[j], s = cs[half + j];
          const float b = w != nullptr ? y[u] * (inv * load_w(P, w, p)) : y[u];
          o = first ? o * c - b * s : o * c + b * s;
        }
        st<DT>(dst, d0 + e * ds, o);
      }
    }
  }
}

typedef __attribute__((ext_vector_type(4))) unsigned u32x4_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

template <int DT, int V> __device__ __forceinline__ void unpack(const u32x4_t &r, float x[V]) {
  if constexpr (DT == SCHED_PD_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = __uint_as_float(r[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned w = r[i];
      if constexpr (DT == SCHED_PD_BF16) {
        x[2 * i] = __uint_as_float(w << 16);
        x[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
      } else {
        const f16x2_t h = __builtin_bit_cast(f16x2_t, w);
        x[2 * i] = (float)h.x;
        x[2 * i + 1] = (float)h.y;
      }
    }
  }
}

template <int DT, int V> __device__ __forceinline__ u32x4_t pack(const float x[V]) {
  u32x4_t r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == SCHED_PD_F32)
      r[i] = __float_as_uint(x[i]);
    else
      r[i] = DT == SCHED_PD_BF16 ? pack_bf16_rne(x[2 * i], x[2 * i + 1])
                                 : pack_f16_rne(x[2 * i], x[2 * i + 1]);
  }
  return r;
}

// N (2, 4 or 8) floats at p, 16-byte aligned (8-byte for two).
template <int N> __device__ __forceinline__ void load_f32(const float *p, float *x) {
  if constexpr (N == 2) {
    typedef __attribute__((ext_vector_type(2))) float f32x2_t;
    const f32x2_t v = *reinterpret_cast<const f32x2_t *>(p);
    x[0] = v.x, x[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const f32x4_t v = *reinterpret_cast<const f32x4_t *>(p + 4 * i);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        x[4 * i + k] = v[k];
    }
  }
}

// x of the lane that differs in bit HLG of its number, by VALU moves: quad permutes, row
// shifts with the banks that take them, a row rotation, the row swaps.
template <int HLG> __device__ __forceinline__ float xor_lane(float x) {
  const int i = __float_as_int(x);
  if constexpr (HLG == 0)
    return __int_as_float(__builtin_amdgcn_update_dpp(0, i, 0xB1, 0xF, 0xF, false));
  else if constexpr (HLG == 1)
    return __int_as_float(__builtin_amdgcn_update_dpp(0, i, 0x4E, 0xF, 0xF, false));
  else if constexpr (HLG == 2) { // banks 0, 2 from 4 lanes up, banks 1, 3 from 4 down
    const int a = __builtin_amdgcn_update_dpp(0, i, 0x104, 0xF, 0x5, false);
    return __int_as_float(__builtin_amdgcn_update_dpp(a, i, 0x114, 0xF, 0xA, false));
  } else if constexpr (HLG == 3)
    return __int_as_float(__builtin_amdgcn_update_dpp(0, i, 0x128, 0xF, 0xF, false));
  else if constexpr (HLG == 4) {
    const auto a = __builtin_amdgcn_permlane16_swap((unsigned)i, (unsigned)i, false, false);
    return __uint_as_float((threadIdx.x & 16u) ? a[0] : a[1]);
  } else {
    const auto a = __builtin_amdgcn_permlane32_swap((unsigned)i, (unsigned)i, false, false);
    return __uint_as_float((threadIdx.x & 32u) ? a[0] : a[1]);
  }
}

// The sum over the 2^LG lanes of a row, on every one of them.
template <int LG> __device__ __forceinline__ float row_sum(float x) {
  if constexpr (LG > 0)
    x += xor_lane<0>(x);
  if constexpr (LG > 1)
    x += xor_lane<1>(x);
  if constexpr (LG > 2)
    x += xor_lane<2>(x);
  if constexpr (LG > 3)
    x += xor_lane<3>(x);
  if constexpr (LG > 4)
    x += xor_lane<4>(x);
  if constexpr (LG > 5)
    x += xor_lane<5>(x);
  return x;
}

// How the vector kernel deals out rows: ts tokens' rows side by side fill the lane groups of
// gridDim.z workgroups; a lane group takes `per` such tokens of its row.
struct Deal {
  uint32_t ts, per;
  float inv_d;
};

// A lane group's tokens of a d-major V head: the lane's 16 bytes of a row go to as many rows
// as they have elements.
template <int EB>
__device__ __forceinline__ void values_apart(const RParams &P, const Span &S, const Deal &D,
                                             uint32_t h, uint32_t d0, uint32_t tsub, int64_t step) {
  typedef typename std::conditional<EB == 4, uint32_t, uint16_t>::type E;
  for (int64_t base = (int64_t)blockIdx.y * step; base < S.n; base += (int64_t)gridDim.y * step) {
    for (uint32_t k = 0; k < D.per; ++k) {
      const int64_t i = base + tsub + (int64_t)k * D.ts;
      if (i >= S.n)
        break;
      const int64_t pos = position_of(P, S.a0 + i);
      const u32x4_t x = *reinterpret_cast<const u32x4_t *>(
          static_cast<const char *>(P.v) + ((S.a0 + i) * P.v_ts + (int64_t)h * P.v_hs + d0) * EB);
      const Place at = place_of(P, S, i);
      if ((uint64_t)pos >= (uint64_t)P.max_pos || at.page < 0)
        continue;
      E *to = static_cast<E *>(P.vp) + at.page * P.vps + (int64_t)h * P.vhs + at.slot + d0 * P.vds;
#pragma unroll
      for (int e = 0; e < 16 / EB; ++e)
        to[e * P.vds] = (E)(x[e * EB / 4] >> (8 * (e * EB % 4)));
    }
  }
}

// Rows that 16-byte loads reach: 2^LG lanes hold a row (V elements each), so a wave holds
// 64 >> LG rows; the sum of squares and the exchange of the pairs' halves (HLG: lanes whose
// numbers differ in that bit hold them; -1: neighbouring pairs, within a lane) stay within
// a row's lanes, in VALU moves. A lane group keeps its row (its weights are loaded once)
// and walks over tokens, U of them at a time, the next ones' rows and positions on their
// way while these are turned.
template <int DT, int LG, int HLG, int U>
__global__ void __launch_bounds__(kBlock) rotary_vec(RParams P, Deal D) {
  constexpr bool INTER = HLG < 0;
  constexpr int V = DT == SCHED_PD_F32 ? 4 : 8; // elements of a lane
  constexpr int EB = DT == SCHED_PD_F32 ? 4 : 2;
  constexpr int NC = INTER ? V / 2 : V;         // angles of a lane
  constexpr uint32_t L = 1u << LG;
  const uint32_t tid = threadIdx.x, li = tid & (L - 1u);
  const uint32_t rows = P.Hq + P.Hkv + P.v_rows, half = P.rot / 2u, d0 = li * V;
  const uint32_t f = blockIdx.z * (kBlock >> LG) + (tid >> LG);
  const uint32_t tsub = f / rows, row = f - tsub * rows;
  const Span S = span_of(P, blockIdx.x);
  const int64_t step = (int64_t)D.ts * D.per;
  if ((int64_t)blockIdx.y * step >= S.n)
    return;
  const bool live = tsub < D.ts;
  const bool isq = row < P.Hq, isv = row >= P.Hq + P.Hkv;
  const uint32_t h = isq ? row : isv ? row - P.Hq - P.Hkv : row - P.Hq;
  const bool paged = !isq && P.kp != nullptr;
  const bool turned = !isv && d0 < P.rot, first = INTER || d0 < half;
  const void *w = isv ? nullptr : isq ? P.qw : P.kw;
  if (isv && P.vds != 1) {
    if (live)
      values_apart<EB>(P, S, D, h, d0, tsub, step);
    return; // (exchanges stay within a row's lanes)
  }
  float wt[V];
#pragma unroll
  for (int e = 0; e < V; ++e)
    wt[e] = 1.f;
  if (w != nullptr && live) {
    if (P.w_dtype == SCHED_PD_F32) {
      load_f32<V>(static_cast<const float *>(w) + d0, wt);
    } else {
      const uint2 *p = reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(w) + d0);
#pragma unroll
      for (int k = 0; k < V / 4; ++k) {
        const uint2 b = p[k];
        wt[4 * k] = half_w(P.w_dtype, b.x & 0xffffu);
        wt[4 * k + 1] = half_w(P.w_dtype, b.x >> 16);
        wt[4 * k + 2] = half_w(P.w_dtype, b.y & 0xffffu);
        wt[4 * k + 3] = half_w(P.w_dtype, b.y >> 16);
      }
    }
  }
  const char *src = static_cast<const char *>(isq ? P.q : isv ? P.v : P.k) +
                    ((int64_t)h * (isq ? P.q_hs : isv ? P.v_hs : P.k_hs) + d0) * EB;
  const int64_t src_ts = (isq ? P.q_ts : isv ? P.v_ts : P.k_ts) * EB;
  char *dst = static_cast<char *>(isq ? P.qo : !paged ? P.ko : isv ? P.vp : P.kp) +
              ((int64_t)h * (isq ? P.qo_hs : !paged ? P.ko_hs : isv ? P.vhs : P.khs) + d0) * EB;
  const int64_t dst_ts = (isq ? P.qo_ts : !paged ? P.ko_ts : isv ? P.vts : P.kts) * EB;
  const int64_t dst_ps = (isv ? P.vps : P.kps) * EB;
  const float *cs0 = P.cs + (INTER ? d0 / 2 : first ? d0 : d0 - half);

  for (int64_t base = (int64_t)blockIdx.y * step; base < S.n; base += (int64_t)gridDim.y * step) {
    // this group's tokens base + tsub + k ts, k < cnt
    const int64_t i0 = base + tsub, end = base + step < S.n ? base + step : S.n;
    const uint32_t cnt = live && i0 < end ? (uint32_t)((end - i0 + D.ts - 1) / D.ts) : 0u;
    const char *from = src + (S.a0 + i0) * src_ts;
    const int64_t hop = (int64_t)D.ts * src_ts;
    u32x4_t raw[U], nraw[U];
    int64_t pos[U], npos[U];
    auto fetch = [&](uint32_t k0) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k0 + u < cnt) {
          npos[u] = position_of(P, S.a0 + i0 + (int64_t)(k0 + u) * D.ts);
          nraw[u] = *reinterpret_cast<const u32x4_t *>(from);
        }
        from += hop;
      }
    };
    fetch(0);
    for (uint32_t k0 = 0; k0 < D.per; k0 += U) {
      float c[U][NC], sn[U][NC];
      char *to[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        raw[u] = nraw[u], pos[u] = npos[u];
        to[u] = nullptr;
        if (k0 + u >= cnt)
          continue;
        const int64_t i = i0 + (int64_t)(k0 + u) * D.ts;
        if ((uint64_t)pos[u] < (uint64_t)P.max_pos) {
          if (paged) {
            const Place at = place_of(P, S, i);
            if (at.page >= 0)
              to[u] = dst + at.page * dst_ps + at.slot * dst_ts;
            else if (P.errors && row == P.Hq && li == 0u)
              atomicAdd(P.errors, P.Hkv);
          } else {
            to[u] = dst + (S.a0 + i) * dst_ts;
          }
          if (turned) {
            const float *cs = cs0 + pos[u] * P.cs_stride;
            load_f32<NC>(cs, c[u]);
            load_f32<NC>(cs + half, sn[u]);
          }
        } else if (P.errors && row == 0u && li == 0u) {
          atomicAdd(P.errors, 1u);
        }
      }
      if (k0 + U < D.per)
        fetch(k0 + U);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[V];
        unpack<DT, V>(raw[u], x);
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e)
          ss += x[e] * x[e];
        ss = row_sum<LG>(ss);
        const float inv = w != nullptr ? rsqrtf(ss * D.inv_d + P.eps) : 1.f;
#pragma unroll
        for (int e = 0; e < V; ++e)
          x[e] *= inv * wt[e];
        if constexpr (INTER) {
          if (turned) {
#pragma unroll
            for (int e = 0; e < V; e += 2) {
              const float a = x[e], b = x[e + 1];
              x[e] = a * c[u][e / 2] - b * sn[u][e / 2];
              x[e + 1] = b * c[u][e / 2] + a * sn[u][e / 2];
            }
          }
        } else {
          float b[V];
#pragma unroll
          for (int e = 0; e < V; ++e)
            b[e] = xor_lane<HLG>(x[e]); // every lane takes part
          if (turned) {
#pragma unroll
            for (int e = 0; e < V; ++e)
              x[e] = x[e] * c[u][e] + (first ? -b[e] : b[e]) * sn[u][e];
          }
        }
        if (to[u] != nullptr)
          *reinterpret_cast<u32x4_t *>(to[u]) = isv ? raw[u] : pack<DT, V>(x);
      }
    }
  }
}

// The values of many tokens into a d-major cache: a tile of positions through LDS, read by
// rows and written in 16 bytes of a dim where all of its tokens go there. 8 prompts of up to
// 3000 tokens, 32 / 8 heads of 128 bf16, with the norm and rotation: 163 us; the values by
// element among the other rows 272; into a token-major cache 151.
template <int EB> __global__ void __launch_bounds__(kBlock) values_turned(RParams P) {
  typedef typename std::conditional<EB == 4, uint32_t, uint16_t>::type E;
  constexpr uint32_t TT = 128 / EB, TOK = 16 / EB, NG = TT / TOK;
  __shared__ __attribute__((aligned(4))) E s_row[TT][256 + 4 / EB];
  __shared__ int64_t s_to[TT];
  const uint32_t tid = threadIdx.x, h = blockIdx.z, units = P.d / TOK;
  const Span S = span_of(P, blockIdx.x);
  const int64_t start = S.ctx - S.n, lowest = start > 0 ? start / TT * TT : 0;
  const char *src = static_cast<const char *>(P.v) + (int64_t)h * P.v_hs * EB;
  char *dst = static_cast<char *>(P.vp) + (int64_t)h * P.vhs * EB;
  for (int64_t t0 = lowest + (int64_t)blockIdx.y * TT; t0 < S.ctx; t0 += (int64_t)gridDim.y * TT) {
    __syncthreads(); // the last tile's have been written
    if (tid < TT) {
      const int64_t i = t0 + tid - start;
      int64_t to = -1;
      if (i >= 0 && i < S.n) {
        const int64_t pos = position_of(P, S.a0 + i);
        const Place at = place_of(P, S, i);
        if ((uint64_t)pos < (uint64_t)P.max_pos && at.page >= 0)
          to = at.page * P.vps + at.slot;
      }
      s_to[tid] = to;
    }
    for (uint32_t u = tid; u < TT * units; u += kBlock) {
      const uint32_t k = u / units, c = u - k * units;
      const int64_t i = t0 + k - start;
      if (i >= 0 && i < S.n) {
        const char *from = src + (S.a0 + i) * P.v_ts * EB + 16u * c;
        const u32x4_t x = *reinterpret_cast<const u32x4_t *>(from);
        uint32_t *to = reinterpret_cast<uint32_t *>(&s_row[k][c * TOK]);
#pragma unroll
        for (int w = 0; w < 4; ++w)
          to[w] = x[w];
      }
    }
    __syncthreads();
    for (uint32_t p = tid; p < NG * P.d; p += kBlock) {
      const uint32_t k0 = p % NG * TOK, e = p / NG;
      char *row = dst + (int64_t)e * P.vds * EB;
      uint32_t w[4] = {0u, 0u, 0u, 0u};
      bool all = true;
#pragma unroll
      for (uint32_t t = 0; t < TOK; ++t) {
        all = all && s_to[k0 + t] >= 0;
        w[t * EB / 4] |= (uint32_t)s_row[k0 + t][e] << (8 * (t * EB % 4));
      }
      if (all) {
        *reinterpret_cast<u32x4_t *>(row + s_to[k0] * EB) = u32x4_t{w[0], w[1], w[2], w[3]};
      } else {
#pragma unroll
        for (uint32_t t = 0; t < TOK; ++t)
          if (s_to[k0 + t] >= 0)
            *reinterpret_cast<E *>(row + s_to[k0 + t] * EB) = s_row[k0 + t][e];
      }
    }
  }
}

typedef void (*VecFn)(RParams, Deal);

// A row's lanes (log2) and the lane bit that pairs' halves differ in (-1: none): full,
// half and quarter rotation of a head.
template <int DT, int LG, int U> VecFn vec_of(int hlg) {
  if (hlg < 0)
    return rotary_vec<DT, LG, -1, U>;
  if (hlg == LG - 1)
    return rotary_vec<DT, LG, LG - 1, U>;
  if (hlg == LG - 2)
    return rotary_vec<DT, LG, LG - 2, U>;
  if constexpr (LG >= 3)
    if (hlg == LG - 3)
      return rotary_vec<DT, LG, LG - 3, U>;
  return nullptr;
}

template <int DT, int U> VecFn vec_of(int lg, int hlg) {
  if (lg == 2)
    return vec_of<DT, 2, U>(hlg);
  if (lg == 3)
    return vec_of<DT, 3, U>(hlg);
  if (lg == 4)
    return vec_of<DT, 4, U>(hlg);
  if (lg == 5)
    return vec_of<DT, 5, U>(hlg);
  if constexpr (DT == SCHED_PD_F32)
    if (lg == 6)
      return vec_of<DT, 6, U>(hlg);
  return nullptr;
}

template <int U> VecFn vec_of(uint32_t dt, int lg, int hlg) {
  return dt == SCHED_PD_F32    ? vec_of<SCHED_PD_F32, U>(lg, hlg)
         : dt == SCHED_PD_BF16 ? vec_of<SCHED_PD_BF16, U>(lg, hlg)
                               : vec_of<SCHED_PD_F16, U>(lg, hlg);
}

int log2_of(uint32_t x) { // -1: not a power of two
  if (x == 0 || (x & (x - 1u)))
    return -1;
  int n = 0;
  while ((1u << n) < x)
    ++n;
  return n;
}

uint32_t esize(uint32_t dt) { return dt == SCHED_PD_F32 ? 4u : 2u; }

bool is_float(uint32_t dt) {
  return dt == SCHED_PD_F32 || dt == SCHED_PD_BF16 || dt == SCHED_PD_F16;
}

} // namespace

extern "C" {

void sched_rotary_default_args(SchedRotaryArgs *a) {
  if (!a)
    return;
  *a = SchedRotaryArgs{};
  a->abi_version = SCHED_ROTARY_ABI_VERSION;
  a->dtype = SCHED_PD_BF16;
  a->w_dtype = SCHED_PD_F32;
  a->eps = 1e-6f;
  a->vp_dim_stride = 1;
}

int sched_qk_norm_rope(const SchedRotaryArgs *a, void *stream) {
  if (!a)
    return set_error(-1, "sched_qk_norm_rope: args is NULL");
  if (a->abi_version != SCHED_ROTARY_ABI_VERSION)
    return set_error(-1, "sched_qk_norm_rope: abi_version %u, library has %u", a->abi_version,
                     SCHED_ROTARY_ABI_VERSION);
  if (!is_float(a->dtype) || !is_float(a->w_dtype))
    return set_error(-1, "sched_qk_norm_rope: dtypes %u, %u (F32, BF16 or F16)", a->dtype,
                     a->w_dtype);
  if (a->num_q_heads == 0 || a->num_kv_heads == 0 || a->num_q_heads > 65535u ||
      a->num_kv_heads > 65535u)
    return set_error(-1, "sched_qk_norm_rope: %u query and %u key heads", a->num_q_heads,
                     a->num_kv_heads);
  if (a->head_dim == 0 || a->head_dim % 4 || a->head_dim > 256)
    return set_error(-1, "sched_qk_norm_rope: head_dim %u (multiple of 4, <= 256)", a->head_dim);
  if (a->rot_dim < 2 || a->rot_dim % 2 || a->rot_dim > a->head_dim)
    return set_error(-1, "sched_qk_norm_rope: rot_dim %u (even, 2 .. head_dim %u)", a->rot_dim,
                     a->head_dim);
  if (!(a->eps >= 0.f))
    return set_error(-1, "sched_qk_norm_rope: eps %g", (double)a->eps);
  if (a->num_tokens > 0x7fffffffu)
    return set_error(-1, "sched_qk_norm_rope: num_tokens %u", a->num_tokens);
  const bool cache = a->k_pool != nullptr;
  if (a->num_tokens == 0 || (cache && a->num_requests == 0))
    return 0;
  if (!a->q || !a->k || !a->q_out || !a->positions || !a->cos_sin || a->max_pos == 0)
    return set_error(-1, "sched_qk_norm_rope: a required pointer is NULL (or max_pos 0)");
  if (!cache && !a->k_out)
    return set_error(-1, "sched_qk_norm_rope: needs k_out or a cache for the key rows");
  if (a->cs_stride < (int64_t)a->rot_dim)
    return set_error(-1, "sched_qk_norm_rope: cs_stride %lld for rot_dim %u",
                     (long long)a->cs_stride, a->rot_dim);
  if (cache) {
    if (!a->v || !a->v_pool || !a->append_indptr || !a->ctx_lens || !a->block_table)
      return set_error(-1, "sched_qk_norm_rope: a cache needs v, v_pool, append_indptr, "
                           "ctx_lens and block_table");
    if (a->page_size == 0 || a->num_pages == 0 || a->num_pages > 0x7fffffffull ||
        a->num_requests > 0x7fffffffu)
      return set_error(-1, "sched_qk_norm_rope: page_size %u, num_pages %llu", a->page_size,
                       (unsigned long long)a->num_pages);
    if (!a->page_indptr && a->bt_stride == 0)
      return set_error(-1, "sched_qk_norm_rope: bt_stride is 0 with a 2-D block table");
    if (a->vp_tok_stride != 1 && a->vp_dim_stride != 1)
      return set_error(-1, "sched_qk_norm_rope: V needs vp_tok_stride == 1 (d-major) or "
                           "vp_dim_stride == 1 (token-major)");
  }
  const uint32_t es = esize(a->dtype);
  for (const void *p : {a->q, a->k, a->v, (const void *)a->q_out, (const void *)a->k_out,
                        (const void *)a->k_pool, (const void *)a->v_pool})
    if ((uintptr_t)p % es)
      return set_error(-1, "sched_qk_norm_rope: a tensor is not aligned to its elements");

  RParams P{};
  P.q = a->q, P.k = a->k, P.v = a->v;
  P.q_ts = a->q_tok_stride, P.q_hs = a->q_head_stride;
  P.k_ts = a->k_tok_stride, P.k_hs = a->k_head_stride;
  P.v_ts = a->v_tok_stride, P.v_hs = a->v_head_stride;
  P.qo = a->q_out, P.ko = a->k_out;
  P.qo_ts = a->qo_tok_stride, P.qo_hs = a->qo_head_stride;
  P.ko_ts = a->ko_tok_stride, P.ko_hs = a->ko_head_stride;
  P.qw = a->q_weight, P.kw = a->k_weight;
  P.pos = a->positions, P.cs = a->cos_sin, P.cs_stride = a->cs_stride;
  P.errors = a->errors;
  P.T = a->num_tokens, P.Hq = a->num_q_heads, P.Hkv = a->num_kv_heads;
  P.d = a->head_dim, P.rot = a->rot_dim, P.max_pos = a->max_pos;
  P.w_dtype = a->w_dtype, P.inter = a->interleaved ? 1u : 0u, P.pos64 = a->pos_i64 ? 1u : 0u;
  P.eps = a->eps;
  if (cache) {
    P.kp = a->k_pool, P.vp = a->v_pool;
    P.kps = a->kp_page_stride, P.khs = a->kp_head_stride, P.kts = a->kp_tok_stride;
    P.vps = a->vp_page_stride, P.vhs = a->vp_head_stride, P.vts = a->vp_tok_stride;
    P.vds = a->vp_dim_stride;
    P.app = a->append_indptr, P.ctx = a->ctx_lens, P.table = a->block_table;
    P.pind = a->page_indptr, P.ps = a->page_size, P.bt_stride = a->bt_stride;
    P.num_pages = a->num_pages;
  }
  // a grid over (request, token), tokens striding past 65535
  uint32_t most = cache && a->max_append ? a->max_append : a->num_tokens;
  if (most > a->num_tokens)
    most = a->num_tokens;
  dim3 grid(cache ? a->num_requests : 1u, most < 65535u ? most : 65535u);
  hipStream_t s = static_cast<hipStream_t>(stream);
  // 16-byte pieces: whole in each row, aligned everywhere, pairs' halves in whole pieces
  const uint32_t v = 16u / es;
  auto pieces = [&](int64_t x) { return x % v == 0; };
  bool vec = a->head_dim % v == 0 && a->rot_dim % v == 0 && a->cs_stride % 4 == 0 &&
             (P.inter || (a->rot_dim / 2u) % v == 0) && (a->rot_dim / 2u) % 4 == 0 &&
             (uintptr_t)a->cos_sin % 16 == 0 && pieces(P.q_ts) && pieces(P.q_hs) &&
             pieces(P.k_ts) && pieces(P.k_hs) && pieces(P.qo_ts) && pieces(P.qo_hs);
  if (cache)
    vec = vec && pieces(P.v_ts) && pieces(P.v_hs) && pieces(P.kps) && pieces(P.khs) &&
          pieces(P.kts) &&
          (P.vds != 1 || (pieces(P.vps) && pieces(P.vhs) && pieces(P.vts)));
  else
    vec = vec && pieces(P.ko_ts) && pieces(P.ko_hs);
  for (const void *p : {a->q, a->k, cache ? a->v : nullptr, (const void *)a->q_out,
                        cache ? nullptr : (const void *)a->k_out, (const void *)a->k_pool,
                        (const void *)(cache && P.vds == 1 ? a->v_pool : nullptr)})
    vec = vec && (uintptr_t)p % 16 == 0;
  for (const void *p : {a->q_weight, a->k_weight})
    vec = vec && (uintptr_t)p % (a->w_dtype == SCHED_PD_F32 ? 16 : 8) == 0;
  VecFn fn = nullptr;
  Deal D{1u, 1u, 1.f / (float)a->head_dim};
  bool turn = false;
  P.v_rows = cache ? P.Hkv : 0u;
  if (vec) {
    uint32_t rows = P.Hq + P.Hkv + P.v_rows;
    const uint32_t groups = kBlock / (a->head_dim / v);
    auto across = [&](uint32_t t) { return (t * rows + groups - 1u) / groups; };
    // many tokens' values into a d-major cache: a launch of their own
    turn = cache && P.vds != 1 && P.ps % v == 0 && pieces(P.vps) && pieces(P.vhs) &&
           pieces(P.vds) && (uintptr_t)a->v_pool % 16 == 0 &&
           (uint64_t)P.T * across(1) >= kOneToken;
    if (turn)
      P.v_rows = 0u, rows -= P.Hkv;
    // as many tokens side by side, at most 8, as leave the fewest lane groups idle
    uint32_t ts = 1, best = ~0u;
    for (uint32_t t = 1; t <= 8; ++t) {
      const uint32_t idle = (across(t) * groups - t * rows) * 1000u / (across(t) * groups);
      if (idle < best)
        best = idle, ts = t;
    }
    const uint64_t work = (uint64_t)P.T * across(ts) / ts;
    const bool walk = work >= kOneToken;
    const int lg = log2_of(a->head_dim / v), hlg = P.inter ? -1 : log2_of(a->rot_dim / 2u / v);
    if (lg >= 0 && (P.inter || hlg >= 0))
      fn = walk ? vec_of<2>(a->dtype, lg, hlg) : vec_of<1>(a->dtype, lg, hlg);
    if (walk) {
      const uint64_t per = work / kFill;
      D.ts = ts;
      D.per = (uint32_t)(per < kLeastPer ? kLeastPer : per > kMostPer ? kMostPer : per) & ~1u;
    }
    if (fn) {
      grid.z = across(D.ts);
      const uint64_t gy = ((uint64_t)most + D.ts * D.per - 1u) / (D.ts * D.per);
      grid.y = (uint32_t)(gy < 65535u ? gy : 65535u);
    }
  }
  if (fn) {
    hipLaunchKernelGGL(fn, grid, dim3(kBlock), 0, s, P, D);
    if (turn) {
      const uint32_t tiles = (most + 128u / es - 1u) / (128u / es) + 1u;
      const dim3 over(a->num_requests, tiles < 65535u ? tiles : 65535u, P.Hkv);
      hipLaunchKernelGGL(es == 4 ? values_turned<4> : values_turned<2>, over, dim3(kBlock), 0, s,
                         P);
    }
  } else {
    P.v_rows = cache ? P.Hkv : 0u;
    auto every = a->dtype == SCHED_PD_F32    ? rotary_rows<SCHED_PD_F32>
                 : a->dtype == SCHED_PD_BF16 ? rotary_rows<SCHED_PD_BF16>
                                             : rotary_rows<SCHED_PD_F16>;
    hipLaunchKernelGGL(every, grid, dim3(kBlock), 0, s, P);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return set_error(-1, "sched_qk_norm_rope: launch failed: %s", hipGetErrorString(e));
  return 0;
}

} // extern "C"

// maps.h -- what the kernels of the decode with handed-on attention maps share
// (sched_decode_maps): the parameter block, how a task is cut into chunks, and
// where scores and partial results lie.
//
// A map row is one softmax: q-head g of a kv-head's group (weighted), or map a of
// q-head g as row 2g + a (difference). Per row the stream of a task's tokens gives
// the running maximum m and sum l of 2^s (s = score * log2(e) / scale) and the
// unnormalised products O = sum 2^(s - m) v. Chunks of a task join as
//   M = max m_c,  L = sum l_c 2^(m_c - M),  O = sum O_c 2^(m_c - M).
// The weights need every token's 2^(s - M) / L, which is known only when all of
// the task has been read: the stream leaves its scores behind in 32 bits, and the
// join turns them into weights.
#pragma once

#include "common.h"

namespace schedpd {

struct MapParams {
  const void *q;
  void *out;
  const void *k_pool, *v_pool;
  int64_t kps, khs, kts;
  int64_t vps, vhs, vts, vds;
  const float *k_scale, *v_scale;
  uint32_t scale_stride;
  const int32_t *bt, *indptr, *ctx;
  uint32_t R, Hq, Hkv, G, rows; // rows: maps per kv-head (G, or 2 G)
  uint32_t D, ps, bt_stride, max_pages, num_pages;
  uint32_t q_dtype, o_dtype;
  uint32_t nsplit, chunk; // most chunks of a task; tokens of one, about (map_chunk)
  uint32_t join_from;     // the join has tasks of more chunks than this to do
  float scale_log2;
  // weighted
  float *w;
  int64_t w_ps, w_hs;
  const int32_t *counted;
  float decay;
  uint32_t w_vec;      // four slots' weights are one 16-byte access
  float *scores;       // [16-token block of the batch][kv-head][row][16]
  uint64_t score_blocks; // blocks it holds
  // difference
  const float *lam, *nw;
  float eps, mul;
  // partials of chunk c of task t, item t * nsplit + c: (m, l) per row, O per row
  float *ml, *acc;
};

// A request's tokens: its context, as far as its table reaches.
__device__ __forceinline__ uint32_t map_tokens(const MapParams &P, uint32_t r) {
  const int32_t c = P.ctx[r];
  uint32_t pages = P.max_pages;
  if (P.indptr) {
    const int32_t have = P.indptr[r + 1] - P.indptr[r];
    pages = have > 0 ? (uint32_t)have : 0u;
  }
  const uint64_t cap = (uint64_t)pages * P.ps;
  return c <= 0 ? 0u : (uint64_t)c < cap ? (uint32_t)c : (uint32_t)cap;
}

__device__ __forceinline__ int64_t map_row(const MapParams &P, uint32_t r) {
  return P.indptr ? (int64_t)P.indptr[r] : (int64_t)r * P.bt_stride;
}

// Tokens of a chunk of an n-token task: all of them up to 3/2 P.chunk, else as many equal
// chunks as P.chunk tokens each would make; in multiples of 64.
__device__ __forceinline__ uint32_t map_chunk(const MapParams &P, uint32_t n) {
  const uint32_t nch = n <= P.chunk + P.chunk / 2u ? 1u : (n + P.chunk - 1u) / P.chunk;
  return ((n + nch - 1u) / nch + 63u) & ~63u;
}

// Score blocks of the requests before r (one wave or more; every lane takes part
// and gets the sum).
__device__ __forceinline__ uint64_t blocks_before(const MapParams &P, uint32_t r) {
  unsigned long long s = 0;
  for (uint32_t i = threadIdx.x & 63u; i < r; i += 64u)
    s += (map_tokens(P, i) + 15u) / 16u;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    s += __shfl_xor(s, o);
  return s;
}

// Score of row g, token i of a block: block blk of the request whose first block is b0.
__device__ __forceinline__ float *score_block(const MapParams &P, uint64_t b0, uint32_t blk,
                                              uint32_t h) {
  return P.scores + ((b0 + blk) * P.Hkv + h) * P.rows * 16u;
}

__device__ __forceinline__ void map_store(const MapParams &P, int64_t i, float v) {
  if (P.o_dtype == SCHED_PD_F32)
    static_cast<float *>(P.out)[i] = v;
  else if (P.o_dtype == SCHED_PD_F16)
    static_cast<_Float16 *>(P.out)[i] = (_Float16)v;
  else
    static_cast<uint16_t *>(P.out)[i] = f32_to_bf16_rne(v);
}

__device__ __forceinline__ float map_load_q(const MapParams &P, int64_t i) {
  return P.q_dtype == SCHED_PD_F32   ? static_cast<const float *>(P.q)[i]
         : P.q_dtype == SCHED_PD_F16 ? (float)static_cast<const _Float16 *>(P.q)[i]
                                     : bf16_bits_to_f32(static_cast<const uint16_t *>(P.q)[i]);
}

// The weights of four tokens t .. t + 3 of a request (t a multiple of 4): their scores at s
// (row g: s + 16 g floats), M and 1 / L of the rows in s_M, s_Li. Tokens from n on keep what
// their slots hold.
__device__ __forceinline__ void map_weights4(const MapParams &P, uint32_t h, uint32_t page,
                                             uint32_t t, uint32_t n, int64_t have,
                                             const float *s, const float *s_M,
                                             const float *s_Li) {
  typedef __attribute__((ext_vector_type(4))) float f32x4;
  float *wp = P.w + (int64_t)page * P.w_ps + (int64_t)h * P.w_hs + t % P.ps;
  f32x4 a = {0.f, 0.f, 0.f, 0.f}, old = {0.f, 0.f, 0.f, 0.f};
  const bool vec = P.w_vec && t + 4u <= n;
  if (vec) {
    if ((int64_t)t < have)
      old = *reinterpret_cast<const f32x4 *>(wp);
  } else {
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (t + k < n && (int64_t)(t + k) < have)
        old[k] = wp[k];
  }
#pragma unroll 4
  for (uint32_t g = 0; g < P.rows; ++g) {
    const f32x4 x = *reinterpret_cast<const f32x4 *>(s + g * 16u);
    const float M = s_M[g], li = s_Li[g];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      a[k] += __builtin_amdgcn_exp2f(x[k] - M) * li;
  }
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k)
    a[k] = (int64_t)(t + k) < have ? old[k] * P.decay + a[k] : a[k];
  if (vec) {
    *reinterpret_cast<f32x4 *>(wp) = a;
  } else {
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (t + k < n)
        wp[k] = a[k];
  }
}

} // namespace schedpd

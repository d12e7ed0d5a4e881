// maps_mfma.h -- the stream of sched_decode_maps on the CDNA4 matrix cores: fp32, 16-bit or
// fp8 e4m3fn caches, head dims 64, 128 and 256, either V layout, up to 16 map rows.
//
// The tiles are decode_mfma.h's (S^T = K Q^T over 16 tokens, then O^T += V^T P^T with the
// probabilities in place as the second product's operand); this kernel keeps what
// that one drops, the scores, and has its own epilogues:
// - weighted: a chunk's scores stay in LDS ([16-token block][row][16], 32 bits), so the
//   ring of cache loads is not held up by stores between them (one counter serves
//   both). A task that is one chunk turns them into weights right there; the chunks
//   of a longer one write them out for the join.
// - difference: row 2g + a holds q-head g's half a with the other half's dims zero: the
//   two maps are two columns of one product over the same K rows, and V is read once
//   for both. A task that is one chunk writes the normed difference itself.
//
// The probability operand carries p in two halves of the cache's type (bf16: 2^-17 of p;
// fp16: p scaled by 2^12 first, so that its tail stays above the subnormals: 2^-22 of p
// or 2^-37 at least). V of tokens past the context is selected to zero: 0 times what an
// unwritten slot holds would not be 0 if that is a NaN.
//
// fp32 caches keep fp32 all the way, through the fp32 matrix instruction (4 dims, or 4
// tokens, a step): a lane's 16 bytes of a key row are its dims of four steps, the lane's four
// probabilities the tokens 4 (lane / 16) + t of step t. Its 8 flops a byte are 50 TFLOP/s
// at the rate of the bytes, a third of what that instruction does.
//
// Bound by the cache's bytes. Measured: 64 requests of 2048 tokens, 32 / 8 heads of 128, bf16,
// weighted 87 us (6.3 TB/s; the plain decode 83); 48 of 200..2900, differential, 62 us (4.9);
// fp32, 64 of 1000 tokens, 3 kv-heads, differential 36 us (5.4); one request of 100003 in 64
// chunks 69 us (6.0), then 7 us of join.
#pragma once

#include "decode_mfma.h"
#include "maps.h"

namespace schedpd {

enum MapKv { kMapBf16, kMapF16, kMapFp8, kMapF32 };

// Registers of one 16-token block in flight.
template <int KV, int D> struct BlockRegs {
  static constexpr int EB = KV == kMapFp8 ? 1 : KV == kMapF32 ? 4 : 2;
  static constexpr int NK = D * EB / 64;         // 16-byte K loads of a lane
  static constexpr int NV = D * EB / 64;         // 16-byte V registers of a lane
  u32x4_t k[NK], v[NV];
  float ks, vs;
};

struct MapTask {
  uint32_t h, n, blk0, nblk, w; // blocks blk0 + w + NW i of the task are this wave's
  int64_t row;
  const uint8_t *kbase, *vbase; // the kv-head's
  int64_t kpage, vpage, ksub, vsub, k8, vstep; // bytes
  uint32_t klane, vlane;
  uint32_t per, magic; // blocks of a page; ceil(2^32 / per)
};

// A block's place: its page, and which 16 tokens of it.
struct MapBlock {
  uint32_t page, sub;
};

template <int KV, int D>
__device__ __forceinline__ void map_issue_k(const MapParams &P, const MapTask &T, MapBlock at,
                                            BlockRegs<KV, D> &B) {
  typedef BlockRegs<KV, D> R;
  const uint8_t *kp = T.kbase + at.page * T.kpage + (int64_t)at.sub * T.ksub;
  if constexpr (R::NK == 1) {
    B.k[0] = gload<true>(reinterpret_cast<const u32x4_t *>(kp + T.klane));
  } else {
    const uint8_t *kp8 = kp + T.k8;
#pragma unroll
    for (int i = 0; i < R::NK; ++i)
      B.k[i] = gload<true>(
          reinterpret_cast<const u32x4_t *>(((i & 1) ? kp8 : kp) + 128 * (i >> 1) + T.klane));
  }
  if constexpr (KV == kMapFp8) {
    const int64_t si = ((int64_t)at.page * P.Hkv + T.h) * P.scale_stride;
    B.ks = P.k_scale[si];
    B.vs = P.v_scale[si];
  }
}

template <int KV, int D, bool VT>
__device__ __forceinline__ void map_issue_v(const MapParams &P, const MapTask &T, MapBlock at,
                                            BlockRegs<KV, D> &B) {
  typedef BlockRegs<KV, D> R;
  const uint8_t *vp = T.vbase + at.page * T.vpage + (int64_t)at.sub * T.vsub;
  if constexpr (VT) {
    // the lane's dims of tokens 4 g4 + t: 4, 8 or 16 bytes a token, or two 16-byte
    // pieces 128 dims apart
    constexpr int LB = D / 16 * R::EB;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint8_t *a = vp + t * T.vstep + T.vlane;
      if constexpr (KV == kMapF32) { // 4 dims of each 64
#pragma unroll
        for (int g = 0; g < D / 64; ++g)
          B.v[4 * g + t] = gload<true>(reinterpret_cast<const u32x4_t *>(a + 256 * g));
      } else if constexpr (LB == 4) {
        B.v[0][t] = gload<true>(reinterpret_cast<const unsigned *>(a));
      } else if constexpr (LB == 8) {
        const u32x2_t x = gload<true>(reinterpret_cast<const u32x2_t *>(a));
        B.v[t >> 1][2 * (t & 1)] = x.x;
        B.v[t >> 1][2 * (t & 1) + 1] = x.y;
      } else {
        B.v[t] = gload<true>(reinterpret_cast<const u32x4_t *>(a));
        if constexpr (LB == 32)
          B.v[4 + t] = gload<true>(reinterpret_cast<const u32x4_t *>(a + 256));
      }
    }
  } else {
    // dim rows, several blocks of a page in one: ordinary loads, so that the lines one
    // wave fetched are still there for the next block's
#pragma unroll
    for (int i = 0; i < R::NV; ++i)
      B.v[i] = *reinterpret_cast<const u32x4_t *>(vp + i * T.vstep + T.vlane);
  }
}

template <int KV, int D> struct MapState {
  float m, l;
  f32x4_t acc[D / 16];
  u32x4_t q[KV == kMapF32 ? D / 16 : D / 32]; // the lane's dims of each step, or of four
};

// The A operand of dim block blk: 4 tokens of one dim. fp8 blocks come as one dword of
// four codes from `v8`.
template <int KV, int D, bool VT>
__device__ __forceinline__ s16x4_t map_v_operand(const u32x4_t *v, const unsigned *v8, int blk) {
  static_assert(KV != kMapF32, "fp32 values are operands as they are");
  if constexpr (KV == kMapFp8)
    return __builtin_bit_cast(s16x4_t, fp8x4_to_bf16x4(v8[blk]));
  else if constexpr (!VT)
    return __builtin_bit_cast(s16x4_t, (blk & 1) ? u32x2_t{v[blk >> 1].z, v[blk >> 1].w}
                                                 : u32x2_t{v[blk >> 1].x, v[blk >> 1].y});
  else if constexpr (D == 64)
    return vt_operand64(v, blk);
  else
    return bf16_vt_operand(v + 4 * (blk >> 3), blk & 7);
}

// The dim that output row rr (4 (lane / 16) + i) of dim block blk stands for.
template <int KV, int D, bool VT> __device__ __forceinline__ uint32_t map_dim(int blk, uint32_t rr) {
  if constexpr (!VT)
    return 16u * blk + rr;
  else if constexpr (KV == kMapF32)
    return 64u * (blk >> 2) + 4u * rr + (blk & 3);
  else if constexpr (KV != kMapFp8 && D == 256)
    return 128u * (blk >> 3) + 8u * rr + (blk & 7);
  else
    return D / 16 * rr + blk;
}

constexpr float kF16P = 4096.f; // fp16 probabilities travel times this

// One block: scores, then `next_k` (the block's keys are done with), then the softmax and
// the products.
template <int KV, int D, bool VT, bool DIFF, typename F>
__device__ __forceinline__ void map_compute(const MapParams &P, const MapTask &T, MapState<KV, D> &S,
                                            const BlockRegs<KV, D> &B, uint32_t blk_in_chunk,
                                            float *s_sc, uint32_t c16, uint32_t g4, F next_k) {
  typedef BlockRegs<KV, D> R;
  u32x4_t kk[R::NK];
#pragma unroll
  for (int i = 0; i < R::NK; ++i)
    kk[i] = B.k[i];
  if constexpr (R::NK > 1)
    k_operands(kk);
  f32x4_t sc = {0.f, 0.f, 0.f, 0.f};
  if constexpr (KV == kMapF32) {
    f32x4_t sd = {0.f, 0.f, 0.f, 0.f}; // two chains
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const unsigned k0 = kk[i][e], k1 = kk[i][e + 1], q0 = S.q[i][e], q1 = S.q[i][e + 1];
        sc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k0), __uint_as_float(q0), sc, 0, 0, 0);
        sd = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k1), __uint_as_float(q1), sd, 0, 0, 0);
      }
    sc += sd;
  }
#pragma unroll
  for (int kb = 0; kb < (KV == kMapF32 ? 0 : D / 32); ++kb) {
    bf16x8_t a;
    if constexpr (KV != kMapFp8) {
      a = __builtin_bit_cast(bf16x8_t, kk[kb]);
    } else {
      const u32x4_t raw = kk[kb >> 1];
      const u32x2_t lo = fp8x4_to_bf16x4((kb & 1) ? raw.z : raw.x);
      const u32x2_t hi = fp8x4_to_bf16x4((kb & 1) ? raw.w : raw.y);
      a = __builtin_bit_cast(bf16x8_t, u32x4_t{lo.x, lo.y, hi.x, hi.y});
    }
    sc = mfma_qk<KV == kMapF16>(a, __builtin_bit_cast(bf16x8_t, S.q[kb]), sc);
  }
  const float ks = KV == kMapFp8 ? P.scale_log2 * B.ks : P.scale_log2, vs = B.vs;
  next_k();
  // tokens of the block, counted from this lane's first
  const int left = (int)(T.n - (T.blk0 + blk_in_chunk) * 16u) - 4 * (int)g4;
  const bool full = T.n >= (T.blk0 + blk_in_chunk) * 16u + 16u;
  f32x4_t s;
#pragma unroll
  for (int v = 0; v < 4; ++v)
    s[v] = sc[v] * ks;
  if (!full) {
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (v >= left)
        s[v] = kNegInf;
  }
  if constexpr (!DIFF) {
    if (c16 < P.rows)
      *reinterpret_cast<f32x4_t *>(s_sc + (blk_in_chunk * P.rows + c16) * 16u + 4u * g4) = s;
  }
  const float mn = fmaxf(S.m, max_rows(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))));
  if (__builtin_amdgcn_ballot_w64(mn > S.m)) {
    const float c = __builtin_amdgcn_exp2f(S.m - mn);
    S.l *= c;
#pragma unroll
    for (int b = 0; b < D / 16; ++b)
      S.acc[b] *= c;
  }
  S.m = mn;
  float p[4];
#pragma unroll
  for (int v = 0; v < 4; ++v)
    p[v] = __builtin_amdgcn_exp2f(s[v] - mn);
  S.l += (p[0] + p[1]) + (p[2] + p[3]);
  u32x2_t hi = {0u, 0u}, lo = {0u, 0u};
  if constexpr (KV == kMapF32) {
    // p stays fp32
  } else if constexpr (KV == kMapF16) {
#pragma unroll
    for (int v = 0; v < 4; ++v)
      p[v] *= kF16P;
    // (a bit cast of a vector's element by name takes the vector's first: scalars)
    const unsigned w0 = pack_f16_rne(p[0], p[1]), w1 = pack_f16_rne(p[2], p[3]);
    const f16x2_t h0 = __builtin_bit_cast(f16x2_t, w0), h1 = __builtin_bit_cast(f16x2_t, w1);
    hi = u32x2_t{w0, w1};
    lo = u32x2_t{pack_f16_rne(p[0] - (float)h0.x, p[1] - (float)h0.y),
                 pack_f16_rne(p[2] - (float)h1.x, p[3] - (float)h1.y)};
  } else {
    if constexpr (KV == kMapFp8) {
#pragma unroll
      for (int v = 0; v < 4; ++v)
        p[v] *= vs;
    }
    hi = u32x2_t{pack_bf16_rne(p[0], p[1]), pack_bf16_rne(p[2], p[3])};
    lo = u32x2_t{pack_bf16_rne(p[0] - __uint_as_float(hi.x << 16),
                               p[1] - __uint_as_float(hi.x & 0xffff0000u)),
                 pack_bf16_rne(p[2] - __uint_as_float(hi.y << 16),
                               p[3] - __uint_as_float(hi.y & 0xffff0000u))};
  }
  const s16x4_t ph = __builtin_bit_cast(s16x4_t, hi), pl = __builtin_bit_cast(s16x4_t, lo);

  u32x4_t vv[R::NV];
#pragma unroll
  for (int i = 0; i < R::NV; ++i)
    vv[i] = B.v[i];
  if (!full) { // tokens past the context
    unsigned mt[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
      mt[t] = t < left ? ~0u : 0u;
    if constexpr (VT) {
      constexpr int LB = D / 16 * R::EB;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if constexpr (KV == kMapF32) {
#pragma unroll
          for (int g = 0; g < D / 64; ++g)
            vv[4 * g + t] &= mt[t];
        } else if constexpr (LB == 4) {
          vv[0][t] &= mt[t];
        } else if constexpr (LB == 8) {
          vv[t >> 1][2 * (t & 1)] &= mt[t];
          vv[t >> 1][2 * (t & 1) + 1] &= mt[t];
        } else {
          vv[t] &= mt[t];
          if constexpr (LB == 32)
            vv[4 + t] &= mt[t];
        }
      }
    }
  }
  unsigned v8[D / 16];
  if constexpr (KV == kMapFp8) {
    if constexpr (VT && D == 64)
      fp8_vt_transpose(vv[0].x, vv[0].y, vv[0].z, vv[0].w, v8);
    else if constexpr (VT && D == 128)
      fp8_vt_operands(vv, v8);
    else if constexpr (VT) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        fp8_vt_transpose(vv[0][q], vv[1][q], vv[2][q], vv[3][q], v8 + 4 * q);
    } else {
#pragma unroll
      for (int i = 0; i < R::NV; ++i) {
        v8[4 * i] = vv[i].x, v8[4 * i + 1] = vv[i].y;
        v8[4 * i + 2] = vv[i].z, v8[4 * i + 3] = vv[i].w;
        rows_transpose4(v8 + 4 * i);
      }
    }
  } else if constexpr (!VT && KV != kMapF32) {
    bf16_v_operands(vv);
  }
  if constexpr (!VT) {
    if (!full) { // each operand now holds the lane's own four tokens
      if constexpr (KV == kMapF32) {
        const u32x4_t m = {0 < left ? ~0u : 0u, 1 < left ? ~0u : 0u, 2 < left ? ~0u : 0u,
                           3 < left ? ~0u : 0u};
#pragma unroll
        for (int b = 0; b < R::NV; ++b)
          vv[b] &= m;
      } else if constexpr (KV == kMapFp8) {
        unsigned mk = 0u;
#pragma unroll
        for (int t = 0; t < 4; ++t)
          mk |= t < left ? 0xffu << (8 * t) : 0u;
#pragma unroll
        for (int b = 0; b < D / 16; ++b)
          v8[b] &= mk;
      } else {
        const unsigned m0 = (0 < left ? 0xffffu : 0u) | (1 < left ? 0xffff0000u : 0u);
        const unsigned m1 = (2 < left ? 0xffffu : 0u) | (3 < left ? 0xffff0000u : 0u);
#pragma unroll
        for (int i = 0; i < R::NV; ++i)
          vv[i] &= u32x4_t{m0, m1, m0, m1};
      }
    }
  }
#pragma unroll
  for (int b = 0; b < D / 16; ++b) {
    if constexpr (KV == kMapF32) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const unsigned v = VT ? vv[4 * (b >> 2) + t][b & 3] : vv[b][t];
        S.acc[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v), p[t], S.acc[b], 0, 0, 0);
      }
    } else {
      const s16x4_t a = map_v_operand<KV, D, VT>(vv, v8, b);
      S.acc[b] = mfma_pv<KV == kMapF16>(a, ph, S.acc[b]);
      S.acc[b] = mfma_pv<KV == kMapF16>(a, pl, S.acc[b]);
    }
  }
}

// A block's page id (scalar load, at a block of the task) and its place in the page. An
// id outside the pool reads some page of it: its request's rows mean nothing.
__device__ __forceinline__ MapBlock map_block(const MapParams &P, const MapTask &T, uint32_t blk) {
  typedef const __attribute__((address_space(4))) int32_t cint32;
  const uint32_t pg = T.per == 1u ? blk : __umulhi(blk, T.magic);
  const uint32_t id = (uint32_t)((const cint32 *)P.bt)[T.row + pg];
  return {id, blk - pg * T.per};
}
__device__ __forceinline__ MapBlock in_pool(const MapParams &P, MapBlock b) {
  return {min(b.page, P.num_pages - 1u), b.sub};
}

// The wave's blocks with DEPTH of them in flight, a block's keys reloaded as soon as its
// scores are there. Steady loop and tail as in decode_mfma.h: each computed block is
// followed by one block's loads, page ids come a ring ahead, and a short wave re-reads its
// last block into unused slots.
template <int KV, int D, bool VT, bool DIFF, int NW, int DEPTH>
__device__ __forceinline__ void map_stream(const MapParams &P, const MapTask &T, MapState<KV, D> &S,
                                           float *s_sc, uint32_t c16, uint32_t g4) {
  const int cnt = T.nblk > T.w ? (int)((T.nblk - T.w + NW - 1) / NW) : 0;
  if (cnt <= 0)
    return;
  const int last = cnt - 1;
  BlockRegs<KV, D> buf[DEPTH];
  MapBlock next[DEPTH];
  auto at = [&](int i) __attribute__((always_inline)) { return T.blk0 + T.w + NW * (uint32_t)i; };
#pragma unroll
  for (int s = 0; s < DEPTH; ++s) {
    const MapBlock b = in_pool(P, map_block(P, T, at(min(s, last))));
    next[s] = map_block(P, T, at(min(DEPTH + s, last)));
    map_issue_k<KV, D>(P, T, b, buf[s]);
    map_issue_v<KV, D, VT>(P, T, b, buf[s]);
  }
  int j = 0;
  for (; j + 2 * DEPTH <= cnt; j += DEPTH) {
#pragma unroll
    for (int s = 0; s < DEPTH; ++s) {
      const MapBlock b = in_pool(P, next[s]);
      map_compute<KV, D, VT, DIFF>(P, T, S, buf[s], T.w + NW * (uint32_t)(j + s), s_sc, c16, g4,
                                   [&]() __attribute__((always_inline)) {
                                     map_issue_k<KV, D>(P, T, b, buf[s]);
                                   });
      map_issue_v<KV, D, VT>(P, T, b, buf[s]);
      next[s] = map_block(P, T, at(min(j + 2 * DEPTH + s, last)));
    }
  }
  for (; j < cnt; j += DEPTH) {
#pragma unroll
    for (int s = 0; s < DEPTH; ++s) {
      if (j + s < cnt) {
        const bool more = j + DEPTH + s < cnt;
        const MapBlock b = in_pool(P, next[s]);
        map_compute<KV, D, VT, DIFF>(P, T, S, buf[s], T.w + NW * (uint32_t)(j + s), s_sc, c16, g4,
                                     [&]() __attribute__((always_inline)) {
                                       if (more)
                                         map_issue_k<KV, D>(P, T, b, buf[s]);
                                     });
        if (more)
          map_issue_v<KV, D, VT>(P, T, b, buf[s]);
      }
    }
  }
}

// GMAX: map rows the state in LDS is laid out for. The chunk's scores follow it in
// dynamic LDS (P.rows * 64 bytes a block; the host cuts chunks so that they fit).
template <int KV, int D, bool VT, int GMAX, bool DIFF, int NW, int DEPTH, int WPE>
__attribute__((amdgpu_waves_per_eu(WPE)))
__global__ void __launch_bounds__(NW * 64) maps_mfma(MapParams P) {
  constexpr uint32_t NT = NW * 64;
  constexpr int EB = BlockRegs<KV, D>::EB;
  __shared__ float s_acc[NW][GMAX][D];
  __shared__ float s_m[NW][GMAX], s_l[NW][GMAX];
  __shared__ float s_M[GMAX], s_Li[GMAX];
  extern __shared__ float s_sc[];
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t c16 = lane & 15u, g4 = lane >> 4;
  const uint32_t task = blockIdx.x, chunk = blockIdx.y;
  const uint32_t r = task / P.Hkv, h = task % P.Hkv;
  const uint32_t n = __builtin_amdgcn_readfirstlane(map_tokens(P, r)), len = map_chunk(P, n);
  const uint64_t first = (uint64_t)chunk * len;
  if (first >= n && chunk > 0u)
    return;
  const uint32_t t0 = (uint32_t)first, t1 = (uint32_t)(first + len < n ? first + len : n);

  MapTask T;
  T.h = h, T.n = t1, T.w = w;
  T.blk0 = t0 / 16u, T.nblk = (t1 - t0 + 15u) / 16u;
  T.row = P.indptr ? (int64_t)__builtin_amdgcn_readfirstlane(P.indptr[r])
                   : (int64_t)r * P.bt_stride;
  T.kbase = static_cast<const uint8_t *>(P.k_pool) + (int64_t)h * P.khs * EB;
  T.vbase = static_cast<const uint8_t *>(P.v_pool) + (int64_t)h * P.vhs * EB;
  T.kpage = P.kps * EB, T.vpage = P.vps * EB;
  T.ksub = 16 * P.kts * EB, T.k8 = 8 * P.kts * EB;
  const uint32_t krow = (uint32_t)(P.kts * EB);
  T.klane = BlockRegs<KV, D>::NK == 1 ? c16 * krow + 16u * g4
                                      : (c16 & 7u) * krow + 16u * g4 + 64u * (c16 >> 3);
  if constexpr (VT) {
    const uint32_t vrow = (uint32_t)(P.vts * EB);
    T.vsub = 16 * P.vts * EB, T.vstep = P.vts * EB;
    T.vlane = 4u * g4 * vrow + (D / 16 * EB > 16 ? 16u : D / 16 * EB) * c16;
  } else {
    const uint32_t vrow = (uint32_t)(P.vds * EB);
    T.vsub = 16 * EB, T.vstep = (KV == kMapFp8 ? 64 : KV == kMapF32 ? 16 : 32) * P.vds * EB;
    T.vlane = KV == kMapFp8   ? (c16 + 16u * g4) * vrow
              : KV == kMapF32 ? c16 * vrow + 16u * g4
                              : (c16 + 16u * (g4 & 1u)) * vrow + 16u * (g4 >> 1);
  }
  T.per = P.ps / 16u;
  T.magic = T.per == 1u ? 0u : 0xffffffffu / T.per + 1u;

  MapState<KV, D> S;
  S.m = kMInit, S.l = 0.f;
#pragma unroll
  for (int b = 0; b < D / 16; ++b)
    S.acc[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const uint32_t hq = h * P.G + (DIFF ? c16 >> 1 : c16);
#pragma unroll
  for (int i = 0; i < (KV == kMapF32 ? D / 16 : D / 32); ++i) {
    const uint32_t d0 = KV == kMapF32 ? 16u * i + 4u * g4 : qk_dim(KV == kMapFp8, i, g4);
    u32x4_t qv = {0u, 0u, 0u, 0u};
    if (c16 < P.rows && (!DIFF || (d0 >= D / 2) == ((c16 & 1u) != 0u)))
      qv = *reinterpret_cast<const u32x4_t *>(
          static_cast<const uint8_t *>(P.q) +
          (((int64_t)r * P.Hq + hq) * D + d0) * (KV == kMapF32 ? 4 : 2));
    S.q[i] = qv;
  }

  map_stream<KV, D, VT, DIFF, NW, DEPTH>(P, T, S, s_sc, c16, g4);

  const float lt = sum_rows(S.l);
  if (c16 < P.rows) {
    if (g4 == 0) {
      s_m[w][c16] = S.m;
      s_l[w][c16] = lt;
    }
#pragma unroll
    for (int b = 0; b < D / 16; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s_acc[w][c16][map_dim<KV, D, VT>(b, 4u * g4 + i)] =
            KV == kMapF16 ? S.acc[b][i] * (1.f / kF16P) : S.acc[b][i];
  }
  __syncthreads();
  const bool whole = len >= n; // the task is this chunk
  if (tid < P.rows) {
    float M = s_m[0][tid], L = 0.f;
#pragma unroll
    for (int k = 1; k < NW; ++k)
      M = fmaxf(M, s_m[k][tid]);
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const float e = __builtin_amdgcn_exp2f(s_m[k][tid] - M);
      L += s_l[k][tid] * e;
      s_m[k][tid] = e; // from here on: the wave's share of the row
    }
    s_M[tid] = M;
    s_Li[tid] = 1.f / L;
    if (!whole) {
      float *ml = P.ml + (((uint64_t)task * P.nsplit + chunk) * P.rows + tid) * 2u;
      ml[0] = M;
      ml[1] = L;
    }
  }
  __syncthreads();
  auto row_dim = [&](uint32_t g, uint32_t j) __attribute__((always_inline)) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k)
      a += s_acc[k][g][j] * s_m[k][g];
    return a;
  };
  if (!whole) {
    float *acc = P.acc + ((uint64_t)task * P.nsplit + chunk) * P.rows * D;
    for (uint32_t i = tid; i < P.rows * D; i += NT)
      acc[i] = row_dim(i / D, i % D);
    if constexpr (!DIFF) {
      const uint64_t b0 = blocks_before(P, r);
      const uint32_t per = P.rows * 4u; // float4s of a block
      for (uint32_t i = tid; i < T.nblk * per; i += NT) {
        const uint32_t b = i / per;
        if (b0 + T.blk0 + b < P.score_blocks)
          reinterpret_cast<f32x4_t *>(score_block(P, b0, T.blk0 + b, h))[i - b * per] =
              reinterpret_cast<const f32x4_t *>(s_sc)[i];
      }
    }
    return;
  }
  const float nan = __builtin_nanf("");
  if constexpr (DIFF) {
    // one q-head per wave at a time
    for (uint32_t g = w; g < P.G; g += NW) {
      const float la = P.lam[h * P.G + g];
      float o[D / 64], ss = 0.f;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const uint32_t j = lane + 64u * i;
        o[i] = row_dim(2u * g, j) * s_Li[2u * g] - la * (row_dim(2u * g + 1u, j) * s_Li[2u * g + 1u]);
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
        map_store(P, ((int64_t)r * P.Hq + h * P.G + g) * D + j,
                  n ? o[i] * inv * (P.nw ? P.nw[j] : 1.f) : nan);
      }
    }
  } else {
    for (uint32_t i = tid; i < P.rows * D; i += NT) {
      const uint32_t g = i / D, j = i % D;
      map_store(P, ((int64_t)r * P.Hq + h * P.G + g) * D + j, n ? row_dim(g, j) * s_Li[g] : nan);
    }
    const int64_t have = P.counted ? (int64_t)P.counted[r] : (int64_t)n;
    for (uint32_t t = tid * 4u; t < n; t += NT * 4u) {
      const uint32_t page = (uint32_t)P.bt[T.row + t / P.ps];
      if (page < P.num_pages)
        map_weights4(P, h, page, t, n, have, s_sc + (t / 16u) * P.rows * 16u + (t & 15u), s_M, s_Li);
    }
  }
}

} // namespace schedpd

// evict.hip -- eviction by accumulated attention weight (sched_kv_evict): per
// (request, kv-head) the m heaviest of n cached tokens stay, in their order, in slots
// 0 .. m-1. Two launches:
//   select: one workgroup per (request, kv-head) finds the weight T of the last kept
//           token by radix (the bits of a weight as an unsigned number that orders
//           like it, eight at a time from the top: a histogram, then the digit in which
//           the wanted rank falls), then walks the tokens once in order, keeping those
//           above T and the first ties;
//   move:   one workgroup per (request, kv-head, keys or values) copies the kept rows
//           down, a batch of rows at a time. A row's new slot is never behind its old
//           one, so a batch may be written once it and every batch before it have been read.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "common.h"
#include "rt_internal.h"
#include "sched_kv.h"

using namespace schedpd;

namespace {

struct EParams {
  uint8_t *k, *v;
  int64_t kps, khs, kts, vps, vhs, vts, vds; // elements
  float *ks, *vs;
  uint32_t scale_stride;
  const float *w;
  float *wo;
  int64_t w_ps, w_hs;
  const int32_t *bt, *indptr, *ctx, *keep;
  int32_t *kept;
  uint32_t *errors;
  float *new_scale; // fp8: [task][K, V][new_pages]
  uint32_t R, Hkv, D, ps, bt_stride, max_pages, max_keep, new_pages;
  uint32_t sink, recent;
  uint32_t num_pages;
};

struct Req {
  uint32_t n, m;
  int64_t row;
  bool ok; // the table holds the context
};

__device__ __forceinline__ Req req_of(const EParams &P, uint32_t r) {
  Req q;
  const int32_t c = P.ctx[r], k = P.keep[r];
  q.n = c > 0 ? (uint32_t)c : 0u;
  q.m = min(min(q.n, k > 0 ? (uint32_t)k : 0u), P.max_keep);
  q.row = P.indptr ? (int64_t)P.indptr[r] : (int64_t)r * P.bt_stride;
  const int64_t have = P.indptr ? (int64_t)P.indptr[r + 1] - P.indptr[r] : (int64_t)P.max_pages;
  q.ok = (int64_t)((q.n + (uint64_t)P.ps - 1u) / P.ps) <= have;
  return q;
}

// The bits of a weight as a number of the same order: -0 as +0, NaN below all.
__device__ __forceinline__ uint32_t order_bits(float f) {
  if (f != f)
    return 0u;
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kSelect = 1024;
constexpr int kVmcnt0 = 0x0F70; // s_waitcnt vmcnt(0), the other counters at their maxima

__global__ void __launch_bounds__(kSelect) evict_select(EParams P) {
  __shared__ uint32_t s_hist[256];
  __shared__ uint32_t s_wave[2][kSelect / 64];
  __shared__ uint32_t s_pick[2];
  __shared__ uint32_t s_bad;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t task = blockIdx.x, r = task / P.Hkv, h = task % P.Hkv;
  const Req q = req_of(P, r);
  int32_t *kept = P.kept + (int64_t)task * P.max_keep;
  if (tid == 0)
    s_bad = q.ok ? 0u : 1u;
  __syncthreads();
  const uint32_t pages = (uint32_t)((q.n + (uint64_t)P.ps - 1u) / P.ps);
  if (q.ok)
    for (uint32_t b = tid; b < pages; b += kSelect)
      if ((uint32_t)P.bt[q.row + b] >= P.num_pages)
        s_bad = 1u;
  __syncthreads();
  if (s_bad) { // nothing of this request is touched
    for (uint32_t j = tid; j < P.max_keep; j += kSelect)
      kept[j] = -1;
    if (tid == 0 && P.errors)
      atomicAdd(P.errors, 1u);
    return;
  }
  const uint32_t recent = min(q.m, P.recent), sink = min(P.sink, q.m - recent);
  const uint32_t lo = sink, hi = q.n - recent; // the tokens that compete
  const uint32_t want = q.m - recent - sink;
  auto weight = [&](uint32_t t) {
    return P.w[(int64_t)P.bt[q.row + t / P.ps] * P.w_ps + (int64_t)h * P.w_hs + t % P.ps];
  };
  // the want-th largest key, digit by digit; `left` of its equals are kept
  uint32_t T = 0u, left = 0u;
  if (q.m < q.n && want > 0u) {
    left = want;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256u)
        s_hist[tid] = 0u;
      __syncthreads();
      for (uint32_t t = lo + tid; t < hi; t += kSelect) {
        const uint32_t key = order_bits(weight(t));
        if (shift == 24 || (key >> (shift + 8)) == (T >> (shift + 8)))
          atomicAdd(&s_hist[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t d = 255u, above = 0u;
        while (d > 0u && above + s_hist[d] < left) {
          above += s_hist[d];
          --d;
        }
        s_pick[0] = d;
        s_pick[1] = above;
      }
      __syncthreads();
      T |= s_pick[0] << shift;
      left -= s_pick[1];
      __syncthreads();
    }
  }
  // one walk in order: the kept tokens' slots, and their weights moved along
  uint32_t base = 0u, ties = 0u;
  for (uint32_t t0 = 0; t0 < q.n; t0 += kSelect) {
    const uint32_t t = t0 + tid;
    float x = 0.f;
    bool always = false, above = false, tie = false;
    if (t < q.n) {
      x = weight(t);
      always = t < lo || t >= hi || q.m == q.n;
      if (!always && want > 0u) {
        const uint32_t key = order_bits(x);
        above = key > T;
        tie = key == T;
      }
    }
    // in place, another wave writes a slot of this stretch after the barriers below
    __builtin_amdgcn_s_waitcnt(kVmcnt0);
    const unsigned long long mt = __ballot(tie);
    if (lane == 0)
      s_wave[0][wave] = (uint32_t)__popcll(mt);
    __syncthreads();
    uint32_t before = ties + (uint32_t)__popcll(mt & ((1ull << lane) - 1ull)), all = 0u;
    for (uint32_t k = 0; k < kSelect / 64; ++k) {
      before += k < wave ? s_wave[0][k] : 0u;
      all += s_wave[0][k];
    }
    const bool in = always || above || (tie && before < left);
    const unsigned long long mk = __ballot(in);
    if (lane == 0)
      s_wave[1][wave] = (uint32_t)__popcll(mk);
    __syncthreads();
    uint32_t at = base + (uint32_t)__popcll(mk & ((1ull << lane) - 1ull)), some = 0u;
    for (uint32_t k = 0; k < kSelect / 64; ++k) {
      at += k < wave ? s_wave[1][k] : 0u;
      some += s_wave[1][k];
    }
    // every weight of this stretch has been read: a slot behind it is never written
    if (in && at < q.m) {
      kept[at] = (int32_t)t;
      if (t != at || P.wo != P.w)
        P.wo[(int64_t)P.bt[q.row + at / P.ps] * P.w_ps + (int64_t)h * P.w_hs + at % P.ps] = x;
    }
    base += some;
    ties += all;
    __syncthreads();
  }
  for (uint32_t j = q.m + tid; j < P.max_keep; j += kSelect)
    kept[j] = -1;
  // fp8: the new scales of the pages that hold the kept tokens
  if (P.new_scale != nullptr && q.m < q.n) {
    __syncthreads();
    float *ns = P.new_scale + (int64_t)task * 2 * P.new_pages;
    for (uint32_t b = tid; b * P.ps < q.m; b += kSelect) {
      float mk = 0.f, mv = 0.f;
      const uint32_t end = min(q.m, (b + 1u) * P.ps);
      for (uint32_t j = b * P.ps; j < end; ++j) {
        const int64_t si =
            ((int64_t)P.bt[q.row + (uint32_t)kept[j] / P.ps] * P.Hkv + h) * P.scale_stride;
        mk = fmaxf(mk, P.ks[si]);
        mv = fmaxf(mv, P.vs[si]);
      }
      ns[b] = mk;
      ns[P.new_pages + b] = mv;
    }
  }
}

// One e4m3 code from a page of scale s in a page of scale `to` (inv = 1 / to).
__device__ __forceinline__ uint32_t recode(uint32_t c, float s, float inv) {
  if ((c & 0x7fu) == 0x7fu)
    return c;
  const float x = fp8e4m3_to_f32(c) * s * inv;
  return encode2_fp8(x, 0.f) & 0xffu;
}

constexpr int kMove = 512;

// U: the unit a row is moved in (16 bytes where rows are contiguous and aligned, else
// one element); a row is `units` of them, unit_step bytes apart.
template <typename U, bool FP8>
__global__ void __launch_bounds__(kMove) evict_move(EParams P, uint32_t units, int64_t k_step,
                                                    int64_t v_step, uint32_t eb) {
  const uint32_t tid = threadIdx.x;
  const uint32_t task = blockIdx.x >> 1;
  const bool vals = (blockIdx.x & 1u) != 0u;
  const uint32_t r = task / P.Hkv, h = task % P.Hkv;
  const Req q = req_of(P, r);
  const int32_t *kept = P.kept + (int64_t)task * P.max_keep;
  if (q.m == q.n || q.m == 0u || kept[0] < 0)
    return;
  uint8_t *pool = vals ? P.v + (int64_t)h * P.vhs * eb : P.k + (int64_t)h * P.khs * eb;
  const int64_t ps_b = (vals ? P.vps : P.kps) * eb, ts_b = (vals ? P.vts : P.kts) * eb;
  const int64_t step = vals ? v_step : k_step;
  float *scale = vals ? P.vs : P.ks;
  const float *ns = P.new_scale + ((int64_t)task * 2 + (vals ? 1 : 0)) * P.new_pages;
  // kUnits units a lane and round
  constexpr int kUnits = 4;
  const uint64_t total = (uint64_t)q.m * units;
  for (uint64_t u0 = 0; u0 < total; u0 += (uint64_t)kMove * kUnits) {
    U x[kUnits];
    uint8_t *to[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const uint64_t u = u0 + (uint64_t)i * kMove + tid;
      to[i] = nullptr;
      if (u >= total)
        continue;
      const uint32_t j = (uint32_t)(u / units), e = (uint32_t)(u % units);
      const uint32_t src = (uint32_t)kept[j];
      const int64_t sp = P.bt[q.row + src / P.ps], dp = P.bt[q.row + j / P.ps];
      bool moves = src != j;
      float s = 0.f, inv = 0.f;
      if constexpr (FP8) {
        s = scale[(sp * P.Hkv + h) * P.scale_stride];
        const float n = ns[j / P.ps];
        if (s != n) {
          moves = true;
          inv = n > 0.f ? 1.f / n : 0.f;
        } else {
          s = 0.f; // the codes stay
        }
      }
      if (!moves)
        continue;
      x[i] = *reinterpret_cast<const U *>(pool + sp * ps_b + (int64_t)(src % P.ps) * ts_b +
                                          (int64_t)e * step);
      if constexpr (FP8) {
        if (s != 0.f || inv != 0.f) {
          U y = x[i];
          uint8_t *b = reinterpret_cast<uint8_t *>(&y);
          for (uint32_t k = 0; k < sizeof(U); ++k)
            b[k] = (uint8_t)recode(b[k], s, inv);
          x[i] = y;
        }
      }
      to[i] = pool + dp * ps_b + (int64_t)(j % P.ps) * ts_b + (int64_t)e * step;
    }
    __builtin_amdgcn_s_waitcnt(kVmcnt0);
    __syncthreads(); // this round's rows have all been read
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
      if (to[i] != nullptr)
        *reinterpret_cast<U *>(to[i]) = x[i];
  }
  if constexpr (FP8) {
    __syncthreads();
    for (uint32_t b = tid; b * P.ps < q.m; b += kMove)
      scale[((int64_t)P.bt[q.row + b] * P.Hkv + h) * P.scale_stride] = ns[b];
  }
}

uint32_t elem_bytes(uint32_t dt) {
  return dt == SCHED_PD_F32 ? 4u : dt == SCHED_PD_FP8_E4M3 ? 1u : 2u;
}

int check_shape(const SchedEvictArgs *a) {
  if (!a)
    return set_error(-1, "sched_kv_evict: args is NULL");
  if (a->abi_version != SCHED_EVICT_ABI_VERSION)
    return set_error(-1, "sched_kv_evict: abi_version %u, library has %u", a->abi_version,
                     SCHED_EVICT_ABI_VERSION);
  if (a->kv_dtype > SCHED_PD_F16)
    return set_error(-1, "sched_kv_evict: kv dtype %u", a->kv_dtype);
  if (a->num_kv_heads == 0 || (uint64_t)a->num_requests * a->num_kv_heads > (1u << 24))
    return set_error(-1, "sched_kv_evict: %u requests x %u kv-heads", a->num_requests,
                     a->num_kv_heads);
  if (a->head_dim == 0 || a->head_dim % 4 || a->head_dim > 256)
    return set_error(-1, "sched_kv_evict: head_dim %u (multiple of 4, <= 256)", a->head_dim);
  if (a->page_size == 0 || a->page_size % 4 || a->page_size > 256)
    return set_error(-1, "sched_kv_evict: page_size %u (multiple of 4, <= 256)", a->page_size);
  if (a->num_pages == 0 || a->num_pages > 0x7fffffffull)
    return set_error(-1, "sched_kv_evict: num_pages %llu", (unsigned long long)a->num_pages);
  if (a->max_keep > 0x7fffffffu)
    return set_error(-1, "sched_kv_evict: max_keep %u", a->max_keep);
  return 0;
}

uint32_t new_pages_of(const SchedEvictArgs *a) {
  return (uint32_t)(((uint64_t)a->max_keep + a->page_size - 1u) / a->page_size);
}

} // namespace

extern "C" {

void sched_evict_default_args(SchedEvictArgs *a) {
  if (!a)
    return;
  *a = SchedEvictArgs{};
  a->abi_version = SCHED_EVICT_ABI_VERSION;
  a->kv_dtype = SCHED_PD_BF16;
}

int64_t sched_kv_evict_workspace_bytes(const SchedEvictArgs *a) {
  if (check_shape(a))
    return -1;
  if (a->kv_dtype != SCHED_PD_FP8_E4M3)
    return 0;
  return (int64_t)((uint64_t)a->num_requests * a->num_kv_heads * 2u * new_pages_of(a) * 4u);
}

int sched_kv_evict(const SchedEvictArgs *a, void *stream) {
  if (int rc = check_shape(a))
    return rc;
  if (a->num_requests == 0)
    return 0;
  if (!a->k_pool || !a->v_pool || !a->weights || !a->weights_out || !a->block_table ||
      !a->ctx_lens || !a->keep_lens || (!a->kept && a->max_keep > 0))
    return set_error(-1, "sched_kv_evict: a required pointer is NULL");
  const bool fp8 = a->kv_dtype == SCHED_PD_FP8_E4M3;
  if (fp8 && (!a->k_scale || !a->v_scale))
    return set_error(-1, "sched_kv_evict: an fp8 cache needs k_scale and v_scale");
  if (!a->page_indptr && a->bt_stride < a->max_pages)
    return set_error(-1, "sched_kv_evict: bt_stride %u below max_pages %u", a->bt_stride,
                     a->max_pages);
  if (a->v_tok_stride != 1 && a->v_dim_stride != 1)
    return set_error(-1, "sched_kv_evict: V needs v_tok_stride == 1 (d-major) or v_dim_stride "
                         "== 1 (token-major)");
  const uint32_t eb = elem_bytes(a->kv_dtype);
  if ((uintptr_t)a->k_pool % eb || (uintptr_t)a->v_pool % eb)
    return set_error(-1, "sched_kv_evict: a pool is not aligned to its elements");
  const int64_t need = sched_kv_evict_workspace_bytes(a);
  if (need > 0 && (!a->workspace || a->workspace_bytes < (uint64_t)need ||
                   ((uintptr_t)a->workspace & 255u)))
    return set_error(-1, "sched_kv_evict: needs a 256-byte aligned workspace of %lld bytes (got "
                         "%llu)", (long long)need, (unsigned long long)a->workspace_bytes);
  EParams P{};
  P.k = static_cast<uint8_t *>(a->k_pool), P.v = static_cast<uint8_t *>(a->v_pool);
  P.kps = a->k_page_stride, P.khs = a->k_head_stride, P.kts = a->k_tok_stride;
  P.vps = a->v_page_stride, P.vhs = a->v_head_stride, P.vts = a->v_tok_stride;
  P.vds = a->v_dim_stride;
  if (fp8)
    P.ks = a->k_scale, P.vs = a->v_scale, P.new_scale = static_cast<float *>(a->workspace);
  P.scale_stride = (a->k_scale != nullptr && a->v_scale == a->k_scale + 1) ? 2u : 1u;
  P.w = a->weights, P.wo = a->weights_out;
  P.w_ps = a->w_page_stride, P.w_hs = a->w_head_stride;
  P.bt = a->block_table, P.indptr = a->page_indptr, P.ctx = a->ctx_lens, P.keep = a->keep_lens;
  P.kept = a->kept, P.errors = a->errors;
  P.R = a->num_requests, P.Hkv = a->num_kv_heads, P.D = a->head_dim, P.ps = a->page_size;
  P.bt_stride = a->bt_stride, P.max_pages = a->max_pages, P.max_keep = a->max_keep;
  P.new_pages = new_pages_of(a);
  P.sink = a->sink, P.recent = a->recent, P.num_pages = (uint32_t)a->num_pages;

  const uint32_t tasks = P.R * P.Hkv;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(evict_select, dim3(tasks), dim3(kSelect), 0, s, P);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a->max_keep > 0) {
    auto rows16 = [&](int64_t x) { return (x * eb) % 16 == 0; };
    const bool wide = a->v_dim_stride == 1 && (a->head_dim * eb) % 16 == 0 &&
                      (uintptr_t)a->k_pool % 16 == 0 && (uintptr_t)a->v_pool % 16 == 0 &&
                      rows16(P.kps) && rows16(P.khs) && rows16(P.kts) && rows16(P.vps) &&
                      rows16(P.vhs) && rows16(P.vts);
    const uint32_t units = wide ? a->head_dim * eb / 16u : a->head_dim;
    const int64_t k_step = wide ? 16 : eb, v_step = wide ? 16 : a->v_dim_stride * eb;
    const dim3 grid(2u * tasks), block(kMove);
    if (wide && fp8)
      hipLaunchKernelGGL((evict_move<uint4, true>), grid, block, 0, s, P, units, k_step, v_step, eb);
    else if (wide)
      hipLaunchKernelGGL((evict_move<uint4, false>), grid, block, 0, s, P, units, k_step, v_step, eb);
    else if (fp8)
      hipLaunchKernelGGL((evict_move<uint8_t, true>), grid, block, 0, s, P, units, k_step, v_step, eb);
    else if (eb == 2)
      hipLaunchKernelGGL((evict_move<uint16_t, false>), grid, block, 0, s, P, units, k_step, v_step, eb);
    else
      hipLaunchKernelGGL((evict_move<uint32_t, false>), grid, block, 0, s, P, units, k_step, v_step, eb);
    e = hipGetLastError();
  }
  if (e != hipSuccess)
    return set_error(-1, "sched_kv_evict: launch failed: %s", hipGetErrorString(e));
  return 0;
}

} // extern "C"

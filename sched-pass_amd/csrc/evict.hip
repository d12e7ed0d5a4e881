// evict.hip -- eviction by accumulated attention weight (sched_kv_evict): per
// (request, kv-head) the m heaviest of n cached tokens stay, in their order, in slots
// 0 .. m-1.
//   select: one workgroup per (request, kv-head) finds the weight T of the last kept
//           token by radix (the bits of a weight as an unsigned number that orders
//           like it, eight at a time from the highest that differ: a histogram, then the
//           digit in which the wanted rank falls), then keeps, in order, those above T
//           and the first ties. Its keys stay in registers, each weight is read once.
//   move:   one workgroup per (request, kv-head, keys or values, part of the row) copies
//           the kept rows down, a round of rows at a time. A row's new slot is never
//           behind its old one, so what a round overwrites are rows of its own or of
//           earlier rounds: it may be written once all of it has been read, with the next
//           round's reads already under way.
//   fp8: a third launch stores the pages' new scales, behind the last read of the old ones.
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
  uint32_t ps_magic; // ceil(2^32 / ps): t / ps for t up to 2^24
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

constexpr int kVmcnt0 = 0x0F70; // s_waitcnt vmcnt(0), the other counters at their maxima

__device__ __forceinline__ uint32_t div_ps(const EParams &P, uint32_t t) {
  return __umulhi(t, P.ps_magic);
}

// Inclusive sums of x over the workgroup's lanes in order; *all: the sum of all.
template <int NT>
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t *s_wave, uint32_t *all) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o);
    x += lane >= (uint32_t)o ? y : 0u;
  }
  __syncthreads(); // s_wave's previous values have been read
  if (lane == 63u)
    s_wave[wave] = x;
  __syncthreads();
  uint32_t before = 0u, sum = 0u;
#pragma unroll
  for (uint32_t k = 0; k < NT / 64; ++k) {
    before += k < wave ? s_wave[k] : 0u;
    sum += s_wave[k];
  }
  *all = sum;
  return x + before;
}

// The digit of s_hist (256 counts) in which the left-th largest falls, and how many lie
// above it; by the first wave, four digits a lane.
__device__ __forceinline__ void pick_digit(const uint32_t *s_hist, uint32_t left, uint32_t *s_pick) {
  const uint32_t lane = threadIdx.x;
  if (lane >= 64u)
    return;
  // lane 0 has the highest digits
  uint32_t c[4], sum = 0u;
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    c[k] = s_hist[255u - (4u * lane + k)];
    sum += c[k];
  }
  uint32_t incl = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(incl, o);
    incl += lane >= (uint32_t)o ? y : 0u;
  }
  uint32_t above = incl - sum;
  if (above < left && left <= incl) {
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      if (above < left && left <= above + c[k]) {
        s_pick[0] = 255u - (4u * lane + k);
        s_pick[1] = above;
        s_pick[2] = c[k];
      }
      above += c[k];
    }
  }
}

// NT lanes with KREG tokens each in registers, a stretch (its token t0 + i NT + lane). A
// request of one stretch is read once; a longer one stretch by stretch for each digit.
template <int NT, int KREG> __global__ void __launch_bounds__(NT) evict_select(EParams P) {
  constexpr uint32_t NW = NT / 64, SPAN = NT * KREG;
  constexpr uint32_t E = (KREG * NW + NT - 1) / NT; // counts of a lane in a scan
  static_assert(KREG <= 32, "a bit for each token of a lane");
  __shared__ uint32_t s_hist[256];
  __shared__ uint32_t s_cnt[KREG * NW];
  __shared__ uint32_t s_wave[NW], s_pick[3], s_lo[NW], s_hi[NW];
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
    for (uint32_t b = tid; b < pages; b += NT)
      if ((uint32_t)P.bt[q.row + b] >= P.num_pages)
        s_bad = 1u;
  __syncthreads();
  if (s_bad) { // nothing of this request is touched
    for (uint32_t j = tid; j < P.max_keep; j += NT)
      kept[j] = -1;
    if (tid == 0 && P.errors)
      atomicAdd(P.errors, 1u);
    return;
  }
  const uint32_t recent = min(q.m, P.recent), sink = min(P.sink, q.m - recent);
  const uint32_t lo = sink, hi = q.n - recent; // the tokens that compete
  const uint32_t want = q.m - recent - sink;
  const bool cut = q.m < q.n, one = q.n <= SPAN;
  const float *w0 = P.w + (int64_t)h * P.w_hs;

  float x[KREG];
  auto load = [&](uint32_t t0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < KREG; ++i) {
      const uint32_t t = t0 + (uint32_t)i * NT + tid;
      x[i] = 0.f;
      if (t < q.n) {
        const uint32_t b = div_ps(P, t);
        x[i] = w0[(int64_t)P.bt[q.row + b] * P.w_ps + (t - b * P.ps)];
      }
    }
  };
  load(0);
  uint32_t T = 0u, left = 0u;
  if (cut && want > 0u) {
    // the highest bit in which the competing keys differ
    uint32_t kmin = ~0u, kmax = 0u;
    for (uint32_t t0 = 0; t0 < q.n; t0 += SPAN) {
      if (t0 > 0u)
        load(t0);
#pragma unroll
      for (int i = 0; i < KREG; ++i) {
        const uint32_t t = t0 + (uint32_t)i * NT + tid;
        if (t >= lo && t < hi) {
          const uint32_t key = order_bits(x[i]);
          kmin = min(kmin, key);
          kmax = max(kmax, key);
        }
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      kmin = min(kmin, (uint32_t)__shfl_xor(kmin, o));
      kmax = max(kmax, (uint32_t)__shfl_xor(kmax, o));
    }
    if (lane == 0) {
      s_lo[wave] = kmin;
      s_hi[wave] = kmax;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < NW; ++k) {
      kmin = min(kmin, s_lo[k]);
      kmax = max(kmax, s_hi[k]);
    }
    const uint32_t differ = kmin ^ kmax;
    int top = differ ? 32 - __builtin_clz(differ) : 0; // the bits [0, top) differ
    T = top < 32 ? kmax >> top << top : 0u;
    left = want;
    while (top > 0) {
      const int shift = top > 8 ? top - 8 : 0;
      const uint32_t mask = (1u << (top - shift)) - 1u; // a digit of at most eight bits
      for (uint32_t k = tid; k < 256u; k += NT)
        s_hist[k] = 0u;
      __syncthreads();
      for (uint32_t t0 = 0; t0 < q.n; t0 += SPAN) {
        if (!one)
          load(t0);
#pragma unroll
        for (int i = 0; i < KREG; ++i) {
          if (t0 + (uint32_t)i * NT >= q.n)
            break;
          const uint32_t t = t0 + (uint32_t)i * NT + tid;
          const uint32_t key = order_bits(x[i]);
          if (t >= lo && t < hi && (top >= 32 || (key >> top) == (T >> top)))
            atomicAdd(&s_hist[(key >> shift) & mask], 1u);
        }
      }
      __syncthreads();
      pick_digit(s_hist, left, s_pick);
      __syncthreads();
      T |= s_pick[0] << shift;
      left -= s_pick[1];
      top = shift;
      // the whole digit is kept: everything from T on, whatever its lower bits
      if (s_pick[2] == left && T > 0u) {
        T -= 1u;
        left = 0u;
        top = 0;
      }
      __syncthreads();
    }
  }

  // exclusive sums, in token order, of the stretch's counts per (i, wave); returns their sum
  auto scan = [&](uint32_t t0) __attribute__((always_inline)) {
    __syncthreads();
    uint32_t c[E], sum = 0u, all;
#pragma unroll
    for (uint32_t k = 0; k < E; ++k) {
      const uint32_t e = tid * E + k;
      c[k] = e < KREG * NW && t0 + e / NW * NT < q.n ? s_cnt[e] : 0u;
      sum += c[k];
    }
    uint32_t at = block_scan<NT>(sum, s_wave, &all) - sum;
#pragma unroll
    for (uint32_t k = 0; k < E; ++k) {
      const uint32_t e = tid * E + k;
      if (e < KREG * NW)
        s_cnt[e] = at;
      at += c[k];
    }
    __syncthreads();
    return all;
  };
  uint32_t base = 0u, seen = 0u; // kept tokens and ties of the stretches before
  const unsigned long long below = (1ull << lane) - 1ull;
  for (uint32_t t0 = 0; t0 < q.n; t0 += SPAN) {
    if (!one)
      load(t0);
    uint32_t stay = 0u; // bit i: this lane's token i is kept
    if (cut && left > 0u) { // the first `left` tokens of weight T are
#pragma unroll
      for (int i = 0; i < KREG; ++i) {
        if (t0 + (uint32_t)i * NT >= q.n)
          break;
        const uint32_t t = t0 + (uint32_t)i * NT + tid;
        const unsigned long long b = __ballot(t >= lo && t < hi && order_bits(x[i]) == T);
        if (lane == 0)
          s_cnt[i * NW + wave] = (uint32_t)__popcll(b);
      }
      const uint32_t all = scan(t0);
#pragma unroll
      for (int i = 0; i < KREG; ++i) {
        if (t0 + (uint32_t)i * NT >= q.n)
          break;
        const uint32_t t = t0 + (uint32_t)i * NT + tid;
        const bool tie = t >= lo && t < hi && order_bits(x[i]) == T;
        const unsigned long long b = __ballot(tie);
        if (tie && seen + s_cnt[i * NW + wave] + (uint32_t)__popcll(b & below) < left)
          stay |= 1u << i;
      }
      seen += all;
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < KREG; ++i) {
      if (t0 + (uint32_t)i * NT >= q.n)
        break;
      const uint32_t t = t0 + (uint32_t)i * NT + tid;
      if (t < q.n && (!cut || t < lo || t >= hi || (want > 0u && order_bits(x[i]) > T)))
        stay |= 1u << i;
      const unsigned long long b = __ballot((stay >> i) & 1u);
      if (lane == 0)
        s_cnt[i * NW + wave] = (uint32_t)__popcll(b);
    }
    // in place: every lane has this stretch's weights before one is overwritten; those of
    // later stretches lie behind every slot that is written now
    __builtin_amdgcn_s_waitcnt(kVmcnt0);
    const uint32_t all = scan(t0);
#pragma unroll
    for (int i = 0; i < KREG; ++i) {
      if (t0 + (uint32_t)i * NT >= q.n)
        break;
      const uint32_t t = t0 + (uint32_t)i * NT + tid;
      const bool in = (stay >> i) & 1u;
      const unsigned long long b = __ballot(in);
      const uint32_t at = base + s_cnt[i * NW + wave] + (uint32_t)__popcll(b & below);
      if (in && at < q.m) {
        kept[at] = (int32_t)t;
        if (t != at || P.wo != P.w) {
          const uint32_t d = div_ps(P, at);
          P.wo[(int64_t)P.bt[q.row + d] * P.w_ps + (int64_t)h * P.w_hs + (at - d * P.ps)] = x[i];
        }
      }
    }
    base += all;
    __syncthreads();
  }
  for (uint32_t j = q.m + tid; j < P.max_keep; j += NT)
    kept[j] = -1;
  // fp8: the new scales of the pages that hold the kept tokens
  if (P.new_scale != nullptr && cut) {
    __builtin_amdgcn_s_waitcnt(kVmcnt0);
    __syncthreads();
    float *ns = P.new_scale + (int64_t)task * 2 * P.new_pages;
    for (uint32_t b = tid; b * P.ps < q.m; b += NT) {
      float mk = 0.f, mv = 0.f;
      const uint32_t end = min(q.m, (b + 1u) * P.ps);
      for (uint32_t j = b * P.ps; j < end; ++j) {
        const int64_t si =
            ((int64_t)P.bt[q.row + div_ps(P, (uint32_t)kept[j])] * P.Hkv + h) * P.scale_stride;
        mk = fmaxf(mk, P.ks[si]);
        mv = fmaxf(mv, P.vs[si]);
      }
      ns[b] = mk;
      ns[P.new_pages + b] = mv;
    }
  }
}

// Makes the compiler wait for a load into x here.
__device__ __forceinline__ void hold(uint4 &x) {
  asm volatile("" : "+v"(x.x), "+v"(x.y), "+v"(x.z), "+v"(x.w) : : "memory");
}
__device__ __forceinline__ void hold(uint32_t &x) { asm volatile("" : "+v"(x) : : "memory"); }
__device__ __forceinline__ void hold(uint16_t &x) { asm volatile("" : "+v"(x) : : "memory"); }
__device__ __forceinline__ void hold(uint8_t &x) {
  uint32_t y = x;
  asm volatile("" : "+v"(y) : : "memory");
  x = (uint8_t)y;
}

// One e4m3 code from a page of scale s in a page of scale `to` (inv = 1 / to).
__device__ __forceinline__ uint32_t recode(uint32_t c, float s, float inv) {
  if ((c & 0x7fu) == 0x7fu)
    return c;
  const float x = fp8e4m3_to_f32(c) * s * inv;
  return encode2_fp8(x, 0.f) & 0xffu;
}

constexpr int kMove = 512;
constexpr uint32_t kStage = 2048; // rows whose places are in LDS at a time

// U: the unit a row is moved in (16 bytes where rows are contiguous and aligned, else
// one element); a row is `units` of them, k_step / v_step bytes apart, `part` of them this
// workgroup's.
template <typename U, bool FP8>
__global__ void __launch_bounds__(kMove) evict_move(EParams P, uint32_t units, uint32_t part,
                                                    int64_t k_step, int64_t v_step, uint32_t eb) {
  constexpr int N = 4; // units of a lane and round
  // where a row comes from (-1: it stays) and goes to; fp8: its old scale, the new one's inverse
  __shared__ int64_t s_from[kStage], s_to[kStage];
  __shared__ float s_old[FP8 ? kStage : 1], s_inv[FP8 ? kStage : 1];
  const uint32_t tid = threadIdx.x, tasks2 = 2u * P.R * P.Hkv;
  const uint32_t which = blockIdx.x % tasks2, first = blockIdx.x / tasks2 * part;
  const uint32_t task = which >> 1;
  const bool vals = (which & 1u) != 0u;
  const uint32_t r = task / P.Hkv, h = task % P.Hkv;
  const Req q = req_of(P, r);
  const int32_t *kept = P.kept + (int64_t)task * P.max_keep;
  if (q.m == q.n || q.m == 0u || kept[0] < 0)
    return;
  uint8_t *pool = vals ? P.v + (int64_t)h * P.vhs * eb : P.k + (int64_t)h * P.khs * eb;
  const int64_t ps_b = (vals ? P.vps : P.kps) * eb, ts_b = (vals ? P.vts : P.kts) * eb;
  const float *scale = vals ? P.vs : P.ks;
  const float *ns = P.new_scale + ((int64_t)task * 2 + (vals ? 1 : 0)) * P.new_pages;
  const uint32_t e = first + tid % part, rr = tid / part, rows = kMove / part;
  const bool active = rr < rows && e < units;
  const int64_t off = (int64_t)e * (vals ? v_step : k_step);
  const uint32_t round = rows * N;

  for (uint32_t j0 = 0; j0 < q.m; j0 += kStage) {
    const uint32_t cnt = min(kStage, q.m - j0);
    __syncthreads(); // the previous stage's places have been used
    for (uint32_t i = tid; i < cnt; i += kMove) {
      const uint32_t j = j0 + i, src = (uint32_t)kept[j];
      const uint32_t sb = div_ps(P, src), db = div_ps(P, j);
      const int64_t sp = P.bt[q.row + sb], dp = P.bt[q.row + db];
      bool moves = src != j;
      if constexpr (FP8) {
        const float was = scale[(sp * P.Hkv + h) * P.scale_stride], now = ns[db];
        s_old[i] = was;
        s_inv[i] = was != now ? 1.f / now : 0.f; // 0: the codes stay
        moves = moves || was != now;
      }
      s_from[i] = moves ? sp * ps_b + (int64_t)(src - sb * P.ps) * ts_b : -1;
      s_to[i] = dp * ps_b + (int64_t)(j - db * P.ps) * ts_b;
    }
    __syncthreads();
    U x[N], nx[N];
    auto fetch = [&](uint32_t k0) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t k = k0 + (uint32_t)i * rows + rr;
        nx[i] = U{};
        if (active && k < cnt) {
          const int64_t from = s_from[k];
          if (from >= 0)
            nx[i] = *reinterpret_cast<const U *>(pool + from + off);
        }
      }
    };
    fetch(0);
    for (uint32_t k0 = 0; k0 < cnt; k0 += round) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        x[i] = nx[i];
      if (k0 + round < cnt)
        fetch(k0 + round);
      // this round's rows are in registers on every lane before any of them is written: each
      // lane waits for its own here (the next round's stay under way), then the barrier
#pragma unroll
      for (int i = 0; i < N; ++i)
        hold(x[i]);
      asm volatile("s_barrier" ::: "memory");
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t k = k0 + (uint32_t)i * rows + rr;
        if (active && k < cnt && s_from[k] >= 0) {
          if constexpr (FP8) {
            const float inv = s_inv[k];
            if (inv != 0.f) {
              const float was = s_old[k];
              uint8_t *b = reinterpret_cast<uint8_t *>(&x[i]);
#pragma unroll
              for (uint32_t c = 0; c < sizeof(U); ++c)
                b[c] = (uint8_t)recode(b[c], was, inv);
            }
          }
          *reinterpret_cast<U *>(pool + s_to[k] + off) = x[i];
        }
      }
    }
  }
}

// fp8: the new scales, once no move reads the old ones.
__global__ void __launch_bounds__(256) evict_scales(EParams P) {
  const uint32_t task = blockIdx.x, r = task / P.Hkv, h = task % P.Hkv;
  const Req q = req_of(P, r);
  if (q.m == q.n || q.m == 0u || P.kept[(int64_t)task * P.max_keep] < 0)
    return;
  const float *ns = P.new_scale + (int64_t)task * 2 * P.new_pages;
  for (uint32_t b = threadIdx.x; b * P.ps < q.m; b += 256u) {
    const int64_t si = ((int64_t)P.bt[q.row + b] * P.Hkv + h) * P.scale_stride;
    P.ks[si] = ns[b];
    P.vs[si] = ns[P.new_pages + b];
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
  if ((uint64_t)a->max_pages * a->page_size > (1u << 24))
    return set_error(-1, "sched_kv_evict: tables of %u pages of %u tokens (at most 2^24 tokens)",
                     a->max_pages, a->page_size);
  if (a->max_keep > 0x7fffffffu)
    return set_error(-1, "sched_kv_evict: max_keep %u", a->max_keep);
  return 0;
}

// Workgroups of the move that fill the card.
constexpr uint32_t kMoveFill = 512;

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

  P.ps_magic = 0xffffffffu / P.ps + 1u;

  const uint32_t tasks = P.R * P.Hkv;
  const uint64_t longest = (uint64_t)a->max_pages * a->page_size;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (longest <= 256u * 16u)
    hipLaunchKernelGGL((evict_select<256, 16>), dim3(tasks), dim3(256), 0, s, P);
  else
    hipLaunchKernelGGL((evict_select<1024, 32>), dim3(tasks), dim3(1024), 0, s, P);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a->max_keep > 0) {
    auto rows16 = [&](int64_t x) { return (x * eb) % 16 == 0; };
    const bool wide = a->v_dim_stride == 1 && (a->head_dim * eb) % 16 == 0 &&
                      (uintptr_t)a->k_pool % 16 == 0 && (uintptr_t)a->v_pool % 16 == 0 &&
                      rows16(P.kps) && rows16(P.khs) && rows16(P.kts) && rows16(P.vps) &&
                      rows16(P.vhs) && rows16(P.vts);
    const uint32_t units = wide ? a->head_dim * eb / 16u : a->head_dim;
    const int64_t k_step = wide ? 16 : eb, v_step = wide ? 16 : a->v_dim_stride * eb;
    // few tasks: a row in up to four parts, of 64 bytes at least, for more workgroups
    uint32_t parts = 1;
    while (wide && parts < 4u && 2u * tasks * parts < kMoveFill && units / (2u * parts) >= 4u)
      parts *= 2u;
    const uint32_t part = (units + parts - 1u) / parts;
    const dim3 grid(2u * tasks * parts), block(kMove);
    if (wide && fp8)
      hipLaunchKernelGGL((evict_move<uint4, true>), grid, block, 0, s, P, units, part, k_step, v_step, eb);
    else if (wide)
      hipLaunchKernelGGL((evict_move<uint4, false>), grid, block, 0, s, P, units, part, k_step, v_step, eb);
    else if (fp8)
      hipLaunchKernelGGL((evict_move<uint8_t, true>), grid, block, 0, s, P, units, part, k_step, v_step, eb);
    else if (eb == 2)
      hipLaunchKernelGGL((evict_move<uint16_t, false>), grid, block, 0, s, P, units, part, k_step, v_step, eb);
    else
      hipLaunchKernelGGL((evict_move<uint32_t, false>), grid, block, 0, s, P, units, part, k_step, v_step, eb);
    e = hipGetLastError();
    if (e == hipSuccess && fp8) {
      hipLaunchKernelGGL(evict_scales, dim3(tasks), dim3(256), 0, s, P);
      e = hipGetLastError();
    }
  }
  if (e != hipSuccess)
    return set_error(-1, "sched_kv_evict: launch failed: %s", hipGetErrorString(e));
  return 0;
}

} // extern "C"

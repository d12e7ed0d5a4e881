// evict.hip -- eviction by accumulated attention weight (sched_kv_evict): per
// (request, kv-head) the m heaviest of n cached tokens stay, in their order, in slots
// 0 .. m-1.
//   select: one workgroup per (request, kv-head) finds the weight T of the last kept
//           token by radix (the bits of a weight as an unsigned number that orders
//           like it, eight at a time from the highest that differ: a histogram, then the
//           digit in which the wanted rank falls), then keeps, in order, those above T
//           and the first ties. Its keys stay in registers, each weight is read once.
//           Few long requests: a launch per step, many workgroups a task.
//   move:   one workgroup per (request, kv-head, keys or values) copies
//           the kept rows down, a round of rows at a time. A row's new slot is never
//           behind its old one, so what a round overwrites are rows of its own or of
//           earlier rounds: it may be written once all of it has been read, with the next
//           round's reads already under way. Few tasks: chunks of rows on many workgroups.
//   fp8: a third launch stores the pages' new scales, behind the last read of the old ones.
// Bound by the moved bytes, and for few tasks by the launches behind each other. Measured,
// bf16, 8 kv-heads of 128: 32 requests of 2048, half kept, 78 us (selection 18, moves 60: 4.5
// TB/s); one of 65537, an eighth kept, 51 us (selection 34 in six launches, moves 16).
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
  uint32_t row_groups; // evict_move: workgroups that move rows (then those of saved weights)
  // the wide selection: per task three histograms, whether its table is bad, and per chunk
  // its kept tokens and ties
  uint32_t *wide, chunks;
  float *saved; // the wide selection's kept weights, [task][most_kept]
  uint32_t most_kept, save_chunks;
  // evict_move_few: per task and tensor a ticket and a flag for each of its chunks
  uint32_t *moves, move_chunks;
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

// evict_move_few's tickets and flags of a task's keys and values, none taken or set.
__device__ __forceinline__ void clear_moves(const EParams &P, uint32_t task, uint32_t nt) {
  if (P.moves == nullptr)
    return;
  const uint32_t each = 1u + P.move_chunks;
  for (uint32_t k = threadIdx.x; k < 2u * each; k += nt)
    P.moves[(uint64_t)task * 2u * each + k] = 0u;
}

// Histograms come in kCopies, a lane's by its number: weights share their exponents, and
// one counter serves one lane at a time.
constexpr uint32_t kCopies = 8;

// The digit of s_hist (256 counts) in which the left-th largest falls, and how many lie
// above it; by the first wave, four digits a lane.
__device__ __forceinline__ void pick_digit(const uint32_t (*s_hist)[256], uint32_t left,
                                           uint32_t *s_pick) {
  const uint32_t lane = threadIdx.x;
  if (lane >= 64u)
    return;
  // lane 0 has the highest digits
  uint32_t c[4], sum = 0u;
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    c[k] = 0u;
#pragma unroll
    for (uint32_t p = 0; p < kCopies; ++p)
      c[k] += s_hist[p][255u - (4u * lane + k)];
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

// The kept tokens of a stretch in order: NT lanes with KREG tokens each, x their weights (token
// t0 + i NT + lane). Those outside [lo, hi) stay, of the others those whose key is above T
// and the first `left` of key T; *base and *seen are the kept tokens and the ties before
// the stretch, and go on. Their weights go to `saved`, or with WEIGHTS move along (in place: every lane has the
// stretch's before one is overwritten, and those of later stretches lie behind every slot
// that is written here).
template <int NT, int KREG, bool WEIGHTS>
__device__ __forceinline__ void keep_stretch(const EParams &P, const Req &q, uint32_t h,
                                             const float (&x)[KREG], uint32_t t0, uint32_t lo,
                                             uint32_t hi, uint32_t want, uint32_t T,
                                             uint32_t left, int32_t *kept, float *saved,
                                             uint32_t *s_cnt, uint32_t *s_wave, uint32_t *base,
                                             uint32_t *seen) {
  constexpr uint32_t NW = NT / 64;
  constexpr uint32_t E = (KREG * NW + NT - 1) / NT; // counts of a lane in a scan
  static_assert(KREG <= 32, "a bit for each token of a lane");
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const bool cut = q.m < q.n;
  const unsigned long long below = (1ull << lane) - 1ull;
  // exclusive sums, in token order, of the counts per (i, wave); returns their sum
  auto scan = [&]() __attribute__((always_inline)) {
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
  uint32_t stay = 0u; // bit i: this lane's token i is kept
  if (cut && left > 0u) {
#pragma unroll
    for (int i = 0; i < KREG; ++i) {
      if (t0 + (uint32_t)i * NT >= q.n)
        break;
      const uint32_t t = t0 + (uint32_t)i * NT + tid;
      const unsigned long long b = __ballot(t >= lo && t < hi && order_bits(x[i]) == T);
      if (lane == 0)
        s_cnt[i * NW + wave] = (uint32_t)__popcll(b);
    }
    const uint32_t all = scan();
#pragma unroll
    for (int i = 0; i < KREG; ++i) {
      if (t0 + (uint32_t)i * NT >= q.n)
        break;
      const uint32_t t = t0 + (uint32_t)i * NT + tid;
      const bool tie = t >= lo && t < hi && order_bits(x[i]) == T;
      const unsigned long long b = __ballot(tie);
      if (tie && *seen + s_cnt[i * NW + wave] + (uint32_t)__popcll(b & below) < left)
        stay |= 1u << i;
    }
    *seen += all;
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
  __builtin_amdgcn_s_waitcnt(kVmcnt0);
  const uint32_t all = scan();
#pragma unroll
  for (int i = 0; i < KREG; ++i) {
    if (t0 + (uint32_t)i * NT >= q.n)
      break;
    const uint32_t t = t0 + (uint32_t)i * NT + tid;
    const bool in = (stay >> i) & 1u;
    const unsigned long long b = __ballot(in);
    const uint32_t at = *base + s_cnt[i * NW + wave] + (uint32_t)__popcll(b & below);
    if (in && at < q.m) {
      kept[at] = (int32_t)t;
      if (!WEIGHTS)
        saved[at] = x[i];
      if (WEIGHTS && (t != at || P.wo != P.w)) {
        const uint32_t d = div_ps(P, at);
        P.wo[(int64_t)P.bt[q.row + d] * P.w_ps + (int64_t)h * P.w_hs + (at - d * P.ps)] = x[i];
      }
    }
  }
  *base += all;
  __syncthreads();
}

// fp8: the new scales of the pages that will hold a task's kept tokens (`kept` written and
// visible), whole pages of up to NT tokens at a time, from round y on, every ny-th: a
// page's is the largest of its tokens' old ones (scales are not negative: their bits
// order like them).
template <int NT>
__device__ __forceinline__ void new_scales(const EParams &P, const Req &q, uint32_t task, uint32_t h,
                                           const int32_t *kept, uint32_t y, uint32_t ny) {
  __shared__ uint32_t s_max[2][NT / 4];
  float *ns = P.new_scale + (int64_t)task * 2 * P.new_pages;
  const uint32_t pages = NT / P.ps, span = pages * P.ps; // (ps is 4 to 256, NT 256 or more)
  for (uint32_t j0 = y * span; j0 < q.m; j0 += ny * span) {
    for (uint32_t b = threadIdx.x; b < pages; b += NT)
      s_max[0][b] = s_max[1][b] = 0u;
    __syncthreads();
    const uint32_t j = j0 + threadIdx.x;
    if (threadIdx.x < span && j < q.m) {
      const int64_t si =
          ((int64_t)P.bt[q.row + div_ps(P, (uint32_t)kept[j])] * P.Hkv + h) * P.scale_stride;
      const uint32_t b = div_ps(P, threadIdx.x);
      atomicMax(&s_max[0][b], __float_as_uint(fmaxf(P.ks[si], 0.f)));
      atomicMax(&s_max[1][b], __float_as_uint(fmaxf(P.vs[si], 0.f)));
    }
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < pages && j0 + b * P.ps < q.m; b += NT) {
      ns[j0 / P.ps + b] = __uint_as_float(s_max[0][b]);
      ns[P.new_pages + j0 / P.ps + b] = __uint_as_float(s_max[1][b]);
    }
    __syncthreads();
  }
}

// NT lanes with KREG tokens each in registers, a stretch (its token t0 + i NT + lane). A
// request of one stretch is read once; a longer one stretch by stretch for each digit.
template <int NT, int KREG> __global__ void __launch_bounds__(NT) evict_select(EParams P) {
  clear_moves(P, blockIdx.x, NT);
  constexpr uint32_t NW = NT / 64, SPAN = NT * KREG;
  __shared__ uint32_t s_hist[kCopies][256];
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
      if (i % 8 == 7) // eight tokens' addresses at a time
        asm volatile("" ::: "memory");
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
      for (uint32_t k = tid; k < kCopies * 256u; k += NT)
        (&s_hist[0][0])[k] = 0u;
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
            atomicAdd(&s_hist[lane % kCopies][(key >> shift) & mask], 1u);
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

  uint32_t base = 0u, seen = 0u; // kept tokens and ties of the stretches before
  for (uint32_t t0 = 0; t0 < q.n; t0 += SPAN) {
    if (!one)
      load(t0);
    keep_stretch<NT, KREG, true>(P, q, h, x, t0, lo, hi, want, T, left, kept, nullptr, s_cnt, s_wave,
                                 &base, &seen);
  }
  for (uint32_t j = q.m + tid; j < P.max_keep; j += NT)
    kept[j] = -1;
  if (P.new_scale != nullptr && cut) {
    __builtin_amdgcn_s_waitcnt(kVmcnt0);
    __syncthreads();
    new_scales<NT>(P, q, task, h, kept, 0u, 1u);
  }
}

// ---- few long requests: a task's tokens over many workgroups ----------------------
// The same selection in steps: wide_start checks the table and clears the histograms; three
// wide_digit launches count the digits [31:21], [20:10] and [9:0] of the keys, each among those
// that agree with the digits before; wide_count counts each chunk's kept tokens and ties;
// wide_keep writes them and saves their weights, which go to their slots beside the rows, in
// evict_move's grid.
// (Tokens of a workgroup, in us for one request of 65537 with 8 kv-heads, two of 25820 with 2,
// 14 of 30000 with 8: 4096 83.9 / 70.0 / 159, 2048 in 256 lanes 71.7 / 57.9 / 151, in 512 62.4 /
// 51.1 / 160, 1024 63.7 / 48.0 / 187.)
constexpr int kWide = 512, kWideReg = 4;
constexpr uint32_t kWideSpan = kWide * kWideReg, kWideBins = 2048;

__device__ __forceinline__ uint32_t *wide_hist(const EParams &P, uint32_t task) {
  return P.wide + (uint64_t)task * (3u * kWideBins + 1u + 2u * P.chunks);
}

// What a task's tokens compete for; false: the request is not cut, or has a bad table.
struct Contest {
  Req q;
  uint32_t task, r, h, lo, hi, want;
};
__device__ __forceinline__ Contest contest_of(const EParams &P) {
  Contest c;
  c.task = blockIdx.x, c.r = c.task / P.Hkv, c.h = c.task % P.Hkv;
  c.q = req_of(P, c.r);
  const uint32_t recent = min(c.q.m, P.recent);
  c.lo = min(P.sink, c.q.m - recent);
  c.hi = c.q.n - recent;
  c.want = c.q.m - recent - c.lo;
  return c;
}

__global__ void __launch_bounds__(kWide) wide_start(EParams P) {
  __shared__ uint32_t s_bad;
  const Contest c = contest_of(P);
  uint32_t *hist = wide_hist(P, c.task);
  clear_moves(P, c.task, kWide);
  if (threadIdx.x == 0)
    s_bad = c.q.ok ? 0u : 1u;
  __syncthreads();
  if (c.q.ok)
    for (uint32_t b = threadIdx.x; b * (uint64_t)P.ps < c.q.n; b += kWide)
      if ((uint32_t)P.bt[c.q.row + b] >= P.num_pages)
        s_bad = 1u;
  for (uint32_t k = threadIdx.x; k < 3u * kWideBins; k += kWide)
    hist[k] = 0u;
  __syncthreads();
  const uint32_t bad = s_bad;
  if (threadIdx.x == 0) {
    hist[3u * kWideBins] = bad;
    if (bad && P.errors)
      atomicAdd(P.errors, 1u);
  }
  int32_t *kept = P.kept + (int64_t)c.task * P.max_keep;
  for (uint32_t j = (bad ? 0u : c.q.m) + threadIdx.x; j < P.max_keep; j += kWide)
    kept[j] = -1;
}

// The key prefix of the last kept token after `digits` digits, and how many of the tokens that
// share it are kept.
__device__ __forceinline__ void wide_pick(const uint32_t *hist, int digits, uint32_t want,
                                          uint32_t *s_wave, uint32_t *s_pick, uint32_t *T,
                                          uint32_t *left) {
  constexpr uint32_t PER = kWideBins / kWide;
  *T = 0u, *left = want;
  for (int p = 0; p < digits; ++p) {
    uint32_t c[PER], sum = 0u, all;
#pragma unroll
    for (uint32_t k = 0; k < PER; ++k) { // lane 0 has the highest digits
      c[k] = hist[p * kWideBins + kWideBins - 1u - (threadIdx.x * PER + k)];
      sum += c[k];
    }
    uint32_t above = block_scan<kWide>(sum, s_wave, &all) - sum;
#pragma unroll
    for (uint32_t k = 0; k < PER; ++k) {
      if (above < *left && *left <= above + c[k]) {
        s_pick[0] = kWideBins - 1u - (threadIdx.x * PER + k);
        s_pick[1] = above;
      }
      above += c[k];
    }
    __syncthreads();
    *T |= s_pick[0] << (p == 0 ? 21 : p == 1 ? 10 : 0);
    *left -= s_pick[1];
    __syncthreads();
  }
}

__device__ __forceinline__ void wide_load(const EParams &P, const Contest &c, uint32_t t0,
                                          float (&x)[kWideReg]) {
  const float *w0 = P.w + (int64_t)c.h * P.w_hs;
#pragma unroll
  for (int i = 0; i < kWideReg; ++i) {
    const uint32_t t = t0 + (uint32_t)i * kWide + threadIdx.x;
    x[i] = 0.f;
    if (t < c.q.n) {
      const uint32_t b = div_ps(P, t);
      x[i] = w0[(int64_t)P.bt[c.q.row + b] * P.w_ps + (t - b * P.ps)];
    }
  }
}

__global__ void __launch_bounds__(kWide) wide_digit(EParams P, int digit) {
  __shared__ uint32_t s_hist[kWideBins], s_wave[kWide / 64], s_pick[2];
  const Contest c = contest_of(P);
  uint32_t *hist = wide_hist(P, c.task);
  const uint32_t t0 = blockIdx.y * kWideSpan;
  if (t0 >= c.q.n || c.q.m == c.q.n || c.want == 0u || hist[3u * kWideBins])
    return;
  float x[kWideReg];
  wide_load(P, c, t0, x);
  for (uint32_t k = threadIdx.x; k < kWideBins; k += kWide)
    s_hist[k] = 0u;
  uint32_t T, left;
  wide_pick(hist, digit, c.want, s_wave, s_pick, &T, &left);
  __syncthreads();
  const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, top = digit == 1 ? 21 : 10;
  const uint32_t mask = digit == 2 ? 1023u : 2047u;
#pragma unroll
  for (int i = 0; i < kWideReg; ++i) {
    const uint32_t t = t0 + (uint32_t)i * kWide + threadIdx.x, key = order_bits(x[i]);
    if (t >= c.lo && t < c.hi && (digit == 0 || (key >> top) == (T >> top)))
      atomicAdd(&s_hist[(key >> shift) & mask], 1u);
  }
  __syncthreads();
  for (uint32_t k = threadIdx.x; k < kWideBins; k += kWide)
    if (s_hist[k])
      atomicAdd(&hist[digit * kWideBins + k], s_hist[k]);
}

__global__ void __launch_bounds__(kWide) wide_count(EParams P) {
  __shared__ uint32_t s_wave[kWide / 64], s_pick[2];
  const Contest c = contest_of(P);
  uint32_t *hist = wide_hist(P, c.task), *cnt = hist + 3u * kWideBins + 1u;
  const uint32_t t0 = blockIdx.y * kWideSpan;
  if (t0 >= c.q.n || c.q.m == c.q.n || hist[3u * kWideBins])
    return;
  float x[kWideReg];
  wide_load(P, c, t0, x);
  uint32_t T = 0u, left = 0u;
  if (c.want > 0u)
    wide_pick(hist, 3, c.want, s_wave, s_pick, &T, &left);
  uint32_t stay = 0u, ties = 0u, all;
#pragma unroll
  for (int i = 0; i < kWideReg; ++i) {
    const uint32_t t = t0 + (uint32_t)i * kWide + threadIdx.x, key = order_bits(x[i]);
    const bool mid = t >= c.lo && t < c.hi;
    stay += t < c.q.n && (!mid || (c.want > 0u && key > T));
    ties += mid && c.want > 0u && key == T;
  }
  block_scan<kWide>(stay, s_wave, &all);
  if (threadIdx.x == 0)
    cnt[2u * blockIdx.y] = all;
  block_scan<kWide>(ties, s_wave, &all);
  if (threadIdx.x == 0)
    cnt[2u * blockIdx.y + 1u] = all;
}

__global__ void __launch_bounds__(kWide) wide_keep(EParams P) {
  __shared__ uint32_t s_cnt[kWideReg * (kWide / 64)], s_wave[kWide / 64], s_pick[2];
  const Contest c = contest_of(P);
  uint32_t *hist = wide_hist(P, c.task), *cnt = hist + 3u * kWideBins + 1u;
  const uint32_t t0 = blockIdx.y * kWideSpan;
  if (t0 >= c.q.n || hist[3u * kWideBins])
    return;
  const bool cut = c.q.m < c.q.n;
  float x[kWideReg];
  wide_load(P, c, t0, x);
  uint32_t T = 0u, left = 0u, base = 0u, seen = 0u;
  if (cut) {
    if (c.want > 0u)
      wide_pick(hist, 3, c.want, s_wave, s_pick, &T, &left);
    uint32_t a = 0u, b = 0u;
    for (uint32_t k = threadIdx.x; k < blockIdx.y; k += kWide) {
      a += cnt[2u * k];
      b += cnt[2u * k + 1u];
    }
    block_scan<kWide>(a, s_wave, &base);
    block_scan<kWide>(b, s_wave, &seen);
    base += min(seen, left);
  } else {
    base = t0;
  }
  keep_stretch<kWide, kWideReg, false>(P, c.q, c.h, x, t0, c.lo, c.hi, c.want, T, left,
                                       P.kept + (int64_t)c.task * P.max_keep,
                                       P.saved + (int64_t)c.task * P.most_kept, s_cnt, s_wave, &base,
                                       &seen);
}

__global__ void __launch_bounds__(1024) wide_scales(EParams P) {
  const Contest c = contest_of(P);
  const int32_t *kept = P.kept + (int64_t)c.task * P.max_keep;
  if (c.q.m < c.q.n && c.q.m > 0u && kept[0] >= 0)
    new_scales<1024>(P, c.q, c.task, c.h, kept, blockIdx.y, gridDim.y);
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

// Four e4m3 codes, each times its f and encoded anew; where f is below 0, and NaN codes, as
// they are.
__device__ __forceinline__ uint32_t recode4(uint32_t c, const float (&f)[4]) {
  typedef __attribute__((ext_vector_type(2))) float f32x2_t;
  const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false);
  const f32x2_t b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  const float q[4] = {a.x * f[0], a.y * f[1], b.x * f[2], b.y * f[3]};
  uint32_t y = encode4_fp8(q);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t m = 0x7fu << (8 * k), all = 0xffu << (8 * k);
    y = (c & m) == m || !(f[k] >= 0.f) ? (y & ~all) | (c & all) : y;
  }
  return y;
}
__device__ __forceinline__ uint32_t recode4(uint32_t c, float f) {
  const float g[4] = {f, f, f, f};
  return recode4(c, g);
}
__device__ __forceinline__ void recode(uint4 &x, float f) {
  x.x = recode4(x.x, f), x.y = recode4(x.y, f), x.z = recode4(x.z, f), x.w = recode4(x.w, f);
}
__device__ __forceinline__ void recode(uint8_t &x, float f) { x = (uint8_t)recode4(x, f); }
template <typename U> __device__ __forceinline__ void recode(U &, float) {}

constexpr int kMove = 512;
constexpr uint32_t kStage = 2048; // rows whose places are in LDS at a time

// Saved weights to their slots: chunk `which` % save_chunks of a task. (Gathered from their old
// slots by one workgroup a task, a round read before it is written, the 50000 kept weights
// of one request of 100000 took 69 us more.)
constexpr uint32_t kSaved = kMove * 8;

__device__ __forceinline__ void put_weights(const EParams &P, uint32_t which) {
  const uint32_t task = which / P.save_chunks, j0 = which % P.save_chunks * kSaved;
  const uint32_t r = task / P.Hkv, h = task % P.Hkv;
  const Req q = req_of(P, r);
  if (j0 >= q.m || P.kept[(int64_t)task * P.max_keep] < 0 || (q.m == q.n && P.wo == P.w))
    return;
  const float *saved = P.saved + (int64_t)task * P.most_kept;
  const uint32_t end = min(q.m, j0 + kSaved);
  for (uint32_t j = j0 + threadIdx.x; j < end; j += kMove) {
    const uint32_t b = div_ps(P, j);
    P.wo[(int64_t)P.bt[q.row + b] * P.w_ps + (int64_t)h * P.w_hs + (j - b * P.ps)] = saved[j];
  }
}

// How a tensor's tokens are moved: element by element, in 16-byte units of their rows, or
// (d-major values) in 16 bytes of tokens of one dim.
enum Mode : uint32_t { kElems, kRows, kTurned };

template <int EB> struct Elem;
template <> struct Elem<1> { typedef uint8_t type; };
template <> struct Elem<2> { typedef uint16_t type; };
template <> struct Elem<4> { typedef uint32_t type; };

// One of a task's two tensors: where its tokens are, in bytes.
struct Side {
  uint8_t *pool; // the kv-head's
  int64_t page, tok, dim;
  const float *scale, *ns; // fp8: the pages' scales and the new ones
};

template <int EB>
__device__ __forceinline__ Side side_of(const EParams &P, uint32_t task, uint32_t h, bool vals) {
  Side S;
  S.pool = (vals ? P.v + (int64_t)h * P.vhs * EB : P.k + (int64_t)h * P.khs * EB);
  S.page = (vals ? P.vps : P.kps) * EB, S.tok = (vals ? P.vts : P.kts) * EB;
  S.dim = (vals ? P.vds : 1) * EB;
  S.scale = vals ? P.vs : P.ks;
  S.ns = P.new_scale + ((int64_t)task * 2 + (vals ? 1 : 0)) * P.new_pages;
  return S;
}

// The places of kept tokens j0 .. j0 + cnt - 1: from (with kStays: the token is there already,
// as it will be), to, and for fp8 the old scale over the new one (below 0: the codes stay).
constexpr int64_t kStays = INT64_MIN;
template <bool FP8>
__device__ __forceinline__ void places(const EParams &P, const Req &q, uint32_t h, const Side &S,
                                       const int32_t *kept, uint32_t j0, uint32_t cnt,
                                       int64_t *s_from, int64_t *s_to, float *s_ratio) {
  for (uint32_t i = threadIdx.x; i < cnt; i += kMove) {
    const uint32_t j = j0 + i, src = (uint32_t)kept[j];
    const uint32_t sb = div_ps(P, src), db = div_ps(P, j);
    const int64_t sp = P.bt[q.row + sb], dp = P.bt[q.row + db];
    bool moves = src != j;
    if constexpr (FP8) {
      const float was = S.scale[(sp * P.Hkv + h) * P.scale_stride], now = S.ns[db];
      s_ratio[i] = was != now ? was / now : -1.f;
      moves = moves || was != now;
    }
    s_from[i] = (sp * S.page + (int64_t)(src - sb * P.ps) * S.tok) | (moves ? 0 : kStays);
    s_to[i] = dp * S.page + (int64_t)(j - db * P.ps) * S.tok;
  }
}

// kTurned: 16 bytes of one dim, the values of 16 / EB tokens from k0 on (`pool` at the dim).
// False: none of them moves. (Loads under no condition, in flight together: a token from
// cnt on reads as the last.)
template <int EB>
__device__ __forceinline__ bool gather16(const uint8_t *pool, const int64_t *s_from, uint32_t k0,
                                         uint32_t cnt, uint4 &x) {
  typedef typename Elem<EB>::type E;
  constexpr int TOK = 16 / EB, PER = 4 / EB; // tokens of it, and of a word
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  bool any = false;
#pragma unroll
  for (int t = 0; t < TOK; ++t) {
    const int64_t from = s_from[min(k0 + t, cnt - 1u)];
    any = any || from >= 0;
    const uint32_t e = *reinterpret_cast<const E *>(pool + (from & ~kStays));
    w[t / PER] |= e << (8 * EB * (t % PER));
  }
  x = uint4{w[0], w[1], w[2], w[3]};
  return any;
}

// Behind piece i of N: 32 of gather16's loads in flight at most (a piece's come apart in
// registers until it is whole).
template <int EB, int N> __device__ __forceinline__ void gather_step(int i, uint4 (&x)[N]) {
  if (i % EB == EB - 1) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j > i - 2 * EB && j <= i - EB)
        hold(x[j]);
    asm volatile("" ::: "memory");
  }
}

template <int EB>
__device__ __forceinline__ void scatter16(uint8_t *pool, const int64_t *s_to, const float *s_ratio,
                                          uint32_t k0, uint32_t cnt, uint4 x) {
  typedef typename Elem<EB>::type E;
  constexpr int TOK = 16 / EB, PER = 4 / EB;
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
  if constexpr (EB == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[4];
      bool any = false;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f[t] = k0 + 4 * i + t < cnt ? s_ratio[k0 + 4 * i + t] : -1.f;
        any = any || f[t] >= 0.f;
      }
      if (any)
        w[i] = recode4(w[i], f);
    }
  }
  if (k0 + TOK <= cnt) {
    *reinterpret_cast<uint4 *>(pool + s_to[k0]) = uint4{w[0], w[1], w[2], w[3]};
  } else {
#pragma unroll
    for (int t = 0; t < TOK; ++t)
      if (k0 + t < cnt)
        *reinterpret_cast<E *>(pool + s_to[k0 + t]) = (E)(w[t / PER] >> (8 * EB * (t % PER)));
  }
}

// A stage's tokens in units U, `units` of them a token and `step` bytes apart.
template <typename U, int N, bool FP8>
__device__ __forceinline__ void move_units(uint8_t *pool, uint32_t units, int64_t step,
                                           uint32_t cnt, const int64_t *s_from,
                                           const int64_t *s_to, const float *s_ratio) {
  const uint32_t tid = threadIdx.x, e = tid % units, rr = tid / units, rows = kMove / units;
  const bool active = rr < rows;
  const uint32_t round = rows * N;
  pool += (int64_t)e * step;
  U x[N], nx[N];
  auto fetch = [&](uint32_t k0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t k = k0 + (uint32_t)i * rows + rr;
      nx[i] = U{};
      if (active && k < cnt) {
        const int64_t from = s_from[k];
        if (from >= 0)
          nx[i] = *reinterpret_cast<const U *>(pool + from);
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
    // the round's rows are in registers on every lane before any of them is written: each
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
          const float f = s_ratio[k];
          if (f >= 0.f)
            recode(x[i], f);
        }
        *reinterpret_cast<U *>(pool + s_to[k]) = x[i];
      }
    }
  }
}

// A stage's tokens in 16 bytes of one dim, a round of kMove * N pieces in the order of their
// tokens: what a later round reads of a dim lies behind what this one writes of it.
template <int EB>
__device__ __forceinline__ void move_turned(uint8_t *pool, uint32_t dims, int64_t step,
                                            uint32_t cnt, const int64_t *s_from,
                                            const int64_t *s_to, const float *s_ratio) {
  constexpr int N = EB == 4 ? 4 : 2;
  constexpr uint32_t TOK = 16 / EB;
  const uint32_t pieces = (cnt + TOK - 1u) / TOK * dims;
  for (uint32_t p0 = 0; p0 < pieces; p0 += kMove * N) {
    uint4 x[N];
    bool moves[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t p = p0 + (uint32_t)i * kMove + threadIdx.x, pc = min(p, pieces - 1u);
      moves[i] = gather16<EB>(pool + pc % dims * step, s_from, pc / dims * TOK, cnt, x[i]);
      moves[i] = moves[i] && p < pieces;
      gather_step<EB>(i, x);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      hold(x[i]);
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t p = p0 + (uint32_t)i * kMove + threadIdx.x;
      if (moves[i])
        scatter16<EB>(pool + p % dims * step, s_to, s_ratio, p / dims * TOK, cnt, x[i]);
    }
  }
}

template <int EB>
__global__ void __launch_bounds__(kMove, 4) evict_move(EParams P, Mode k_mode, Mode v_mode) {
  typedef typename Elem<EB>::type E;
  constexpr bool FP8 = EB == 1;
  __shared__ int64_t s_from[kStage], s_to[kStage];
  __shared__ float s_ratio[FP8 ? kStage : 1];
  if (blockIdx.x >= P.row_groups) { // the wide selection's weights
    put_weights(P, blockIdx.x - P.row_groups);
    return;
  }
  const uint32_t task = blockIdx.x >> 1;
  const bool vals = (blockIdx.x & 1u) != 0u;
  const uint32_t r = task / P.Hkv, h = task % P.Hkv;
  const Req q = req_of(P, r);
  const int32_t *kept = P.kept + (int64_t)task * P.max_keep;
  if (q.m == q.n || q.m == 0u || kept[0] < 0)
    return;
  const Side S = side_of<EB>(P, task, h, vals);
  const Mode mode = vals ? v_mode : k_mode;
  for (uint32_t j0 = 0; j0 < q.m; j0 += kStage) {
    const uint32_t cnt = min(kStage, q.m - j0);
    __syncthreads(); // the previous stage's places have been used
    places<FP8>(P, q, h, S, kept, j0, cnt, s_from, s_to, s_ratio);
    __syncthreads();
    if (mode == kRows)
      move_units<uint4, 4, FP8>(S.pool, P.D * EB / 16u, 16, cnt, s_from, s_to, s_ratio);
    else if (mode == kTurned)
      move_turned<EB>(S.pool, P.D, S.dim, cnt, s_from, s_to, s_ratio);
    else
      move_units<E, 4, FP8>(S.pool, P.D, S.dim, cnt, s_from, s_to, s_ratio);
  }
}

// Few tasks: a task's tokens over many workgroups. Each takes the next chunk of its (task, keys
// or values) by a ticket, reads the chunk's tokens into registers, says so, and writes them
// once all chunks before it have said so: what it overwrites are tokens of theirs or its own.
// A chunk waits for earlier tickets only, whose workgroups are running and wait for nothing
// before they say so; every wait ends.
//
// 16-byte units of a lane, 8 and 4: one request of 65537 tokens, an eighth kept, 51 / 55 us, 4
// of 8000 55 / 59; with d-major values 2 of 2000 33 / 26, 64 of 1000 fp8 143 / 128, one of 65537
// 88 / 91.
__host__ __device__ constexpr int few_units(bool turned) { return turned ? 4 : 8; }

// Tokens of a chunk: a multiple of 16, so that a turned unit lies in one chunk.
__host__ __device__ inline uint32_t few_rows(uint32_t units, bool turned) {
  return kMove / units * few_units(turned) & ~15u;
}

template <int EB, bool TURNED>
__global__ void __launch_bounds__(kMove) evict_move_few(EParams P) {
  constexpr bool FP8 = EB == 1;
  constexpr int UNITS = few_units(TURNED);
  constexpr uint32_t MOST = kMove / 4 * UNITS; // tokens of a chunk (4 units each at least)
  constexpr uint32_t TOK = 16 / EB;
  __shared__ int64_t s_from[MOST], s_to[MOST];
  __shared__ float s_ratio[FP8 ? MOST : 1];
  __shared__ uint32_t s_chunk;
  if (blockIdx.x >= P.row_groups) { // the wide selection's weights
    put_weights(P, blockIdx.x - P.row_groups);
    return;
  }
  const uint32_t tid = threadIdx.x, which = blockIdx.x % (2u * P.R * P.Hkv), task = which >> 1;
  const bool vals = (which & 1u) != 0u;
  const uint32_t r = task / P.Hkv, h = task % P.Hkv;
  const Req q = req_of(P, r);
  const int32_t *kept = P.kept + (int64_t)task * P.max_keep;
  if (q.m == q.n || q.m == 0u || kept[0] < 0)
    return;
  uint32_t *ticket = P.moves + (uint64_t)which * (1u + P.move_chunks), *flag = ticket + 1;
  if (tid == 0)
    s_chunk = atomicAdd(ticket, 1u);
  __syncthreads();
  const uint32_t units = P.D * EB / 16u, each = few_rows(units, TURNED), chunk = s_chunk;
  const uint32_t j0 = chunk * each;
  if (j0 >= q.m)
    return;
  const uint32_t cnt = min(each, q.m - j0);
  const Side S = side_of<EB>(P, task, h, vals);
  places<FP8>(P, q, h, S, kept, j0, cnt, s_from, s_to, s_ratio);
  __syncthreads();
  // turned: unit p is of dim p % D, of the tokens from p / D * TOK on
  const bool turned = TURNED && vals;
  const uint32_t most = (cnt + TOK - 1u) / TOK * P.D;
  const uint32_t rows = kMove / units, rr = tid / units, off = tid % units * 16u;
  uint4 x[UNITS];
  uint32_t moves = 0u;
  if (!turned) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const uint32_t k = (uint32_t)i * rows + rr;
      x[i] = uint4{};
      if (rr < rows && k < cnt && s_from[k] >= 0) {
        moves |= 1u << i;
        x[i] = *reinterpret_cast<const uint4 *>(S.pool + s_from[k] + off);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const uint32_t p = (uint32_t)i * kMove + tid, pc = min(p, most - 1u);
      const bool any =
          gather16<EB>(S.pool + pc % P.D * S.dim, s_from, pc / P.D * TOK, cnt, x[i]);
      moves |= any && p < most ? 1u << i : 0u;
      gather_step<EB>(i, x);
    }
  }
#pragma unroll
  for (int i = 0; i < UNITS; ++i)
    hold(x[i]);
  __builtin_amdgcn_s_waitcnt(kVmcnt0);
  __syncthreads(); // the chunk is in registers: nothing to publish but that
  if (tid == 0)
    __hip_atomic_store(flag + chunk, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (tid < 64u)
    for (uint32_t k = tid; k < chunk; k += 64u)
      while (__hip_atomic_load(flag + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0u)
        __builtin_amdgcn_s_sleep(1);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    if (!((moves >> i) & 1u))
      continue;
    if (turned) {
      const uint32_t p = (uint32_t)i * kMove + tid;
      scatter16<EB>(S.pool + p % P.D * S.dim, s_to, s_ratio, p / P.D * TOK, cnt, x[i]);
    } else {
      const uint32_t k = (uint32_t)i * rows + rr;
      if constexpr (FP8) {
        const float f = s_ratio[k];
        if (f >= 0.f)
          recode(x[i], f);
      }
      *reinterpret_cast<uint4 *>(S.pool + s_to[k] + off) = x[i];
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

// The most tokens that a request of the call keeps: not more than its table holds.
uint32_t most_kept(const SchedEvictArgs *a) {
  return (uint32_t)std::min<uint64_t>(a->max_keep, (uint64_t)a->max_pages * a->page_size);
}
uint32_t new_pages_of(const SchedEvictArgs *a) {
  return (uint32_t)(((uint64_t)most_kept(a) + a->page_size - 1u) / a->page_size);
}

// Tables that reach past one workgroup's registers (evict_select<512, 24>'s 12288 tokens),
// of fewer tasks than half the compute units, take the wide selection: 8 tasks of 65537
// tokens 198 -> 51 us with the moves, 4 of 25820 119 -> 44; 8 of 12000, which fit, 46 -> 51.
constexpr uint32_t kWideTasks = 128, kShort = 256u * 16u, kOneRead = 512u * 24u;

bool wide_applies(const SchedEvictArgs *a) {
  return (uint64_t)a->max_pages * a->page_size > kOneRead &&
         (uint64_t)a->num_requests * a->num_kv_heads < kWideTasks;
}
uint32_t wide_chunks(const SchedEvictArgs *a) {
  return (uint32_t)(((uint64_t)a->max_pages * a->page_size + kWideSpan - 1u) / kWideSpan);
}
uint64_t scale_bytes(const SchedEvictArgs *a) {
  if (a->kv_dtype != SCHED_PD_FP8_E4M3)
    return 0;
  const uint64_t tasks = (uint64_t)a->num_requests * a->num_kv_heads;
  return (tasks * 2u * new_pages_of(a) * 4u + 255u) / 256u * 256u;
}
uint64_t wide_bytes(const SchedEvictArgs *a) {
  if (!wide_applies(a))
    return 0;
  const uint64_t tasks = (uint64_t)a->num_requests * a->num_kv_heads;
  return tasks * (3u * kWideBins + 1u + 2u * wide_chunks(a) + most_kept(a)) * 4u;
}
// Each tensor in 16-byte units where its strides allow. d-major, 8 kv-heads of 128 (us, V by
// element / turned): 32 requests of 2048, half kept, 258 / 160; 2 of 2000 168 / 33; one of
// 65537, an eighth kept, 1067 / 120.
bool in16(const SchedEvictArgs *a, int64_t x) { return x * elem_bytes(a->kv_dtype) % 16 == 0; }
Mode k_mode_of(const SchedEvictArgs *a) {
  return in16(a, a->head_dim) && (uintptr_t)a->k_pool % 16 == 0 && in16(a, a->k_page_stride) &&
                 in16(a, a->k_head_stride) && in16(a, a->k_tok_stride)
             ? kRows
             : kElems;
}
Mode v_mode_of(const SchedEvictArgs *a) {
  if ((uintptr_t)a->v_pool % 16 || !in16(a, a->v_page_stride) || !in16(a, a->v_head_stride))
    return kElems;
  if (a->v_dim_stride == 1)
    return in16(a, a->head_dim) && in16(a, a->v_tok_stride) ? kRows : kElems;
  return in16(a, a->v_dim_stride) && in16(a, a->page_size) ? kTurned : kElems;
}
// Whether the rows are cut over workgroups. In us, with one workgroup per task and tensor
// against chunks (head dim 128, bf16): 8 tasks of 1000 tokens 23.0 / 19.2, 192 of 1200 51.4 /
// 48.8, 192 of 2048 fp8 47.7 / 44.9; at 256 tasks even (1200 tokens 62.1 / 62.8) or worse (2048
// 77.7 / 81.9), and at 360 kept tokens and fewer too (8 of 300 12.9 / 13.2, 32 of 400 17.3 / 17.7).
// d-major: 256 tasks of 2048 fp8 134 / 104, 512 of 1000 215 / 135; bf16 160 / 160, 1024 of
// 1000 428 / 420.
constexpr uint32_t kMoveFill = 512; // workgroups of evict_move that fill the card
constexpr uint32_t kTurnFill = 4096;
constexpr uint32_t kFewKeep = 512;
bool few_applies(const SchedEvictArgs *a) {
  const uint32_t fill = a->v_dim_stride == 1 ? kMoveFill : kTurnFill;
  return 2ull * a->num_requests * a->num_kv_heads < fill &&
         a->head_dim * elem_bytes(a->kv_dtype) >= 64u && most_kept(a) > kFewKeep;
}
uint32_t few_chunks(const SchedEvictArgs *a) {
  const uint32_t units = a->head_dim * elem_bytes(a->kv_dtype) / 16u;
  const uint32_t rows = few_rows(units, a->v_dim_stride != 1);
  return (most_kept(a) + rows - 1u) / rows;
}
uint64_t move_bytes(const SchedEvictArgs *a) {
  if (!few_applies(a))
    return 0;
  return 2ull * a->num_requests * a->num_kv_heads * (1u + few_chunks(a)) * 4u;
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
  return (int64_t)(scale_bytes(a) + wide_bytes(a) + move_bytes(a));
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
  for (int64_t st : {a->k_page_stride, a->k_head_stride, a->k_tok_stride, a->v_page_stride,
                     a->v_head_stride, a->v_tok_stride, a->v_dim_stride})
    if (st < 0)
      return set_error(-1, "sched_kv_evict: a pool's stride is negative");
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
  const Mode k_mode = k_mode_of(a), v_mode = v_mode_of(a);
  const bool many = wide_applies(a), few = few_applies(a) && k_mode == kRows && v_mode != kElems;
  if (few) {
    P.moves = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(a->workspace) + scale_bytes(a) +
                                           wide_bytes(a));
    P.move_chunks = few_chunks(a);
  }
  if (many) {
    P.wide = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(a->workspace) + scale_bytes(a));
    P.chunks = wide_chunks(a);
    P.most_kept = most_kept(a), P.save_chunks = (P.most_kept + kSaved - 1u) / kSaved;
    P.saved = reinterpret_cast<float *>(P.wide + (uint64_t)tasks * (3u * kWideBins + 1u +
                                                                   2u * P.chunks));
    const dim3 grid(tasks, P.chunks);
    hipLaunchKernelGGL(wide_start, dim3(tasks), dim3(kWide), 0, s, P);
    for (int digit = 0; digit < 3; ++digit)
      hipLaunchKernelGGL(wide_digit, grid, dim3(kWide), 0, s, P, digit);
    hipLaunchKernelGGL(wide_count, grid, dim3(kWide), 0, s, P);
    hipLaunchKernelGGL(wide_keep, grid, dim3(kWide), 0, s, P);
    if (fp8)
      hipLaunchKernelGGL(wide_scales, dim3(tasks, std::max(1u, (most_kept(a) + 767u) / 768u)),
                         dim3(1024), 0, s, P); // (a round has 769 tokens or more)
  } else if (longest <= kShort) {
    hipLaunchKernelGGL((evict_select<256, 16>), dim3(tasks), dim3(256), 0, s, P);
  } else {
    hipLaunchKernelGGL((evict_select<512, 24>), dim3(tasks), dim3(512), 0, s, P);
  }
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a->max_keep > 0) {
    P.row_groups = 2u * tasks * (few ? P.move_chunks : 1u);
    const dim3 grid(P.row_groups + (many ? tasks * P.save_chunks : 0u)), block(kMove);
    if (few) {
      const bool turned = v_mode == kTurned;
      auto fn = eb == 1   ? (turned ? evict_move_few<1, true> : evict_move_few<1, false>)
                : eb == 2 ? (turned ? evict_move_few<2, true> : evict_move_few<2, false>)
                          : (turned ? evict_move_few<4, true> : evict_move_few<4, false>);
      hipLaunchKernelGGL(fn, grid, block, 0, s, P);
    } else {
      auto fn = eb == 1 ? evict_move<1> : eb == 2 ? evict_move<2> : evict_move<4>;
      hipLaunchKernelGGL(fn, grid, block, 0, s, P, k_mode, v_mode);
    }
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

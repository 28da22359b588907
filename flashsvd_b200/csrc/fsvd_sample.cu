// Choice of the next token (fsvd_sample of include/flashsvd_b200.h): temperature, top-k, top-p, min-p, one uniform number.
//
// The vocabulary is ordered by logit (descending, lower index first); every filter keeps a prefix of that order, so the
// kept set is {key > t} and the first r of {key = t} in index order, for one threshold key t.  It is found without a
// sort: a histogram of 1024 bins over the values narrows the threshold to one bin, and a few dozen candidates are then
// ranked directly; where a bin holds too many, bins over the integer keys inside it narrow it on.
//
// Weights are integers, exp((l - max) / T) * 2^frac: their sums do not depend on the order of addition (the histograms
// are built by atomics), and comparisons of running sums with u Z and p Z are exact in them.  A weight is good to 2^-29
// of itself: between V boundaries of a flat row a draw lands on another token than in exact arithmetic once in
// 2^29 / sqrt(V) rows.  (32-bit exponentials miss 64 times as often, 64-bit ones take a third of the kernel's time.)
//
// A row belongs to a cluster of up to eight CTAs, each with a contiguous piece of it in shared memory, so that HBM is read
// once; sums and histograms meet through distributed shared memory.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>
#include <type_traits>

#include "../../include/flashsvd_b200.h"
#include "fsvd_tc.cuh"
#include "fsvd_tile.h"

namespace fsvd_sample_impl {

using fsvd_tile::cluster_sync;
typedef unsigned long long u64;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kLimbs = 4, kLimbBits = 12;   // a weight of at most 2^46 as four numbers of 12 bits: 2^20 of them fit 32-bit sums
constexpr int kList = 96;                   // candidates that are ranked directly
constexpr int kBlock = 128;                 // elements of a warp's step: four neighbours per lane
constexpr int kMaxCluster = 8;
constexpr int kMaxVocab = 1 << 22;

struct Args {
  const void* logits;
  long long stride;
  const float *u, *temperature, *top_p, *min_p;
  const int* top_k;
  float T_all, p_all, m_all;
  int k_all;
  int* tokens;
  float* probs;
  int V, chunk, frac;   // chunk: elements of a CTA, a multiple of kBlock
};

// What a CTA shows to the others of its cluster.
struct Slot {
  u64 best, count, mass, sum, above;   // (each written once between two reads by the others)
  float low;
  uint32_t n, kmin, kmax, eq;
};

struct Shared {
  uint32_t hist[kLimbs][kBins];
  u64 total[kBins];
  u64 warp_sum[kWarps];
  uint32_t warp_eq[kWarps];
  u64 scan[kWarps];
  uint32_t list_key[kList];
  int list_at[kList];
  uint32_t all_key[kList];
  int all_at[kList];
  u64 all_w[kList];
  uint32_t table[64];
  Slot slot;
  Slot red[kWarps];
  int pick_lo, pick_hi, list_n;
  u64 pick_above;
  uint32_t pick_key;
  u64 pick_ties;
};

// Ascending keys for ascending numbers above -infinity; 0 for -infinity.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return x == -INFINITY ? 0u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
__device__ __forceinline__ float plain(float x) { return x > -INFINITY ? x + 0.0f : -INFINITY; }   // NaN counts as -infinity; one zero
__device__ __forceinline__ float logit(const float* row, int i) { return plain(row[i]); }
__device__ __forceinline__ float logit(const __nv_bfloat16* row, int i) { return plain(__bfloat162float(row[i])); }

__device__ __forceinline__ uint32_t remote(const void* p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(fsvd_tile::smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t peek(const uint32_t* p, int rank) {
  uint32_t x;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(remote(p, rank)) : "memory");
  return x;
}
__device__ __forceinline__ u64 peek(const u64* p, int rank) {
  u64 x;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(remote(p, rank)) : "memory");
  return x;
}
__device__ __forceinline__ void poke(u64* p, int rank, u64 x) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(p, rank)), "l"(x) : "memory");
}
__device__ __forceinline__ int cluster_rank() {
  int r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ int cluster_size() {
  int r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
template <typename F>
__device__ __forceinline__ u64 warp_reduce(u64 x, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ u64 warp_add(u64 x) {
  return warp_reduce(x, [](u64 a, u64 b) { return a + b; });
}

// exp((x - max) / T) as an integer.  log2 of it is formed in 64 bits as a fixed-point number: added to 1.5 * 2^20 its
// fraction fills the low 32 bits of the sum.  2^fraction = 2^(j / 64) (1 + q), j the top six bits, q a polynomial in the
// other 26 (Taylor: the next term is below 2^-38).
struct Weigher {
  double max, c;   // c = log2(e) / T
  float half_max, fc2;     // for a 32-bit logarithm: halves, so that a difference of finite numbers stays finite
  int frac;
  const uint32_t* table;   // 2^(31 + j / 64)
  __device__ __forceinline__ float log2f32(float x) const { return fmaf(0.5f, x, -half_max) * fc2; }   // to 2^-22 of itself
  __device__ __forceinline__ u64 operator()(float x) const {
    if (!(log2f32(x) > -60.0f)) return 0;
    const double t = fma((double)x - max, c, 1572864.0);
    const uint32_t lo = (uint32_t)__double2loint(t);
    const int n = 0x41380000 - __double2hiint(t);   // 2^-n
    const float z = __uint_as_float(0x3f800000u | ((lo & 0x3ffffffu) >> 3)) - 1.0f;   // 64 times the rest, in [0, 1)
    constexpr float a1 = 0.69314718056f;   // 64 q = a1 z + a1^2 z^2 / 128 + a1^3 z^3 / (6 * 64^2) + a1^4 z^4 / (24 * 64^3)
    const float q = z * (a1 + z * (a1 * a1 / 128.0f + z * (a1 * a1 * a1 / 24576.0f + z * (a1 * a1 * a1 * a1 / 6291456.0f))));
    const uint32_t m = (__float_as_uint(1.0f + q) & 0x7fffffu) << 3;   // q 2^32
    const uint32_t T = table[lo >> 26];
    return ((u64)(T + __umulhi(T, m)) << (frac - 31)) >> n;
  }
};

template <typename T, bool RESIDENT>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Args a) {
  extern __shared__ float vals[];   // RESIDENT: this CTA's piece, -infinity behind the end
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  const int rank = cluster_rank(), C = cluster_size(), b = blockIdx.x / C;
  const int base = rank * a.chunk, len = max(0, min(a.chunk, V - base));
  const T* row = reinterpret_cast<const T*>(a.logits) + (size_t)b * a.stride;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid < 64) s.table[tid] = (uint32_t)__double2ll_rn(exp2((double)tid / 64.0) * 2147483648.0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float temp = fminf(a.temperature ? a.temperature[b] : a.T_all, 3.402823466e38f);
  int k = a.top_k ? a.top_k[b] : a.k_all;
  const float p = a.top_p ? a.top_p[b] : a.p_all, mp = fminf(a.min_p ? a.min_p[b] : a.m_all, 1.0f);
  if (k <= 0 || k > V) k = V;

  // ---- the row into shared memory; its largest element (lowest index among equals) and its smallest finite one
  u64 best = 0;
  float low = INFINITY;
  {
    constexpr int U = 8;
    const int padded = (len + kBlock - 1) / kBlock * kBlock;
    for (int i0 = tid; i0 < padded; i0 += U * kThreads) {
      float x[U];
#pragma unroll
      for (int e = 0; e < U; ++e) {
        const int i = i0 + e * kThreads;
        x[e] = i < len ? logit(row, base + i) : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < U; ++e) {
        const int i = i0 + e * kThreads;
        if (RESIDENT && i < padded) vals[i] = x[e];
        best = max(best, ((u64)key_of(x[e]) << 32) | (uint32_t)~(base + i));
        if (x[e] > -INFINITY) low = fminf(low, x[e]);
      }
    }
  }
  auto larger = [](u64 x, u64 y) { return x > y ? x : y; };
  best = warp_reduce(best, larger);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  if (lane == 0) {
    s.red[warp].best = best;
    s.red[warp].low = low;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w) {
      best = larger(best, s.red[w].best);
      low = fminf(low, s.red[w].low);
    }
    s.slot.best = best;
    s.slot.low = low;
  }
  cluster_sync();
  best = 0;
  low = INFINITY;
  for (int r = 0; r < C; ++r) {
    best = larger(best, peek(&s.slot.best, r));
    low = fminf(low, __uint_as_float(peek(reinterpret_cast<const uint32_t*>(&s.slot.low), r)));
  }
  const uint32_t kbest = (uint32_t)(best >> 32);
  if (kbest == 0u || !(temp > 0.0f) || k == 1) {
    if (rank == 0 && tid == 0) {
      a.tokens[b] = kbest == 0u ? 0 : (int)~(uint32_t)best;
      if (a.probs) a.probs[b] = kbest == 0u ? 0.0f : 1.0f;
    }
    cluster_sync();   // (the others may still be reading this CTA's slot)
    return;
  }
  // An infinite maximum: the elements that equal it share everything, the others get nothing.
  const bool inf = value_of(kbest) == INFINITY;
  const float top = inf ? 0.0f : value_of(kbest);
  if (inf) low = 0.0f;
  const int nblk = (len + kBlock - 1) / kBlock, per = (nblk + kWarps - 1) / kWarps;
  const int blk0 = min(nblk, warp * per), blk1 = min(nblk, blk0 + per);
  auto get4 = [&](int blk, float (&x)[4]) {
    const int i = blk * kBlock + 4 * lane;
    if constexpr (RESIDENT) {
      const float4 v = *reinterpret_cast<const float4*>(vals + i);
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = i + e < len ? logit(row, base + i + e) : -INFINITY;
    }
    if (inf) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = x[e] == INFINITY ? 0.0f : -INFINITY;
    }
  };
  Weigher W;
  W.max = (double)top;
  W.c = 1.4426950408889634074 / (double)temp;
  W.half_max = 0.5f * top;
  W.fc2 = (float)fmin(2.0 * W.c, 3.402823466e38);
  W.frac = a.frac;
  W.table = s.table;

  // Sum over the cluster of one number per thread (a slot field that the caller chooses).
  auto cluster_total = [&](u64 x, u64 Slot::* field) -> u64 {
    x = warp_add(x);
    __syncthreads();
    if (lane == 0) s.scan[warp] = x;
    __syncthreads();
    if (tid == 0) {
      u64 t = 0;
      for (int w = 0; w < kWarps; ++w) t += s.scan[w];
      s.slot.*field = t;
    }
    cluster_sync();
    u64 t = 0;
    for (int r = 0; r < C; ++r) t += peek(&(s.slot.*field), r);
    return t;
  };

  // Narrows down the element (in the vocabulary's order) at which the running count (MASS: weight, of elements above
  // `floor_key`) first exceeds `target`: `key` is its key, `ties` how many of the elements with that key lie up to and
  // including it, `equal` how many there are.  The running sum is known to exceed the target somewhere.
  auto narrow = [&](auto mass, u64 target, u64 all, uint32_t floor_key, uint32_t& key, u64& ties, uint32_t& equal) {
    constexpr bool MASS = decltype(mass)::value;
    u64 above = 0;
    uint32_t klo = MASS ? max(floor_key, 1u) : 1u, khi = key_of(top);
    float vlo = low;
    if (MASS) vlo = fmaxf(fmaxf(vlo, top - 124.0f / W.fc2), floor_key ? value_of(floor_key) : -INFINITY);
    // bins over the values: half the width, so that the difference of two finite numbers stays finite
    const float width = 0.5f * top - 0.5f * vlo, grain = width > 0.0f ? (float)kBins / width : 0.0f;
    const bool by_value = grain > 0.0f && grain < INFINITY;
    // round 0 of MASS adds weights as 32-bit numbers in units of `all` / 2^31 (which finds a few bins that must hold the
    // place), everything else is exact
    const float unit = MASS ? 2147483648.0f / (float)((double)all * ldexp(1.0, -a.frac)) : 0.0f;
    for (int round = 0; round < 8; ++round) {   // (a round over keys cuts their range by 1024: at most five)
      const bool value_bins = round == 0 && by_value, rough = MASS && round == 0;
      const uint32_t span = khi - klo;
      const int shift = max(0, 22 - __clz(span | 1u));   // (span >> shift) < 1024
      auto bin_of = [&](float x, uint32_t xk) -> int {
        if (value_bins) return (int)fminf((0.5f * top - 0.5f * x) * grain, (float)(kBins - 1));
        return (int)((khi - xk) >> shift);
      };
      auto candidate = [&](uint32_t xk) { return MASS && round == 0 ? xk > floor_key : (xk >= klo && xk <= khi); };
      const int limbs = MASS && !rough ? kLimbs : 1;
      for (int i = tid; i < limbs * kBins; i += kThreads) (&s.hist[0][0])[i] = 0;
      if (tid == 0) s.list_n = 0;
      __syncthreads();
      for (int blk = blk0; blk < blk1; ++blk) {
        float x[4];
        get4(blk, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t xk = key_of(x[e]);
          const bool in = xk != 0u && candidate(xk);
          if (rough) {
            const float w = in ? exp2f(W.log2f32(x[e])) * unit : 0.0f;
            if (w >= 1.0f) atomicAdd(&s.hist[0][bin_of(x[e], xk)], (uint32_t)w);
          } else if (!MASS) {
            // (equal logits, as bf16 has many of, meet in one bin: a warp that agrees adds once)
            const int bin = in ? bin_of(x[e], xk) : -1;
            const int lead = __shfl_sync(0xffffffffu, bin, 0);
            const unsigned same = __ballot_sync(0xffffffffu, bin == lead);
            if (same == 0xffffffffu) {
              if (lane == 0 && lead >= 0) atomicAdd(&s.hist[0][lead], 32u);
            } else if (in) {
              atomicAdd(&s.hist[0][bin], 1u);
            }
          } else if (in) {
            const int bin = bin_of(x[e], xk);
            u64 w = W(x[e]);
#pragma unroll
            for (int l = 0; l < kLimbs; ++l, w >>= kLimbBits)
              if (w & ((1u << kLimbBits) - 1u)) atomicAdd(&s.hist[l][bin], (uint32_t)w & ((1u << kLimbBits) - 1u));
          }
        }
      }
      cluster_sync();
      // each CTA adds up a slice of the bins over the cluster and hands it to everyone
      for (int i = rank * (kBins / C) + tid; i < (rank + 1) * (kBins / C); i += kThreads) {
        u64 t = 0;
        for (int l = 0; l < limbs; ++l) {
          u64 x = 0;
          for (int r = 0; r < C; ++r) x += peek(&s.hist[l][i], r);
          t += x << (l * kLimbBits);
        }
        for (int r = 0; r < C; ++r) poke(&s.total[i], r, t);
      }
      if (tid == 0) {
        s.pick_lo = kBins - 1;
        s.pick_hi = kBins - 1;
        s.pick_above = 0;
      }
      cluster_sync();
      {
        constexpr int E = kBins / kThreads;
        u64 x[E], sum = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) sum += x[e] = s.total[tid * E + e];
        u64 inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        if (lane == 31) s.scan[warp] = inc;
        __syncthreads();
        u64 run = inc - sum;
        for (int w = 0; w < warp; ++w) run += s.scan[w];
        // a rough sum is short by less than one unit an element and off by 2^-16 of itself
        const u64 want = rough ? (u64)((double)target / (double)all * 2147483648.0) : target - above;
        const u64 slack_lo = rough ? (u64)V + (1u << 15) : 0, slack_hi = rough ? (1u << 15) + 1 : 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const u64 next = run + x[e];
          if (run + slack_lo <= want && next + slack_lo > want) {
            s.pick_lo = tid * E + e;
            s.pick_above = run;
          }
          if (tid * E + e == 0 && slack_lo > want) s.pick_lo = 0;
          if (run <= want + slack_hi && next > want + slack_hi) s.pick_hi = tid * E + e;
          run = next;
        }
        __syncthreads();
      }
      const int lo = s.pick_lo, hi = max(lo, s.pick_hi);
      if (!rough) above += s.pick_above;
      // what lies in those bins, and (after a rough round) the exact weight of what lies in front of them
      u64 front = 0;
      uint32_t n = 0, kmin = 0xffffffffu, kmax = 0;
      for (int blk = blk0; blk < blk1; ++blk) {
        float x[4];
        get4(blk, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t xk = key_of(x[e]);
          if (xk == 0u || !candidate(xk)) continue;
          const int bin = bin_of(x[e], xk);
          if (bin < lo) {
            if (rough) front += W(x[e]);
          } else if (bin <= hi) {
            ++n;
            kmin = min(kmin, xk);
            kmax = max(kmax, xk);
            const int at = atomicAdd(&s.list_n, 1);
            if (at < kList) {
              s.list_key[at] = xk;
              s.list_at[at] = base + blk * kBlock + 4 * lane + e;
            }
          }
        }
      }
      front = warp_add(front);
      n = __reduce_add_sync(0xffffffffu, n);
      kmin = __reduce_min_sync(0xffffffffu, kmin);
      kmax = __reduce_max_sync(0xffffffffu, kmax);
      if (lane == 0) {
        s.red[warp].above = front;
        s.red[warp].n = n;
        s.red[warp].kmin = kmin;
        s.red[warp].kmax = kmax;
      }
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < kWarps; ++w) {
          front += s.red[w].above;
          n += s.red[w].n;
          kmin = min(kmin, s.red[w].kmin);
          kmax = max(kmax, s.red[w].kmax);
        }
        s.slot.above = front;
        s.slot.n = n;
        s.slot.kmin = kmin;
        s.slot.kmax = kmax;
      }
      cluster_sync();
      u64 ahead = 0;
      n = 0;
      kmin = 0xffffffffu;
      kmax = 0;
      int off = 0;
      for (int r = 0; r < C; ++r) {
        ahead += peek(&s.slot.above, r);
        const uint32_t nr = peek(&s.slot.n, r);
        if (r < rank) off += (int)nr;
        n += nr;
        kmin = min(kmin, peek(&s.slot.kmin, r));
        kmax = max(kmax, peek(&s.slot.kmax, r));
      }
      if (rough) above = ahead;
      if (n == 0) {   // (not reached while the sums say that the place is there)
        key = klo;
        ties = 0;
        equal = 0;
        return;
      }
      if (kmin == kmax) {
        key = kmin;
        equal = n;
        const u64 w = MASS ? W(value_of(kmin)) : 1;
        ties = w ? (target - above) / w + 1 : n;
        if (ties > n) ties = n;
        return;
      }
      if (n <= kList) {   // rank them: every CTA gathers all lists
        for (int r = 0, o = 0; r < C; ++r) {
          const int nr = (int)peek(&s.slot.n, r);
          for (int i = tid; i < nr; i += kThreads) {
            const uint32_t xk = peek(&s.list_key[i], r);
            s.all_key[o + i] = xk;
            s.all_at[o + i] = (int)peek(reinterpret_cast<const uint32_t*>(&s.list_at[i]), r);
            s.all_w[o + i] = MASS ? W(value_of(xk)) : 1;
          }
          o += nr;
        }
        __syncthreads();
        if (tid < (int)n) {
          const uint32_t xk = s.all_key[tid];
          const int at = s.all_at[tid];
          u64 before = above;
          uint32_t eq = 0, eq_before = 0;
          for (int i = 0; i < (int)n; ++i) {
            const uint32_t yk = s.all_key[i];
            const bool ahead_of = yk > xk || (yk == xk && s.all_at[i] < at);
            if (ahead_of) before += s.all_w[i];
            eq += yk == xk;
            eq_before += yk == xk && ahead_of;
          }
          if (before <= target && target < before + s.all_w[tid]) {
            s.pick_key = xk;
            s.pick_ties = eq_before + 1;
            s.slot.eq = eq;
          }
        }
        __syncthreads();
        key = s.pick_key;
        ties = s.pick_ties;
        equal = s.slot.eq;
        cluster_sync();   // the lists have been read
        return;
      }
      klo = kmin;
      khi = kmax;
    }
    key = klo;
    ties = equal = 0;
  };

  // ---- threshold
  uint32_t t = 0u, equal = 0;
  u64 ties = 0;   // t = 0: everything above -infinity is kept
  if (k < V) {
    // (fewer than k elements above -infinity: all of them stay)
    u64 n = 0;
    for (int blk = blk0; blk < blk1; ++blk) {
      float x[4];
      get4(blk, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) n += x[e] > -INFINITY;
    }
    n = cluster_total(n, &Slot::count);
    if ((u64)k < n) narrow(std::false_type{}, (u64)k - 1, 0, 0u, t, ties, equal);
  }
  if (p < 1.0f) {
    u64 z = 0;
    for (int blk = blk0; blk < blk1; ++blk) {
      float x[4];
      get4(blk, x);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (key_of(x[e]) > t) z += W(x[e]);
    }
    const u64 strictly = cluster_total(z, &Slot::mass);
    const u64 wt = t ? W(value_of(t)) : 0, all = strictly + ties * wt;
    const u64 target = p > 0.0f ? __umul64hi((u64)((double)p * 18446744073709551616.0), all) : 0;
    if (target < strictly) {
      uint32_t t2;
      narrow(std::true_type{}, target, strictly, t, t2, ties, equal);
      t = t2;
    } else if (wt) {   // the border lies among the ties of top-k
      ties = min(ties, (target - strictly) / wt + 1);
    }
  }
  const bool some = t != 0u && ties < equal;   // only the first of the elements that equal the threshold stay
  u64 seen0 = 0;                               // ties in front of this warp's part
  if (some) {
    uint32_t eq = 0;
    for (int blk = blk0; blk < blk1; ++blk) {
      float x[4];
      get4(blk, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) eq += key_of(x[e]) == t;
    }
    eq = __reduce_add_sync(0xffffffffu, eq);
    __syncthreads();
    if (lane == 0) s.warp_eq[warp] = eq;
    __syncthreads();
    if (tid == 0) {
      uint32_t e = 0;
      for (int w = 0; w < kWarps; ++w) e += s.warp_eq[w];
      s.slot.eq = e;
    }
    cluster_sync();
    for (int r = 0; r < rank; ++r) seen0 += peek(&s.slot.eq, r);
    for (int w = 0; w < warp; ++w) seen0 += s.warp_eq[w];
  }
  // ---- kept weights in index order
  const u64 mfix = mp > 0.0f ? (u64)((double)mp * ldexp(1.0, a.frac)) : 0;
  auto kept4 = [&](int blk, u64& seen, u64 (&w)[4]) {
    float x[4];
    get4(blk, x);
    u64 rank4 = 0;
    uint32_t mine = 0;
    if (some) {
#pragma unroll
      for (int e = 0; e < 4; ++e) mine += key_of(x[e]) == t;
      uint32_t inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      rank4 = seen + inc - mine;
      seen += __shfl_sync(0xffffffffu, inc, 31);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t xk = key_of(x[e]);
      bool keep = xk > t || (t && xk == t);
      if (some && xk == t) keep = rank4++ < ties;
      w[e] = 0;
      if (keep && xk) {
        w[e] = W(x[e]);
        if (mp > 0.0f) {
          const long long d = (long long)(w[e] - mfix);
          const long long near = (long long)(mfix >> 26) + 2;
          bool ok = d >= 0;
          if (d <= near && d >= -near) ok = exp(((double)x[e] - W.max) / (double)temp) >= (double)mp;   // next to the border: in 64 bits
          if (!ok) w[e] = 0;
        }
      }
    }
  };
  u64 sum = 0, seen = seen0;
  for (int blk = blk0; blk < blk1; ++blk) {
    u64 w[4];
    kept4(blk, seen, w);
    sum += (w[0] + w[1]) + (w[2] + w[3]);
  }
  sum = warp_add(sum);
  __syncthreads();
  if (lane == 0) s.warp_sum[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    u64 x = 0;
    for (int w = 0; w < kWarps; ++w) x += s.warp_sum[w];
    s.slot.sum = x;
  }
  cluster_sync();
  u64 z = 0, ahead = 0;
  for (int r = 0; r < C; ++r) {
    const u64 x = peek(&s.slot.sum, r);
    if (r < rank) ahead += x;
    z += x;
  }
  for (int w = 0; w < warp; ++w) ahead += s.warp_sum[w];
  const float u = a.u[b];
  const double uu = u >= 0.0f ? fmin((double)u, 1.0 - 0x1p-24) : 0.0;
  const u64 target = __umul64hi((u64)(uu * 18446744073709551616.0), z);
  if (ahead <= target && target < ahead + sum) {   // the warp that holds the token
    seen = seen0;
    for (int blk = blk0; blk < blk1; ++blk) {
      u64 w[4];
      kept4(blk, seen, w);
      const u64 mine = (w[0] + w[1]) + (w[2] + w[3]);
      u64 inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, ahead + inc > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          u64 run = ahead + inc - mine;
          int e = 0;
          for (; e < 3 && run + w[e] <= target; ++e) run += w[e];
          a.tokens[b] = base + blk * kBlock + 4 * lane + e;
          if (a.probs) a.probs[b] = (float)((double)w[e] / (double)z);
        }
        break;
      }
      ahead += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  cluster_sync();   // (the others may still be reading this CTA's slot)
}

static int fail(int code, const char* msg) {
  fsvd_tile_set_error(code, msg);
  return code;
}

}  // namespace fsvd_sample_impl

extern "C" int fsvd_sample(const void* logits, long long row_stride, int dtype, const float* uniforms, const float* temperature,
                           const int* top_k, const float* top_p, const float* min_p, float temperature_all, int top_k_all,
                           float top_p_all, float min_p_all, int* tokens, float* probs, int B, int V, void* stream) {
  using namespace fsvd_sample_impl;
  if (!logits || !uniforms || !tokens) return fail(FSVD_ERR_ARG, "null argument");
  if (dtype != FSVD_DTYPE_F32 && dtype != FSVD_DTYPE_BF16) return fail(FSVD_ERR_ARG, "logits are float32 or bfloat16");
  if (B < 0 || V < 1 || row_stride < 0) return fail(FSVD_ERR_ARG, "bad sizes");
  if (V > kMaxVocab) return fail(FSVD_ERR_UNSUPPORTED, "a vocabulary beyond 2^22 is unsupported");
  if (B > (1 << 24)) return fail(FSVD_ERR_UNSUPPORTED, "more than 2^24 rows are unsupported");
  if (temperature_all != temperature_all || top_p_all != top_p_all || min_p_all != min_p_all)
    return fail(FSVD_ERR_ARG, "NaN setting");
  if (B == 0) return 0;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  int bits = 0;
  while ((1 << bits) < V) ++bits;
  // CTAs of a row: enough that a piece is at most 50 KB (three CTAs per SM), and that few rows use the whole GPU as long
  // as a CTA has 2048 elements to work on.
  int C = 1;
  while (C < kMaxCluster && (V / C > 12800 || (B * C < sms && V / C > 2048))) C *= 2;
  Args a;
  a.logits = logits; a.stride = row_stride; a.u = uniforms; a.temperature = temperature; a.top_k = top_k; a.top_p = top_p;
  a.min_p = min_p; a.T_all = temperature_all; a.k_all = top_k_all; a.p_all = top_p_all; a.m_all = min_p_all;
  a.tokens = tokens; a.probs = probs; a.V = V; a.frac = std::min(46, 62 - bits);
  a.chunk = ((V + C - 1) / C + kBlock - 1) / kBlock * kBlock;
  const bool resident = a.chunk <= 48 * 1024;
  const size_t smem = resident ? (size_t)a.chunk * 4 : 0;
  const void* fn = dtype == FSVD_DTYPE_F32 ? (resident ? (const void*)sample_kernel<float, true> : (const void*)sample_kernel<float, false>)
                                           : (resident ? (const void*)sample_kernel<__nv_bfloat16, true>
                                                       : (const void*)sample_kernel<__nv_bfloat16, false>);
  cudaError_t e = cudaSuccess;
  if (smem > 16 * 1024) e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * C));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    void* params[] = {&a};
    e = cudaLaunchKernelExC(&cfg, fn, params);
  }
  if (e != cudaSuccess) {
    char msg[160];
    snprintf(msg, sizeof(msg), "kernel launch failed: %s", cudaGetErrorString(e));
    return fail(FSVD_ERR_CUDA, msg);
  }
  fsvd_tile_count_launch();
  return 0;
}

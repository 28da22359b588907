// Choice of the next token (fsvd_sample of include/flashsvd_b200.h): temperature, top-k, top-p, min-p, one uniform number.
//
// The vocabulary is ordered by logit (descending, lower index first); every filter keeps a prefix of that order, so the
// kept set is {key > t} and the first r of {key = t} in index order, for one threshold key t.  It is found without a
// sort: a histogram of 1024 bins over the values narrows the threshold to a few of them, and a hundred candidates are
// then ranked directly; where there are more, bins over the integer keys inside narrow it on.
//
// Weights exp((l - max) / T) are 64-bit numbers good to 2^-39, and every sum has a fixed order, or is one of integers where
// its terms come in any order.  32-bit weights would put a draw from a flat row of 10^5 tokens on another token than exact
// arithmetic once in 10^4 rows.
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
#include "fsvd_smem.h"
#include "fsvd_tc.cuh"
#include "fsvd_tile.h"

namespace fsvd_sample_impl {

typedef unsigned long long u64;
constexpr int kThreads = 1024, kWarps = kThreads / 32;
static_assert(kWarps == 32, "a warp folds one number of every warp");
constexpr int kBins = 1024;
constexpr int kPer = 32, kPerLog = 5;       // bins of a factor of two in the weight
constexpr int kFrac = 40;                   // bits of a weight as an integer, beside the largest candidate's (2^20 of them fit)
constexpr int kLimbs = 4, kLimbBits = 12;   // such an integer as four numbers of 12 bits: 2^20 of them fit 32-bit sums
constexpr int kList = 1024;                 // candidates of a CTA that are listed
constexpr int kRank = 192;                  // candidates of a row that are ranked directly
constexpr int kBlock = 128;                 // elements of a warp's step: four neighbours per lane
constexpr int kPackPiece = 256, kPackAlone = 896;   // elements that a warp's short list holds, beside the piece and without
constexpr int kMaxCluster = 8;
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxPiece = (1 << 17) + kBlock;        // elements of a CTA
constexpr u64 kMostUpper = 27802;                    // of what `masses` adds in 32 bits
static_assert(kMaxPiece * kMostUpper < (1ull << 32) && kMaxPiece * 16383ull < (1ull << 32));
constexpr float kHuge = 3.402823466e38f;

struct Args {
  const void* logits;
  long long stride;
  const float *u, *temperature, *top_p, *min_p;
  const int* top_k;
  float T_all, p_all, m_all;
  int k_all;
  int* tokens;
  float* probs;
  int V, chunk;   // chunk: elements of a CTA, a multiple of kBlock
};

// What a CTA shows to the others of its cluster (each number is written once between two reads by the others).
struct Slot {
  double count, mass, sum;
  float top, low;
  uint32_t first, finite, n, kmin, kmax, eq;
};

struct Shared {
  uint32_t hist[kLimbs][kBins];
  u64 total[kBins];
  double table[kPer];
  double warp_sum[kWarps], scan_d[kWarps];
  u64 scan[kWarps];
  uint32_t warp_eq[kWarps];
  uint32_t list_key[kList], list_at[kList];
  u64 all_key[kRank], all_w[kRank];
  Slot slot, red[kWarps];
  int pick, list_n;
  u64 pick_above;
  double pick_front;
  u64 pick_key;
};

// Ascending keys for ascending numbers above -infinity (the zeros share theirs); 0 for -infinity and NaN.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return !(x > -INFINITY) ? 0u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
__device__ __forceinline__ float num(float x) { return x; }
__device__ __forceinline__ float num(__nv_bfloat16 x) { return __bfloat162float(x); }

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
__device__ __forceinline__ float peek(const float* p, int rank) {
  return __uint_as_float(peek(reinterpret_cast<const uint32_t*>(p), rank));
}
__device__ __forceinline__ double peek(const double* p, int rank) {
  double x;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(x) : "r"(remote(p, rank)) : "memory");
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
template <typename N, typename F>
__device__ __forceinline__ N warp_fold(N x, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ double warp_add(double x) {
  return warp_fold(x, [](double p, double q) { return p + q; });
}
__device__ __forceinline__ float warp_min(float x) {
  return warp_fold(x, [](float p, float q) { return fminf(p, q); });
}
// Inclusive prefix sums over the lanes.
template <typename N>
__device__ __forceinline__ N warp_scan(N x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}
// fp32 -> fp64 of a finite number by its bits (the conversion instruction runs at an eighth of the rate of additions; a
// zero comes out as 2^-127, which no sum here sees)
__device__ __forceinline__ double wide(float x) {
  const uint32_t b = __float_as_uint(x);
  return __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(b << 29));
}

// exp((x - max) / T) = 2^(k / 32) 2^(r / 32) with k whole and |r| <= 1/2: a table of 32, a polynomial of degree four
// (Taylor; the next term is below 2^-39), and k / 32 into the exponent.  For x >= cut; callers raise what is below to it and
// drop the result, so that four weights are formed side by side without a branch (each is a chain of a dozen steps).
struct Weigher {
  double max, c;           // c = 32 log2(e) / T
  float cut;               // below it a weight is under 2^-60 and counts as zero; finite
  const double* table;     // 2^(j / 32)
  __device__ __forceinline__ double operator()(float x, int& bin, int& q) const {   // q: w = 2^(-bin / 32) (1 + q 2^-34)
    constexpr double magic = 6755399441055744.0, a = 0.69314718055994530942 / kPer;   // 1.5 * 2^52; ln(2) / 32
    const double d = wide(x) - max, k = fma(d, c, magic);
    const int lo = __double2loint(k);
    const double r = fma(d, c, -(k - magic));
    const double e = fma(r, fma(r, fma(r, fma(r, a * a * a * a / 24.0, a * a * a / 6.0), a * a / 2.0), a), 1.0);
    const double w = table[lo & (kPer - 1)] * e;
    bin = -lo;             // 32nds of a factor of two below the maximum
    q = __double2loint(e + 393216.0);   // (1.5 * 2^18: the low word counts 2^-34; |q| < 1.9e8 as |e - 1| < 0.011)
    return __hiloint2double(__double2hiint(w) + ((lo >> kPerLog) << 20), __double2loint(w));
  }
  __device__ __forceinline__ double operator()(float x, int& bin) const {
    int q;
    return (*this)(x, bin, q);   // (what nobody asks for costs nothing)
  }
  __device__ __forceinline__ int bin_of(float x) const { return -__double2loint(fma(wide(x) - max, c, 6755399441055744.0)); }
  __device__ __forceinline__ double operator()(float x) const {
    int bin;
    return x >= cut ? (*this)(x, bin) : 0.0;
  }
  __device__ __forceinline__ u64 fixed(float x, double one) const { return (u64)__double2ll_rn((*this)(x) * one); }
};

// (out of line: it is hardly ever called)
__device__ __noinline__ double library_exp(double x) { return exp(x); }

template <typename T, bool RESIDENT>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const Args a) {
  constexpr int kPack = RESIDENT ? kPackPiece : kPackAlone;
  // short lists of the warps (what may still be kept, in index order): values, and places in the warp's part; then, if
  // RESIDENT, this CTA's elements as they are in memory
  extern __shared__ __align__(16) unsigned char dynamic[];
  unsigned char* piece = dynamic + kWarps * kPack * 6;
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  const int rank = cluster_rank(), C = cluster_size(), b = blockIdx.x / C;
  const T* row = reinterpret_cast<const T*>(a.logits) + (size_t)b * a.stride;
  // Elements are counted from the 16-byte boundary in front of the row: place i is element i - shift.
  constexpr int kVec = 16 / sizeof(T);
  const int shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  row -= shift;
  const int base = rank * a.chunk, i_end = min(base + a.chunk, V + shift), i_begin = max(base, shift);
  const int len = max(0, i_end - base);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid < kPer) s.table[tid] = exp2((double)tid / kPer);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float temp = fminf(a.temperature ? a.temperature[b] : a.T_all, kHuge);
  if (temp > 0.0f) temp = fmaxf(temp, 0x1p-64f);   // (`wide` makes a zero +-2^-127, which has to stay nothing beside it)
  int k = a.top_k ? a.top_k[b] : a.k_all;
  const float p = a.top_p ? a.top_p[b] : a.p_all, mp = fminf(a.min_p ? a.min_p[b] : a.m_all, 1.0f);
  if (k <= 0 || k > V) k = V;

  // ---- the row into shared memory: whole 16-byte pieces asynchronously, the ragged ends one by one
  const int nblk = (len + kBlock - 1) / kBlock, per = (nblk + kWarps - 1) / kWarps;
  const int blk0 = min(nblk, warp * per), blk1 = min(nblk, blk0 + per);
  if constexpr (RESIDENT) {
    T* vals = reinterpret_cast<T*>(piece);
    for (int v = tid; v < nblk * (kBlock / kVec); v += kThreads) {
      const int i = base + v * kVec;
      if (i >= i_begin && i + kVec <= i_end) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(fsvd_tile::smem_u32(vals + v * kVec)), "l"(row + i) : "memory");
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          vals[v * kVec + e] = i + e >= i_begin && i + e < i_end ? row[i + e] : T(-INFINITY);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
  }
  // a barrier of the cluster (a CTA by itself has a cheaper one)
  auto meet = [&] {
    if (C > 1) fsvd_tile::cluster_sync();
    else __syncthreads();
  };
  bool inf = false;   // an infinite maximum: the elements that equal it share everything, the others get nothing
  float* short_x = reinterpret_cast<float*>(dynamic) + warp * kPack;
  uint16_t* short_at = reinterpret_cast<uint16_t*>(dynamic + kWarps * kPack * 4) + warp * kPack;
  int packed = -1;   // elements in the warp's short list; -1: the warp goes through all of its part
  auto get4 = [&](int blk, float (&x)[4]) {
    const int v = blk * kBlock + 4 * lane;
    if constexpr (RESIDENT && sizeof(T) == 4) {
      const float4 f = *reinterpret_cast<const float4*>(piece + 4 * v);
      x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
    } else if constexpr (RESIDENT) {
      const uint2 w = *reinterpret_cast<const uint2*>(piece + 2 * v);
      x[0] = __uint_as_float(w.x << 16); x[1] = __uint_as_float(w.x & 0xffff0000u);
      x[2] = __uint_as_float(w.y << 16); x[3] = __uint_as_float(w.y & 0xffff0000u);
    } else {
      const int i = base + v;
      if (i >= i_begin && i + 4 <= i_end) {
        if constexpr (sizeof(T) == 4) {
          const float4 f = __ldg(reinterpret_cast<const float4*>(row + i));
          x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
        } else {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(row + i));
          x[0] = __uint_as_float(w.x << 16); x[1] = __uint_as_float(w.x & 0xffff0000u);
          x[2] = __uint_as_float(w.y << 16); x[3] = __uint_as_float(w.y & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = i + e >= i_begin && i + e < i_end ? num(row[i + e]) : -INFINITY;
      }
    }
  };
  // fn(block, its four elements of this lane) for the blocks [first, end): from memory two blocks are under way.
  auto each = [&](int first, int end, auto fn) {
    if (packed >= 0) {
      for (int blk = 0; blk * kBlock < packed; ++blk) {
        const float4 f = *reinterpret_cast<const float4*>(short_x + blk * kBlock + 4 * lane);
        const float x[4] = {f.x, f.y, f.z, f.w};
        fn(blk, x);
      }
      return;
    }
    auto call = [&](int blk, float (&x)[4]) {
      if (inf) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = x[e] == INFINITY ? 0.0f : -INFINITY;
      }
      fn(blk, x);
    };
    if constexpr (RESIDENT) {
      for (int blk = first; blk < end; ++blk) {
        float x[4];
        get4(blk, x);
        call(blk, x);
      }
    } else {
      constexpr int D = 2;
      float ahead[D][4], x[4];
#pragma unroll
      for (int d = 0; d < D; ++d)
        if (first + d < end) get4(first + d, ahead[d]);
      for (int blk = first; blk < end; ++blk) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = ahead[0][e];
#pragma unroll
          for (int d = 0; d + 1 < D; ++d) ahead[d][e] = ahead[d + 1][e];
        }
        if (blk + D < end) get4(blk + D, ahead[D - 1]);
        call(blk, x);
      }
    }
  };
  auto index_of = [&](int blk, int e) {
    if (packed >= 0) return base + blk0 * kBlock + (int)short_at[blk * kBlock + 4 * lane + e] - shift;
    return base + blk * kBlock + 4 * lane + e - shift;
  };
  // Building the short list while a pass goes through the part: the elements with in[], in order.
  int filling = 0;
  auto pack = [&](int blk, const float (&x)[4], const bool (&in)[4]) {
    const uint32_t in_front = (1u << lane) - 1u;
    uint32_t who[4];
    int at = filling;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      who[e] = __ballot_sync(0xffffffffu, in[e]);
      at += __popc(who[e] & in_front);
      filling += __popc(who[e]);
    }
    if (filling > kPack) return;   // (a list that is too short is not used)
    const int place = (blk - blk0) * kBlock + 4 * lane;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (in[e]) {
        short_x[at] = x[e];
        short_at[at] = (uint16_t)(place + e);
        ++at;
      }
  };
  auto use_pack = [&] {
    if (filling <= kPack && per * kBlock <= 65536) {
      for (int i = filling + lane; i < (filling + kBlock - 1) / kBlock * kBlock; i += 32) short_x[i] = -INFINITY;
      packed = filling;
    }
    __syncwarp();
  };

  // ---- the largest element (a maximum passes over NaN)
  const auto larger = [](float x, float y) { return fmaxf(x, y); };
  float top = -INFINITY, low = INFINITY;   // for top-k also the smallest above -infinity, and how many there are
  uint32_t finite = 0;
  each(blk0, blk1, [&](int blk, const float (&x)[4]) {
    top = fmaxf(top, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    if (k < V) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = x[e] > -INFINITY;
        finite += in;
        low = fminf(low, in ? x[e] : INFINITY);
      }
    }
  });
  top = warp_fold(top, larger);
  low = warp_min(low);
  finite = __reduce_add_sync(0xffffffffu, finite);
  if (lane == 0) {
    s.red[warp].top = top;
    s.red[warp].low = low;
    s.red[warp].finite = finite;
  }
  __syncthreads();
  if (warp == 0) {
    top = warp_fold(s.red[lane].top, larger);
    low = warp_min(s.red[lane].low);
    finite = __reduce_add_sync(0xffffffffu, s.red[lane].finite);
    if (lane == 0) {
      s.slot.top = top;
      s.slot.low = low;
      s.slot.finite = finite;
    }
  }
  meet();
  top = peek(&s.slot.top, lane % C);
  low = peek(&s.slot.low, lane % C);
  finite = peek(&s.slot.finite, lane % C);
  top = warp_fold(top, larger);
  low = warp_min(low);
  finite = __reduce_add_sync(0xffffffffu, lane < C ? finite : 0u);
  if (top == -INFINITY || !(temp > 0.0f) || k == 1) {
    uint32_t first = 0xffffffffu;   // the lowest index that holds it
    each(blk0, top > -INFINITY ? blk1 : blk0, [&](int blk, const float (&x)[4]) {
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (x[e] == top) first = min(first, (uint32_t)index_of(blk, e));
    });
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) s.red[warp].first = first;
    __syncthreads();
    if (warp == 0) {
      first = __reduce_min_sync(0xffffffffu, s.red[lane].first);
      if (lane == 0) s.slot.first = first;
    }
    meet();
    if (rank == 0 && warp == 0) {
      first = __reduce_min_sync(0xffffffffu, peek(&s.slot.first, lane % C));
      if (lane == 0) {
        a.tokens[b] = top > -INFINITY ? (int)first : 0;
        if (a.probs) a.probs[b] = top > -INFINITY ? 1.0f : 0.0f;
      }
    }
    meet();   // (rank 0 reads the others' slots)
    return;
  }
  inf = top == INFINITY;
  if (inf) top = low = 0.0f;
  Weigher W;
  W.max = wide(top);
  W.c = kPer * 1.4426950408889634074 / (double)temp;
  const double octave = (double)temp * 0.69314718055994530942;   // a factor of two in the weight
  W.cut = fmaxf((float)(W.max - 60.0 * octave), -kHuge);
  W.table = s.table;

  // The least number from W.cut on whose bin is at most `bin`.  Bins fall with the number, so 32 lanes narrow the range of
  // keys 33 times a step; first the 32 keys around the place by the formula.
  auto least_of = [&](int bin) -> float {
    uint32_t lo = key_of(W.cut), hi = key_of((float)W.max);   // lo: not yet, unless W.cut itself is; hi: is
    if (W.bin_of(W.cut) <= bin) return W.cut;
    const uint32_t guess = key_of(fmaxf(W.cut, fminf((float)W.max, (float)(W.max - ((double)bin + 0.5) * (octave / kPer)))));
    uint32_t from = max(lo, guess > 16 ? guess - 16 : 0u), step = 1;
    while (hi - lo > 1) {
      const uint32_t mine = from + step * (uint32_t)lane;
      const unsigned is = __ballot_sync(0xffffffffu, mine < hi && mine > lo && W.bin_of(value_of(mine)) <= bin);
      const unsigned in = __ballot_sync(0xffffffffu, mine < hi && mine > lo);
      if (is) hi = from + step * (uint32_t)(__ffs(is) - 1);
      if (in & ~is) lo = from + step * (uint32_t)(31 - __clz(in & ~is));
      step = (hi - lo + 32) / 33;
      from = lo + step;
    }
    return value_of(hi);
  };
  // Sum over the cluster of one number per thread.
  auto cluster_total = [&](double x, double Slot::* field) -> double {
    x = warp_add(x);
    if (lane == 0) s.scan_d[warp] = x;
    __syncthreads();
    if (warp == 0) {
      x = warp_add(s.scan_d[lane]);
      if (lane == 0) s.slot.*field = x;
    }
    meet();
    return warp_add(lane < C ? peek(&(s.slot.*field), lane) : 0.0);
  };
  auto clear_hist = [&](int limbs) {
    for (int i = tid; i < limbs * kBins; i += kThreads) (&s.hist[0][0])[i] = 0;
    if (tid == 0) s.list_n = 0;
    __syncthreads();
  };
  // The histograms of the cluster added up, in everyone's `total`: each CTA takes a slice of the bins.
  auto merge_hist = [&](auto combine) {
    meet();
    // (C neighbouring lanes to a bin, each reads its CTA's numbers and writes its CTA's total)
    for (int j = tid; j < kBins; j += kThreads) {
      const int i = rank * (kBins / C) + j / C, r = j % C;
      u64 t = combine(i, r);
      for (int o = C >> 1; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      poke(&s.total[i], r, t);
    }
    if (tid == 0) {
      s.pick = kBins - 1;
      s.pick_above = 0;
      s.pick_front = 0.0;
    }
    meet();
  };
  auto counts = [&](int i, int r) -> u64 { return peek(&s.hist[0][i], r); };
  auto limbs = [&](int i, int r) -> u64 {
    u64 t = 0;
#pragma unroll
    for (int l = 0; l < kLimbs; ++l) t += (u64)peek(&s.hist[l][i], r) << (l * kLimbBits);
    return t;
  };
  // A weight of bin i is 2^(-i / 32) (1 + q 2^-34): the bin holds how many there are, and the sums of the 14 lower bits and
  // the upper ones (at most (2^34 (2^(1/64) - 1) + 2^28) / 2^14 = kMostUpper) of q + 2^28.  In units of 2^(-i / 32) 2^-34:
  auto masses = [&](int i, int r) -> u64 {
    return (u64)peek(&s.hist[0][i], r) * ((1ull << 34) - (1ull << 28)) + ((u64)peek(&s.hist[2][i], r) << 14) + peek(&s.hist[1][i], r);
  };
  // The bin at which the running sum of f(total, bin) first exceeds `want`, and the sum in front of it.
  auto find_bin = [&](auto zero, auto f, decltype(zero) want, auto* scan, decltype(zero)& in_front) -> int {
    using N = decltype(zero);
    constexpr int E = kBins / kThreads;
    N x[E], sum = zero;
#pragma unroll
    for (int e = 0; e < E; ++e) sum += x[e] = f(s.total[tid * E + e], tid * E + e);
    const N inc = warp_scan(sum, lane), left = __shfl_up_sync(0xffffffffu, inc, 1);
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    const N upto = warp_scan(scan[lane], lane), all = __shfl_sync(0xffffffffu, upto, kWarps - 1);
    N run = __shfl_sync(0xffffffffu, upto, max(warp - 1, 0));
    run = (warp ? run : zero) + (lane ? left : zero);   // (not inc - sum: a bin that nobody counted stands for more than all others)
    // (a sum that was formed in another order may end a rounding short of the place)
    if constexpr (std::is_integral_v<N>) want = all > 0 ? min(want, all - 1) : want;
    else want = fmin(want, all);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (run <= want && run + x[e] > want) {
        s.pick = tid * E + e;
        if constexpr (std::is_integral_v<N>) s.pick_above = run;
        else s.pick_front = run;
      }
      run += x[e];
    }
    __syncthreads();
    if constexpr (std::is_integral_v<N>) in_front = s.pick_above;
    else in_front = s.pick_front;
    return s.pick;
  };

  // Candidates of a narrowing step: how many, their keys' range, and (in any order) the first kList of them.
  struct Found { uint32_t n, kmin, kmax; };
  auto note = [&](Found& f, uint32_t xk, int at) {
    ++f.n;
    f.kmin = min(f.kmin, xk);
    f.kmax = max(f.kmax, xk);
    if (*reinterpret_cast<volatile int*>(&s.list_n) > kList) return;
    const int i = atomicAdd(&s.list_n, 1);
    if (i < kList) {
      s.list_key[i] = xk;
      s.list_at[i] = (uint32_t)at;
    }
  };
  // Adds up Found over the cluster.
  auto gather = [&](Found& f) {
    f.n = __reduce_add_sync(0xffffffffu, f.n);
    f.kmin = __reduce_min_sync(0xffffffffu, f.kmin);
    f.kmax = __reduce_max_sync(0xffffffffu, f.kmax);
    if (lane == 0) {
      Slot& r = s.red[warp];
      r.n = f.n; r.kmin = f.kmin; r.kmax = f.kmax;
    }
    __syncthreads();
    if (warp == 0) {
      const Slot& r = s.red[lane];
      const uint32_t n = __reduce_add_sync(0xffffffffu, r.n);
      const uint32_t lo = __reduce_min_sync(0xffffffffu, r.kmin), hi = __reduce_max_sync(0xffffffffu, r.kmax);
      if (lane == 0) {
        s.slot.n = n; s.slot.kmin = lo; s.slot.kmax = hi;
      }
    }
    meet();
    const int r = lane % C;
    const uint32_t n = peek(&s.slot.n, r), lo = peek(&s.slot.kmin, r), hi = peek(&s.slot.kmax, r);
    f.n = __reduce_add_sync(0xffffffffu, lane < C ? n : 0u);
    f.kmin = __reduce_min_sync(0xffffffffu, lo);
    f.kmax = __reduce_max_sync(0xffffffffu, hi);
  };
  uint32_t t = 0u, equal = 0;   // threshold key (0: everything above -infinity is kept), elements that have it
  uint32_t ties = 0;            // and how many of them are kept, the first ones in index order
  // Goes on inside the candidates f: the element at which the running count (MASS: weight) exceeds `target`, `above` of
  // it lies in front of them.  Counts are whole numbers; weights are added as integers here, in units that give the largest
  // candidate kFrac bits: a border far down in the tail is as sharp as one among the likely tokens.
  auto finish = [&](auto mass, Found f, double above, double target) {
    constexpr bool MASS = decltype(mass)::value;
    for (int round = 0; round < 5; ++round) {   // (a round cuts the range of the keys by 1024: at most four)
      if (f.n == 0) return;   // (not reached: the place is known to be there)
      double one = 1.0;
      if constexpr (MASS)   // 2^kFrac over the largest weight's power of two
        one = __hiloint2double((1023 + 1022 + kFrac - (__double2hiint(W(value_of(f.kmax))) >> 20)) << 20, 0);
      const double left = (target - above) * one;
      const u64 want = left > 0.0 ? (u64)left : 0;
      if (f.kmin == f.kmax) {
        const u64 w = MASS ? W.fixed(value_of(f.kmin), one) : 1;
        t = f.kmin;
        equal = f.n;
        ties = w ? (uint32_t)min(want / w + 1, (u64)f.n) : f.n;
        return;
      }
      if (f.n <= kRank) {   // every CTA gathers all lists and ranks them
        const int upto = warp_scan(lane < C ? (int)peek(&s.slot.n, lane % C) : 0, lane);
        int from = 0, r = 0;   // the list that entry `tid` of all of them is in, and where it begins
        for (int c = 0; c + 1 < C; ++c) {
          const int end = __shfl_sync(0xffffffffu, upto, c);
          if (tid >= end) {
            from = end;
            r = c + 1;
          }
        }
        if (tid < (int)f.n) {
          const uint32_t xk = peek(&s.list_key[tid - from], r);
          s.all_key[tid] = ((u64)xk << 32) | ~peek(&s.list_at[tid - from], r);   // larger: in front
          s.all_w[tid] = MASS ? W.fixed(value_of(xk), one) : 1;
        }
        __syncthreads();
        for (int c0 = 4 * warp; c0 < (int)f.n; c0 += 4 * kWarps) {   // eight lanes to a candidate, over all of them
          const int c = min(c0 + lane / 8, (int)f.n - 1);
          const u64 key = s.all_key[c];
          u64 before = 0;
          uint32_t place = 0;
#pragma unroll 4
          for (int i = lane & 7; i < (int)f.n; i += 8)
            if (s.all_key[i] > key) {
              before += s.all_w[i];
              ++place;
            }
#pragma unroll
          for (int o = 1; o < 8; o *= 2) {
            before += __shfl_xor_sync(0xffffffffu, before, o);
            place += __shfl_xor_sync(0xffffffffu, place, o);
          }
          if (before <= want && (want < before + s.all_w[c] || place + 1 == f.n)) s.pick_key = key;
        }
        __syncthreads();
        const u64 key = s.pick_key;
        uint32_t eq = 0, eq_upto = 0;
        for (int i = lane; i < (int)f.n; i += 32) {
          const bool same = (uint32_t)(s.all_key[i] >> 32) == (uint32_t)(key >> 32);
          eq += same;
          eq_upto += same && s.all_key[i] >= key;
        }
        t = (uint32_t)(key >> 32);
        ties = __reduce_add_sync(0xffffffffu, eq_upto);
        equal = __reduce_add_sync(0xffffffffu, eq);
        meet();   // the lists have been read
        return;
      }
      // the list takes the place of the row where it holds all of this CTA's candidates: one to a thread
      static_assert(kList == kThreads);
      const bool listed = s.list_n <= kList;
      const uint32_t my_key = listed && tid < s.list_n ? s.list_key[tid] : 0u, my_at = listed && tid < s.list_n ? s.list_at[tid] : 0u;
      __syncthreads();
      const uint32_t klo = f.kmin, khi = f.kmax;
      const int by = max(0, 22 - __clz((khi - klo) | 1u));   // (khi - klo) >> by < 1024
      clear_hist(MASS ? kLimbs : 1);
      auto add = [&](uint32_t xk) {
        if (xk < klo || xk > khi) return;
        const int bin = (int)((khi - xk) >> by);
        if constexpr (MASS) {
          u64 w = W.fixed(value_of(xk), one);
#pragma unroll
          for (int l = 0; l < kLimbs; ++l, w >>= kLimbBits)
            if (w & ((1u << kLimbBits) - 1u)) atomicAdd(&s.hist[l][bin], (uint32_t)w & ((1u << kLimbBits) - 1u));
        } else {
          atomicAdd(&s.hist[0][bin], 1u);
        }
      };
      if (listed) {
        add(my_key);
      } else {
        each(blk0, blk1, [&](int, const float (&x)[4]) {
#pragma unroll 1
          for (int e = 0; e < 4; ++e) add(key_of(e == 0 ? x[0] : e == 1 ? x[1] : e == 2 ? x[2] : x[3]));
        });
      }
      if constexpr (MASS) merge_hist(limbs);
      else merge_hist(counts);
      u64 in_front;
      const int bin = find_bin((u64)0, [](u64 x, int) { return x; }, want, s.scan, in_front);
      above += (double)in_front / one;
      f = Found{0u, 0xffffffffu, 0u};
      auto inside = [&](uint32_t xk) { return xk >= klo && xk <= khi && (int)((khi - xk) >> by) == bin; };
      if (listed) {
        if (inside(my_key)) note(f, my_key, (int)my_at);
      } else {
        each(blk0, blk1, [&](int blk, const float (&x)[4]) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t xk = key_of(x[e]);
            if (inside(xk)) note(f, xk, index_of(blk, e));
          }
        });
      }
      gather(f);
    }
  };

  // ---- top-k (fewer than k elements above -infinity: all of them stay; an infinite maximum: so do its equals, unless
  // there are more than k)
  if (k < V) {
    uint32_t n = finite;
    if (inf) {
      uint32_t m = 0;
      each(blk0, blk1, [&](int blk, const float (&x)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) m += x[e] == 0.0f;
      });
      n = (uint32_t)cluster_total((double)m, &Slot::count);
    }
    clear_hist(1);
    if ((uint32_t)k < n) {
      // bins over the values (of halves: the difference of two finite numbers stays finite)
      const float width = 0.5f * top - 0.5f * low, grain = (float)kBins / width;
      Found f{0u, 0xffffffffu, 0u};
      double above = 0.0;
      int bin = -1;
      auto bin_of = [&](float x) { return (int)fminf((0.5f * top - 0.5f * x) * grain, (float)(kBins - 1)); };
      const bool by_value = width > 0.0f && grain < INFINITY;
      if (by_value) {
        each(blk0, blk1, [&](int blk, const float (&x)[4]) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (x[e] > -INFINITY) atomicAdd(&s.hist[0][bin_of(x[e])], 1u);   // (NaN fails the comparison)
        });
        merge_hist(counts);
        u64 in_front;
        bin = find_bin((u64)0, [](u64 x, int) { return x; }, (u64)k - 1, s.scan, in_front);
        above = (double)in_front;
      }
      each(blk0, blk1, [&](int blk, const float (&x)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (x[e] > -INFINITY && (!by_value || bin_of(x[e]) == bin)) note(f, key_of(x[e]), index_of(blk, e));
        bool in[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) in[e] = x[e] > -INFINITY && by_value && bin_of(x[e]) <= bin;
        if (__any_sync(0xffffffffu, in[0] || in[1] || in[2] || in[3])) pack(blk, x, in);
      });
      if (by_value) use_pack();
      gather(f);
      finish(std::false_type{}, f, above, (double)(k - 1));
    }
  }
  // ---- top-p
  bool tried = false;   // to list what top-p keeps
  if (p < 1.0f) {
    const float tv = t ? value_of(t) : -INFINITY;
    // the mass above the threshold so far, and its distribution over 32nds of a factor of two (the last bin is everything
    // below 2^-32, which is hardly ever where the border lies: nobody counts it, half a row may add to one number)
    double z = 0.0;
    clear_hist(3);
    each(blk0, blk1, [&](int, const float (&x)[4]) {
      bool in[4];
      int bin[4], q[4];
      double w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        in[e] = x[e] > tv && x[e] >= W.cut;
        w[e] = W(fmaxf(x[e], W.cut), bin[e], q[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (in[e] && bin[e] < kBins - 1) {
          const uint32_t positive = (uint32_t)(q[e] + (1 << 28));
          atomicAdd(&s.hist[0][bin[e]], 1u);
          atomicAdd(&s.hist[1][bin[e]], positive & 0x3fffu);
          atomicAdd(&s.hist[2][bin[e]], positive >> 14);
        }
      z += ((in[0] ? w[0] : 0.0) + (in[1] ? w[1] : 0.0)) + ((in[2] ? w[2] : 0.0) + (in[3] ? w[3] : 0.0));
    });
    const double strictly = cluster_total(z, &Slot::mass);
    const double wt = t ? W(tv) : 0.0;
    const double target = p > 0.0f ? (double)p * (strictly + (double)ties * wt) : 0.0;
    if (target < strictly) {
      merge_hist(masses);
      double front;
      const int bin = find_bin(0.0, [&](u64 x, int i) {
        const double of = s.table[-i & (kPer - 1)];
        const double unit = __hiloint2double(__double2hiint(of) - (((i + kPer - 1) >> kPerLog) << 20), __double2loint(of));
        return i < kBins - 1 ? (double)x * (unit * 0x1p-34) : 1e30;
      }, target, s.scan_d, front);
      // the least numbers of this bin and of the one above it: the pass below only compares
      const float cut = bin == kBins - 1 ? W.cut : least_of(bin), end = bin ? least_of(bin - 1) : INFINITY;
      const bool fill = packed < 0;
      tried = true;
      Found f{0u, 0xffffffffu, 0u};
      filling = 0;
      if (tid == 0) s.list_n = 0;
      __syncthreads();
      each(blk0, blk1, [&](int blk, const float (&x)[4]) {
        bool in[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) in[e] = x[e] > tv && x[e] >= cut;
        if (!__any_sync(0xffffffffu, in[0] || in[1] || in[2] || in[3])) return;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (in[e] && x[e] < end) note(f, key_of(x[e]), index_of(blk, e));
        if (fill && filling <= kPack) pack(blk, x, in);
      });
      if (fill) use_pack();
      gather(f);
      finish(std::true_type{}, f, front, target);
    } else if (wt > 0.0) {   // the border lies among the ties of top-k
      ties = (uint32_t)min((u64)ties, (u64)((target - strictly) / wt) + 1);
    }
  }
  const bool some = t != 0u && ties < equal;   // only the first of the elements that equal the threshold stay
  const float tv = t ? value_of(t) : -INFINITY;
  uint32_t seen0 = 0;                          // ties in front of this warp's part
  if (some) {
    uint32_t eq = 0;
    each(blk0, blk1, [&](int blk, const float (&x)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) eq += x[e] == tv;
    });
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) s.warp_eq[warp] = eq;
    __syncthreads();
    if (warp == 0) {
      eq = __reduce_add_sync(0xffffffffu, s.warp_eq[lane]);
      if (lane == 0) s.slot.eq = eq;
    }
    meet();
    eq = peek(&s.slot.eq, lane % C);
    seen0 = __reduce_add_sync(0xffffffffu, (lane < rank ? eq : 0u) + (lane < warp ? s.warp_eq[lane] : 0u));
  }
  // ---- kept weights in index order
  // what cannot be kept is passed over by one comparison: below the threshold, or 1 % below the least weight
  float cut = fmaxf(W.cut, tv);
  if (mp > 0.0f) cut = fmaxf(cut, (float)(W.max + ((double)__log2f(mp) - 0.01) * octave));   // (the 32-bit logarithm is good to 2^-20)
  // a few kept elements of a long part are listed first: a weight costs thirty times the comparison
  if (packed < 0 && ((t && !tried) || mp > 0.0f)) {
    filling = 0;
    each(blk0, blk1, [&](int blk, const float (&x)[4]) {
      const bool in[4] = {x[0] >= cut, x[1] >= cut, x[2] >= cut, x[3] >= cut};
      if (filling <= kPack && __any_sync(0xffffffffu, in[0] || in[1] || in[2] || in[3])) pack(blk, x, in);
    });
    use_pack();
  }
  const double mp_near = mp > 0.0f ? (double)mp * 1.0000001 : 0.0;
  auto kept4 = [&](const float (&x)[4], uint32_t& seen, double (&w)[4]) -> bool {   // whether any lane has a weight
    uint32_t place = 0;
    if (some) {
      uint32_t mine = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) mine += x[e] == tv;
      uint32_t inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      place = seen + inc - mine;
      seen += __shfl_sync(0xffffffffu, inc, 31);
    }
    bool keep[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      keep[e] = x[e] >= cut;
      if (some && x[e] == tv) keep[e] = keep[e] && place++ < ties;
      w[e] = 0.0;
    }
    if (!__any_sync(0xffffffffu, keep[0] || keep[1] || keep[2] || keep[3])) return false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      int bin;
      const double x0 = W(fmaxf(x[e], cut), bin);
      w[e] = keep[e] ? x0 : 0.0;
    }
    if (mp > 0.0f) {
      bool near = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) near = near || (w[e] != 0.0 && w[e] < mp_near);
      if (near) {   // next to the border of min-p, or below it: with the library's exponential
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
          const double we = e == 0 ? w[0] : e == 1 ? w[1] : e == 2 ? w[2] : w[3];
          const float xe = e == 0 ? x[0] : e == 1 ? x[1] : e == 2 ? x[2] : x[3];
          const bool drop = we < mp_near && library_exp(((double)xe - W.max) / (double)temp) < (double)mp;
          if (drop && e == 0) w[0] = 0.0;
          if (drop && e == 1) w[1] = 0.0;
          if (drop && e == 2) w[2] = 0.0;
          if (drop && e == 3) w[3] = 0.0;
        }
      }
    }
    return true;
  };
  // Lane i keeps the sum of the i-th group of blocks of its warp, and the ties in front of it: the walk at the end then
  // goes through one group.
  const int group = packed >= 0 ? 1 : (per + 7) / 8;
  double my_group = 0.0;
  uint32_t seen = seen0, my_seen = seen0;
  double in_group = 0.0;
  bool any = false;
  int g = 0, to_go = group;
  each(blk0, blk1, [&](int, const float (&x)[4]) {
    if (to_go == group && lane == g) my_seen = seen;
    double w[4];
    if (kept4(x, seen, w)) {
      in_group += (w[0] + w[1]) + (w[2] + w[3]);
      any = true;
    }
    if (--to_go == 0) {
      if (any) {
        in_group = warp_add(in_group);
        if (lane == g) my_group = in_group;
      }
      in_group = 0.0;
      any = false;
      to_go = group;
      ++g;
    }
  });
  in_group = warp_add(in_group);
  if (lane == g) my_group = in_group;   // (a last group that is short)
  const double upto_group = warp_scan(my_group, lane);
  if (lane == 31) s.warp_sum[warp] = upto_group;
  __syncthreads();
  const double upto_warp = warp_scan(s.warp_sum[lane], lane);
  if (tid == 31) s.slot.sum = upto_warp;
  meet();
  // The place u z of the running sum belongs to the last CTA, in it the last warp, in it the last group, and there the last
  // token with a weight whose front is not past it.  (Roundings between the levels move a border by 2^-52 of the sum.)
  const double mine = lane < C ? peek(&s.slot.sum, lane % C) : 0.0;
  if (C > 1) fsvd_tile::cluster_arrive();   // nothing of another CTA is read any more
  const double upto_cta = warp_scan(mine, lane), z = __shfl_sync(0xffffffffu, upto_cta, 31);
  const float u = a.u[b];
  const double target = (u >= 0.0f ? fmin((double)u, 1.0 - 0x1p-24) : 0.0) * z;
  auto last_not_past = [&](double x, double end, double from) -> int {   // lane of it; x: its part, end: the sum up to it
    const unsigned ok = __ballot_sync(0xffffffffu, x > 0.0 && from + (end - x) <= target);
    const unsigned any = __ballot_sync(0xffffffffu, x > 0.0);
    return ok ? 31 - __clz(ok) : any ? __ffs(any) - 1 : -1;
  };
  const int owner = last_not_past(mine, upto_cta, 0.0);
  if (owner == rank) {
    double from = __shfl_sync(0xffffffffu, upto_cta - mine, owner);
    const double wx = s.warp_sum[lane];
    const int ow = last_not_past(wx, upto_warp, from);
    if (ow == warp) {
      from += __shfl_sync(0xffffffffu, upto_warp - wx, ow);
      const int og = last_not_past(my_group, upto_group, from);
      from += __shfl_sync(0xffffffffu, upto_group - my_group, og);
      seen = __shfl_sync(0xffffffffu, my_seen, og);
      int best = 0;
      double best_w = 0.0;
      const int first = blk0 + og * group;
      each(first, min(blk1, first + group), [&](int blk, const float (&x4)[4]) {
        if (packed >= 0 && blk != og) return;   // (a short list has a group per block)
        double w[4];
        kept4(x4, seen, w);
        const double x = (w[0] + w[1]) + (w[2] + w[3]), end = warp_scan(x, lane);
        const int src = last_not_past(x, end, from);
        const bool here = src >= 0 && (best_w == 0.0 || __shfl_sync(0xffffffffu, from + (end - x), src) <= target);
        if (here) {
          double run = from + (end - x), pw = 0.0;
          int pick = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (w[e] > 0.0 && (pw == 0.0 || run <= target)) {
              pick = index_of(blk, e);
              pw = w[e];
            }
            run += w[e];
          }
          best = __shfl_sync(0xffffffffu, pick, src);
          best_w = __shfl_sync(0xffffffffu, pw, src);
        }
        from += __shfl_sync(0xffffffffu, end, 31);
      });
      if (lane == 0) {
        a.tokens[b] = best;
        if (a.probs) a.probs[b] = (float)(best_w / z);
      }
    }
  }
  if (C > 1) fsvd_tile::cluster_wait();   // the others have read this CTA's slot
}

static int fail(int code, const char* msg) {
  if (code == FSVD_ERR_CUDA) cudaGetLastError();   // (off the thread: no later check of the caller's reports it again)
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
  if (V > kMaxVocab) return fail(FSVD_ERR_UNSUPPORTED, "a vocabulary beyond 2^20 is unsupported");
  if (B > (1 << 24)) return fail(FSVD_ERR_UNSUPPORTED, "more than 2^24 rows are unsupported");
  if (temperature_all != temperature_all || top_p_all != top_p_all || min_p_all != min_p_all)
    return fail(FSVD_ERR_ARG, "NaN setting");
  if (B == 0) return 0;
  int dev = 0, sms = 148, optin = 227 * 1024;
  if (cudaGetDevice(&dev) == cudaSuccess) {
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    cudaDeviceGetAttribute(&optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
  }
  // CTAs of a row, by waves x time of a CTA: 20 us for its steps one after the other, and 0.28 us per 1000 elements where they
  // fit its shared memory, 0.36 where every pass reads them again from L2.  (128 rows of 100003: one CTA each 52 us with top-k,
  // top-p and min-p and 77 with top-p alone; four each, which hold them, 116 and 186.)
  const int es = dtype == FSVD_DTYPE_F32 ? 4 : 2;
  const long long places = V + 16 / es - 1;   // a row may start up to 15 bytes behind a 16-byte boundary
  const auto chunk_of = [&](int c) { return ((places + c - 1) / c + kBlock - 1) / kBlock * kBlock; };
  const auto lists = [](bool resident) { return kWarps * (resident ? kPackPiece : kPackAlone) * 6; };
  const long long room = optin - (long long)sizeof(Shared) - lists(true);   // 141 KB
  static_assert(sizeof(Shared) + kWarps * kPackAlone * 6 <= 227 * 1024);
  const auto fits = [&](int c) { return chunk_of(c) * es <= room; };
  const auto cost = [&](int c) { return (double)(((long long)B * c + sms - 1) / sms) * (20.0 + chunk_of(c) * (fits(c) ? 0.28e-3 : 0.36e-3)); };
  int C = 1;
  while (chunk_of(C) > kMaxPiece) C *= 2;   // (at most kMaxCluster)
  for (int c = 2 * C; c <= kMaxCluster; c *= 2)
    if (places / c > 2048 && cost(c) < cost(C)) C = c;
  Args a;
  a.logits = logits; a.stride = row_stride; a.u = uniforms; a.temperature = temperature; a.top_k = top_k; a.top_p = top_p;
  a.min_p = min_p; a.T_all = temperature_all; a.k_all = top_k_all; a.p_all = top_p_all; a.m_all = min_p_all;
  a.tokens = tokens; a.probs = probs; a.V = V;
  a.chunk = (int)chunk_of(C);
  const bool resident = fits(C);
  const size_t smem = (size_t)lists(resident) + (resident ? (size_t)a.chunk * es : 0);
  typedef void (*Kernel)(Args);
  static const Kernel kernels[4] = {sample_kernel<float, false>, sample_kernel<float, true>, sample_kernel<__nv_bfloat16, false>,
                                    sample_kernel<__nv_bfloat16, true>};
  static fsvd_tile::SmemLimit limits[4];
  const int which = (dtype == FSVD_DTYPE_F32 ? 0 : 2) + resident;
  cudaError_t e = limits[which].raise(kernels[which]);
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
    e = cudaLaunchKernelExC(&cfg, (const void*)kernels[which], params);
  }
  if (e != cudaSuccess) {
    char msg[160];
    snprintf(msg, sizeof(msg), "kernel launch failed: %s", cudaGetErrorString(e));
    return fail(FSVD_ERR_CUDA, msg);
  }
  fsvd_tile_count_launch();
  return 0;
}

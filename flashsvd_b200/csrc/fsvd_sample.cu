// Choice of the next token (fsvd_sample of include/flashsvd_b200.h): temperature, top-k, top-p, min-p, one uniform number.
//
// The vocabulary is ordered by logit (descending, lower index first); every filter keeps a prefix of that order, so the
// kept set is {key > t} and the first r of {key = t} in index order, for one threshold key t.  It is found without a
// sort: a radix descent over the bits of an order-preserving integer key, by counts for top-k and by mass for top-p.
// Weights are integers, exp((l - max) / T) * 2^frac with the exponential in 64 bits: their sums do not depend on the
// order of addition, and a running sum sits on the right side of a border unless the border is 2^-40 away.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>

#include "../../include/flashsvd_b200.h"
#include "fsvd_tile.h"

namespace fsvd_sample_impl {

typedef unsigned long long u64;
constexpr int kThreads = 1024, kWarps = kThreads / 32;

struct Args {
  const void* logits;
  long long stride;
  const float *u, *temperature, *top_p, *min_p;
  const int* top_k;
  float T_all, p_all, m_all;
  int k_all;
  int* tokens;
  float* probs;
  int V, frac;
};

// Ascending keys for ascending numbers; NaN and -infinity share the lowest, the zeros share theirs.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
__device__ __forceinline__ float logit(const float* row, int i) { return row[i]; }
__device__ __forceinline__ float logit(const __nv_bfloat16* row, int i) { return __bfloat162float(row[i]); }

struct Row {
  float max, T;
  int frac;
  double scale;
  __device__ double weight(uint32_t key) const {
    if (key == 0u) return 0.0;
    const float x = value_of(key);
    return x == max ? 1.0 : exp(((double)x - (double)max) / (double)T);
  }
  __device__ u64 fixed(double w) const { return (u64)__double2ll_rn(w * scale); }
};

template <typename F>
__device__ __forceinline__ u64 block_sum(u64 x, u64* sh, F) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = x;
  __syncthreads();
  u64 s = 0;
  for (int w = 0; w < kWarps; ++w) s += sh[w];
  return s;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Args a) {
  __shared__ u64 hist[256];
  __shared__ u64 sh[kWarps];
  __shared__ uint32_t pick_bin;
  __shared__ u64 pick_above;
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x, V = a.V;
  const T* row = reinterpret_cast<const T*>(a.logits) + (size_t)b * a.stride;
  const float temp = fminf(a.temperature ? a.temperature[b] : a.T_all, 3.402823466e38f);
  int k = a.top_k ? a.top_k[b] : a.k_all;
  const float p = a.top_p ? a.top_p[b] : a.p_all, mp = a.min_p ? a.min_p[b] : a.m_all;
  if (k <= 0 || k > V) k = V;
  // largest key, its lowest index
  u64 best = 0;
  for (int i = tid; i < V; i += kThreads) best = max(best, ((u64)key_of(logit(row, i)) << 32) | (uint32_t)~i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) sh[warp] = best;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) best = max(best, sh[w]);
  const uint32_t kmax = (uint32_t)(best >> 32);
  const bool none = kmax == 0u;
  if (none || !(temp > 0.0f) || k == 1) {
    if (tid == 0) {
      a.tokens[b] = none ? 0 : (int)~(uint32_t)best;
      if (a.probs) a.probs[b] = none ? 0.0f : 1.0f;
    }
    return;
  }
  Row R{value_of(kmax), temp, a.frac, ldexp(1.0, a.frac)};
  // The key at which the running `weigh` over descending keys first exceeds `target`, and the sum above that key.
  auto descend = [&](auto weigh, u64 target, uint32_t& key, u64& above) {
    key = 0u;
    above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kThreads) {
        const uint32_t x = key_of(logit(row, i));
        if (shift == 24 || (x >> (shift + 8)) == (key >> (shift + 8))) atomicAdd(&hist[(x >> shift) & 255u], weigh(x));
      }
      __syncthreads();
      if (tid == 0) {
        u64 s = above;
        int bin = 255;
        for (; bin > 0 && s + hist[bin] <= target; --bin) s += hist[bin];
        pick_bin = bin;
        pick_above = s;
      }
      __syncthreads();
      key |= pick_bin << shift;
      above = pick_above;
    }
    __syncthreads();
  };
  uint32_t t = 0u;       // threshold key
  u64 ties = ~0ull;      // kept of those that equal it
  if (k < V) {
    u64 above;
    descend([](uint32_t) -> u64 { return 1; }, (u64)k - 1, t, above);
    ties = (u64)k - above;
  }
  if (p < 1.0f) {
    const uint32_t tk = t;
    const u64 wt = R.fixed(R.weight(tk));
    u64 z = 0;
    for (int i = tid; i < V; i += kThreads) {
      const uint32_t x = key_of(logit(row, i));
      if (x > tk) z += R.fixed(R.weight(x));
    }
    z = block_sum(z, sh, 0);
    if (k < V) z += ties * wt;
    else if (tk == 0u) z += 0;
    const u64 target = p > 0.0f ? __umul64hi((u64)((double)p * 18446744073709551616.0), z) : 0;
    uint32_t tp;
    u64 above;
    // (mass at the top-k key is cut to the ties that are kept; it lies last, and what it adds is known)
    descend([&](uint32_t x) -> u64 { return x > tk ? R.fixed(R.weight(x)) : 0; }, target, tp, above);
    const u64 w = R.fixed(R.weight(tp));
    if (tp > tk && w) {
      t = tp;
      ties = (target - above) / w + 1;
    } else if (wt) {   // the border lies among the ties of top-k
      u64 all = 0;
      for (int i = tid; i < V; i += kThreads) {
        const uint32_t x = key_of(logit(row, i));
        if (x > tk) all += R.fixed(R.weight(x));
      }
      all = block_sum(all, sh, 0);
      ties = min(ties, (target - all) / wt + 1);
    }
  }
  // kept mass by warp segment, in index order; ties counted in the same order
  const int seg = (V + kWarps - 1) / kWarps, i0 = warp * seg, i1 = min(V, i0 + seg);
  u64 eq = 0;
  for (int i = i0 + lane; i < i1; i += 32) eq += key_of(logit(row, i)) == t;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) eq += __shfl_xor_sync(0xffffffffu, eq, o);
  __syncthreads();
  if (lane == 0) sh[warp] = eq;
  __syncthreads();
  u64 before = 0;   // ties in front of this warp's segment
  for (int w = 0; w < warp; ++w) before += sh[w];
  __syncthreads();
  auto kept = [&](int i, u64& seen) -> u64 {   // weight of element i if it is kept; seen: ties before the warp's row of 32
    const uint32_t x = i < i1 ? key_of(logit(row, i)) : 0u;
    const bool tie = i < i1 && x == t;
    const unsigned mask = __ballot_sync(0xffffffffu, tie);
    const u64 rank = seen + __popc(mask & ((1u << lane) - 1u));
    seen += __popc(mask);
    if (i >= i1 || !(x > t || (tie && rank < ties))) return 0;
    const double w = R.weight(x);
    return w >= (double)fminf(mp, 1.0f) || !(mp > 0.0f) ? R.fixed(w) : 0;
  };
  u64 sum = 0, seen = before;
  for (int i = i0; i < i1; i += 32) sum += kept(i + lane, seen);
  const u64 mine = sum;
  const u64 z = block_sum(sum, sh, 0);
  u64 wsum = mine;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wsum += __shfl_xor_sync(0xffffffffu, wsum, o);
  u64 ahead = 0;
  for (int w = 0; w < warp; ++w) ahead += sh[w];
  const float u = a.u[b];
  const double uu = u >= 0.0f ? fmin((double)u, 1.0 - 0x1p-24) : 0.0;
  const u64 target = __umul64hi((u64)(uu * 18446744073709551616.0), z);
  if (tid == 0) found = 0;
  __syncthreads();
  if (ahead <= target && target < ahead + wsum) {   // the warp that holds the token
    seen = before;
    for (int i = i0; i < i1; i += 32) {
      const u64 w = kept(i + lane, seen);
      u64 inc = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, ahead + inc > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          a.tokens[b] = i + lane;
          if (a.probs) a.probs[b] = (float)((double)w / (double)z);
        }
        break;
      }
      ahead += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
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
  if (V > (1 << 22)) return fail(FSVD_ERR_UNSUPPORTED, "a vocabulary beyond 2^22 is unsupported");
  if (temperature_all != temperature_all || top_p_all != top_p_all || min_p_all != min_p_all)
    return fail(FSVD_ERR_ARG, "NaN setting");
  if (B == 0) return 0;
  int bits = 0;
  while ((1 << bits) < V) ++bits;
  Args a;
  a.logits = logits; a.stride = row_stride; a.u = uniforms; a.temperature = temperature; a.top_k = top_k; a.top_p = top_p;
  a.min_p = min_p; a.T_all = temperature_all; a.k_all = top_k_all; a.p_all = top_p_all; a.m_all = min_p_all;
  a.tokens = tokens; a.probs = probs; a.V = V; a.frac = std::min(46, 62 - bits);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(B);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = (cudaStream_t)stream;
  const cudaError_t e = dtype == FSVD_DTYPE_F32 ? cudaLaunchKernelEx(&cfg, sample_kernel<float>, a)
                                                : cudaLaunchKernelEx(&cfg, sample_kernel<__nv_bfloat16>, a);
  if (e != cudaSuccess) {
    char msg[160];
    snprintf(msg, sizeof(msg), "kernel launch failed: %s", cudaGetErrorString(e));
    return fail(FSVD_ERR_CUDA, msg);
  }
  fsvd_tile_count_launch();
  return 0;
}

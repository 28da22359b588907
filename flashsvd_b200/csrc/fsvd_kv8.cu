// Rotary positions and the 8-bit key / value cache: rotation, append, read-back and single-query attention
// (fsvd_rope_qk, fsvd_kv8_append, fsvd_kv8_load, fsvd_flash_decode_kv8 of include/flashsvd_b200.h).
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <atomic>

#include "../../include/flashsvd_b200.h"
#include "fsvd_kv8_attn.cuh"
#include "fsvd_rope.cuh"
#include "fsvd_stage.h"
#include "fsvd_tile.h"

namespace fsvd_kv8_impl {

using fsvd::DS_CACHE_FULL;
using fsvd::DS_OK;
using fsvd::SyncState;
using fsvd_rope::Rotary;

static int fail(int code, const char* fmt, ...) {
  char msg[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  fsvd_tile_set_error(code, msg);
  return code;
}
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static int sm_count() {
  static std::atomic<int> cache[16];
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) != cudaSuccess) return n;
  if (dev >= 0 && dev < 16 && (n = cache[dev].load()) > 0) return n;
  n = 148;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (dev >= 0 && dev < 16) cache[dev].store(n);
  return n;
}

// Every kernel of this file may start while the one before it in the stream is still draining, and waits for it
// (griddepcontrol) before it touches memory.
__device__ __forceinline__ void pdl_begin() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... Params, typename... Args>
static int launch(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, void* stream, const Args&... args) {
  // Above the 48 KB that a kernel has by itself the limit is raised at every such launch: a setting of the current
  // device, so nothing is remembered.
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return fail(FSVD_ERR_CUDA, "shared memory of %zu bytes: %s", smem, cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return fail(FSVD_ERR_CUDA, "kernel launch failed: %s", cudaGetErrorString(e));
  fsvd_tile_count_launch();
  return 0;
}

constexpr int kThreads = 256;

// ------------------------------------------------------------------------------------------ rotary positions
struct RopeArgs {
  const void *q, *k;
  void *q_out, *k_out;
  long long q_stride, k_stride;
  const int* positions;
  Rotary rot;
  int T, H, Hk, Dh, tokens, heads;   // tokens and heads of a CTA
};

// A CTA turns `tokens` rows of heads; its threads go through the (token, head, unit) list in steps of kThreads, several units
// at a time so that their loads are under way together.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, 4) rope_kernel(const RopeArgs a) {
  constexpr int N = 2;                              // units at a time
  extern __shared__ __align__(16) float2 table[];   // [tokens][R / 2] cosine, sine
  const int half = a.rot.R >> 1, tid = threadIdx.x, R = a.rot.R, inter = a.rot.interleaved;
  const int t0 = blockIdx.x * a.tokens, nt = min(a.tokens, a.T - t0);
  pdl_begin();
  for (int i = tid; i < nt * half; i += kThreads) {
    double c, s;
    const int t = i / half;
    fsvd_rope::angle(a.positions[t0 + t], a.rot.inv_freq[i - t * half], a.rot.scale, c, s);
    table[i] = make_float2((float)c, (float)s);
  }
  __syncthreads();
  const unsigned U = a.Dh / 16;
  const int h0 = blockIdx.y * a.heads, nh = min(a.heads, a.H + a.Hk - h0);
  const unsigned items = (unsigned)nt * nh * U;
  for (unsigned i0 = tid; i0 < items; i0 += N * kThreads) {
    float x[N][8], y[N][8];
    T* dst[N];
    int token[N], unit[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const unsigned i = i0 + k * kThreads;
      if (i < items) {
        const unsigned row = i / U, t = row / (unsigned)nh;
        const int h = h0 + (int)(row - t * nh);
        const size_t tt = t0 + t;
        token[k] = (int)t;
        unit[k] = (int)(i - row * U);
        const bool q = h < a.H;
        const T* src = q ? reinterpret_cast<const T*>(a.q) + tt * a.q_stride + (size_t)h * a.Dh
                         : reinterpret_cast<const T*>(a.k) + tt * a.k_stride + (size_t)(h - a.H) * a.Dh;
        dst[k] = q ? reinterpret_cast<T*>(a.q_out) + (tt * a.H + h) * a.Dh : reinterpret_cast<T*>(a.k_out) + (tt * a.Hk + h - a.H) * a.Dh;
        fsvd_rope::load_unit<WIDE>(src, unit[k], R, inter, x[k], y[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (i0 + k * kThreads < items) {
        auto turn = [&](int e, float c, float s) {
          const float xe = x[k][e], ye = y[k][e];
          x[k][e] = xe * c - ye * s;
          y[k][e] = ye * c + xe * s;
        };
        const float2* cs = table + token[k] * half + 8 * unit[k];
        // (pairs that are not rotated are copied: an infinity times a sine of zero is no number)
        if constexpr (WIDE) {
          if (8 * unit[k] < half) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float4 two = *reinterpret_cast<const float4*>(cs + e);
              turn(e, two.x, two.y);
              turn(e + 1, two.z, two.w);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (8 * unit[k] + e < half) turn(e, cs[e].x, cs[e].y);
        }
        fsvd_rope::store_unit<WIDE>(dst[k], unit[k], R, inter, x[k], y[k]);
      }
  }
}

// ------------------------------------------------------------------------------------------ append
struct AppendArgs {
  fsvd_kv8 c;
  const __nv_bfloat16 *k, *v, *q;
  __nv_bfloat16* q_out;
  long long kv_batch, kv_token, q_batch, q_token;
  const int *seqlens, *new_lens;
  int* status;
  Rotary rot;       // R = 0: no rotation
  int H, L, groups; // groups: head groups of a (sequence, block)
  int nblk;         // blocks that L tokens can touch
};

// Exponent of the scale for a largest magnitude: the smallest e >= -60 with amax <= 448 2^e (448 = 1.75 * 2^8).
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, -60);
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Two numbers as e4m3 codes; what is not finite becomes NaN.
__device__ __forceinline__ uint32_t code2(float x, float y) {
  uint32_t r = __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
  if (!isfinite(x)) r = (r & 0xff00u) | 0x7fu;
  if (!isfinite(y)) r = (r & 0x00ffu) | 0x7f00u;
  return r;
}
__device__ __forceinline__ float2 decode2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// x c - y s for bf16 x, y and (c, s) given as sums of two fp32 numbers each: the error of the result is that of its
// last rounding, so that a rotated key falls on the same side of a rounding border as in 64 bits.  (Products of a bf16
// and an fp32 number do not fit 24 bits: their rounding errors are carried along.)
__device__ __forceinline__ float turn(float x, float y, float ch, float cl, float sh, float sl) {
  const float p = x * ch, pe = fmaf(x, ch, -p);
  const float q = y * sh, qe = fmaf(y, sh, -q);
  const float d = p - q, z = d - p, de = (p - (d - z)) - (q + z);
  return d + (de + (pe - qe) + (x * cl - y * sl));
}

template <int DH, int BLOCK>
__device__ __forceinline__ int unit_offset(int u, int R, int interleaved, int which) {
  const bool split = !interleaved && 16 * u < R;
  return split ? 8 * u + (which ? (R >> 1) : 0) : 16 * u + 8 * which;
}

// One CTA per (sequence, block of the cache, group of kv heads): a tile of at most BLOCK tokens x DH of a head sits in
// registers (bf16) between the maximum and the rounding, so that each input is read once and each code written once.
template <int DH, int BLOCK, bool WIDE>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs a) {
  constexpr int U = DH / 16, ROWS = kThreads / U, NIT = (BLOCK + ROWS - 1) / ROWS;
  extern __shared__ float4 tab[];   // [tokens][R / 2] cosine and sine as (c_hi, c_lo, s_hi, s_lo)
  __shared__ float red[2][2][kThreads / 32];
  const int tid = threadIdx.x, u = tid % U, r0 = tid / U;
  int idx = blockIdx.x;
  const int grp = idx % a.groups;
  idx /= a.groups;
  const int j = idx % a.nblk, b = idx / a.nblk;
  pdl_begin();
  const int start = max(a.seqlens[b], 0);
  const int count = a.new_lens ? min(max(a.new_lens[b], 0), a.L) : a.L;
  const long long end_ll = (long long)start + count;
  const int end = (int)min(end_ll, (long long)a.c.S_max);
  if (end_ll > a.c.S_max && j == 0 && grp == 0 && tid == 0) atomicCAS(a.status, (int)DS_OK, (int)DS_CACHE_FULL);
  const int blk = start / BLOCK + j;
  const long long blk0 = (long long)blk * BLOCK;
  if (blk0 >= end_ll) return;
  const int lo = (int)max((long long)start, blk0), hi = (int)min((long long)end, blk0 + BLOCK);
  // (queries of tokens beyond the cache are rotated too: their range is not cut at the capacity)
  const int nq = (int)(min(end_ll, blk0 + BLOCK) - lo), n = max(0, hi - lo);
  const int R = a.rot.R, half = R >> 1, inter = a.rot.interleaved;
  if (R) {
    // Cosines and sines of the tile's tokens.  More than a few: of every eighth token and of steps 0..7, and the products of
    // those (64 tokens: 16 evaluations in 64 bits a pair instead of 64).
    auto put = [&](int i, double c, double s) {
      const float ch = (float)c, sh = (float)s;
      tab[i] = make_float4(ch, (float)(c - (double)ch), sh, (float)(s - (double)sh));
    };
    const int coarse = (nq + 7) / 8;
    if (nq <= 8) {
      for (int i = tid; i < nq * half; i += kThreads) {
        const int t = i / half;
        double c, s;
        fsvd_rope::angle(lo + t, a.rot.inv_freq[i - t * half], a.rot.scale, c, s);
        put(i, c, s);
      }
    } else {
      double2* steps = reinterpret_cast<double2*>(tab + min(BLOCK, a.L) * half);   // [8 + coarse][half]
      for (int i = tid; i < (8 + coarse) * half; i += kThreads) {
        const int k = i / half;
        double c, s;
        fsvd_rope::angle(k < 8 ? k : lo + 8 * (k - 8), a.rot.inv_freq[i - k * half], k < 8 ? 1.0f : a.rot.scale, c, s);
        steps[i] = make_double2(c, s);
      }
      __syncthreads();
      for (int i = tid; i < nq * half; i += kThreads) {
        const int t = i / half, p = i - t * half;
        const double2 x = steps[(8 + (t >> 3)) * half + p], y = steps[(t & 7) * half + p];
        put(i, x.x * y.x - x.y * y.y, x.y * y.x + x.x * y.y);
      }
    }
    __syncthreads();
  }
  const int Hk = a.c.Hk, nb = (a.c.S_max + BLOCK - 1) / BLOCK;
  const int hk0 = (int)((long long)Hk * grp / a.groups), hk1 = (int)((long long)Hk * (grp + 1) / a.groups);
  const bool held = start > blk0;   // the block holds tokens already
  int parity = 0;
  for (int hk = hk0; hk < hk1 && n > 0; ++hk, parity ^= 1) {
    uint32_t kreg[NIT][8], vreg[NIT][8];   // packed pairs (a, b)
    float kmax = 0.0f, vmax = 0.0f;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int t = r0 + it * ROWS;
      if (t < n) {
        const size_t off = (size_t)b * a.kv_batch + (size_t)(lo - start + t) * a.kv_token + (size_t)hk * DH;
        float x[8], y[8];
        fsvd_rope::load_unit<WIDE>(a.v + off, u, R, inter, x, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          vreg[it][i] = fsvd_rope::pack2(x[i], y[i]);
          if (isfinite(x[i])) vmax = fmaxf(vmax, fabsf(x[i]));
          if (isfinite(y[i])) vmax = fmaxf(vmax, fabsf(y[i]));
        }
        fsvd_rope::load_unit<WIDE>(a.k + off, u, R, inter, x, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int p = 8 * u + i;
          if (p < half) {
            const float4 cs = tab[t * half + p];
            const float x0 = x[i], y0 = y[i];
            x[i] = turn(x0, y0, cs.x, cs.y, cs.z, cs.w);
            y[i] = turn(y0, -x0, cs.x, cs.y, cs.z, cs.w);
          }
          kreg[it][i] = fsvd_rope::pack2(x[i], y[i]);
          x[i] = __uint_as_float(kreg[it][i] << 16);
          y[i] = __uint_as_float(kreg[it][i] & 0xffff0000u);
          if (isfinite(x[i])) kmax = fmaxf(kmax, fabsf(x[i]));
          if (isfinite(y[i])) kmax = fmaxf(kmax, fabsf(y[i]));
        }
      }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) {
      kmax = fmaxf(kmax, __shfl_xor_sync(0xffffffffu, kmax, x));
      vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, x));
    }
    if ((tid & 31) == 0) {
      red[parity][0][tid >> 5] = kmax;
      red[parity][1][tid >> 5] = vmax;
    }
    const size_t si = ((size_t)b * Hk + hk) * nb + blk;
    const float kold = held ? a.c.k_scale[si] : 0.0f, vold = held ? a.c.v_scale[si] : 0.0f;
    __syncthreads();   // (two halves of `red` in turn: the next head writes the other one)
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      kmax = fmaxf(kmax, red[parity][0][w]);
      vmax = fmaxf(vmax, red[parity][1][w]);
    }
    const int ke = scale_exponent(kmax), ve = scale_exponent(vmax);
    const float ks = fmaxf(kold, two_to(ke)), vs = fmaxf(vold, two_to(ve));
    const size_t base = (((size_t)b * Hk + hk) * a.c.S_max + (size_t)blk0) * DH;
    uint8_t* kc = reinterpret_cast<uint8_t*>(a.c.k8) + base;
    uint8_t* vc = reinterpret_cast<uint8_t*>(a.c.v8) + base;
    if (held) {   // a larger scale: round what the block holds once more
      const int old_bytes = (int)(start - blk0) * DH;
      for (int which = 0; which < 2; ++which) {
        const float was = which ? vold : kold, now = which ? vs : ks;
        if (!(now > was)) continue;
        uint32_t* w = reinterpret_cast<uint32_t*>(which ? vc : kc);
        const float f = was / now;
        for (int i = tid; i < old_bytes / 4; i += kThreads) {
          const uint32_t x = w[i];
          const float2 p = decode2(x & 0xffffu), q = decode2(x >> 16);
          w[i] = code2(p.x * f, p.y * f) | (code2(q.x * f, q.y * f) << 16);
        }
      }
    }
    const float ki = 1.0f / ks, vi = 1.0f / vs;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int t = r0 + it * ROWS;
      if (t < n) {
        const size_t row = (size_t)(lo - blk0 + t) * DH;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
          uint8_t* dst = (which ? vc : kc) + row;
          const float inv = which ? vi : ki;
          uint32_t cd[8];   // codes of the pairs: low byte a, high byte b
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t w = which ? vreg[it][i] : kreg[it][i];
            float x = __uint_as_float(w << 16) * inv, y = __uint_as_float(w & 0xffff0000u) * inv;
            if (inv <= 0x1p-120f) {   // 256 * 2^120 is no 32-bit number any more
              x = fabsf(x) > 240.0f && isfinite(x) ? copysignf(240.0f, x) : x;
              y = fabsf(y) > 240.0f && isfinite(y) ? copysignf(240.0f, y) : y;
            }
            cd[i] = code2(x, y);
          }
          if constexpr (WIDE) {
            const bool split = !inter && 16 * u < R;
            uint2 first, second;
            const uint32_t a03 = __byte_perm(__byte_perm(cd[0], cd[1], 0x0040), __byte_perm(cd[2], cd[3], 0x0040), 0x5410);
            const uint32_t a47 = __byte_perm(__byte_perm(cd[4], cd[5], 0x0040), __byte_perm(cd[6], cd[7], 0x0040), 0x5410);
            const uint32_t b03 = __byte_perm(__byte_perm(cd[0], cd[1], 0x0051), __byte_perm(cd[2], cd[3], 0x0051), 0x5410);
            const uint32_t b47 = __byte_perm(__byte_perm(cd[4], cd[5], 0x0051), __byte_perm(cd[6], cd[7], 0x0051), 0x5410);
            first = split ? make_uint2(a03, a47) : make_uint2(cd[0] | (cd[1] << 16), cd[2] | (cd[3] << 16));
            second = split ? make_uint2(b03, b47) : make_uint2(cd[4] | (cd[5] << 16), cd[6] | (cd[7] << 16));
            *reinterpret_cast<uint2*>(dst + (split ? 8 * u : 16 * u)) = first;
            *reinterpret_cast<uint2*>(dst + (split ? 8 * u + half : 16 * u + 8)) = second;
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int2 at = fsvd_rope::pair_at(8 * u + i, R, inter);
              dst[at.x] = (uint8_t)(cd[i] & 0xffu);
              dst[at.y] = (uint8_t)(cd[i] >> 8);
            }
          }
        }
      }
    }
    if (tid == 0) {
      a.c.k_scale[si] = ks;
      a.c.v_scale[si] = vs;
    }
  }
  if (!a.q) return;
  const int h0 = (int)((long long)a.H * grp / a.groups), h1 = (int)((long long)a.H * (grp + 1) / a.groups);
  for (int i = r0; i < nq * (h1 - h0); i += ROWS) {
    const int t = i / (h1 - h0), h = h0 + i - t * (h1 - h0);
    const size_t tok = (size_t)(lo - start + t);
    float x[8], y[8];
    fsvd_rope::load_unit<WIDE>(a.q + (size_t)b * a.q_batch + tok * a.q_token + (size_t)h * DH, u, R, inter, x, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int p = 8 * u + e;
      if (p < half) {
        const float4 cs = tab[t * half + p];
        const float x0 = x[e], y0 = y[e];
        x[e] = x0 * cs.x - y0 * cs.z;
        y[e] = y0 * cs.x + x0 * cs.z;
      }
    }
    fsvd_rope::store_unit<WIDE>(a.q_out + (((size_t)b * a.L + tok) * a.H + h) * DH, u, R, inter, x, y);
  }
}

// ------------------------------------------------------------------------------------------ read-back
struct LoadArgs {
  fsvd_kv8 c;
  int start, length, seqlen_add;
  const int* seqlens;
  __nv_bfloat16 *k_out, *v_out;
};

// A CTA reads back kThreads * kLoads sixteen-byte pieces in a row of one plane (a sequence's head, keys or values).
constexpr int kLoads = 4;
template <int DH>
__global__ void __launch_bounds__(kThreads) load_kernel(const LoadArgs a) {
  constexpr int V = DH / 16;   // pieces of a row
  pdl_begin();
  const int planes = a.c.B * a.c.Hk, per_plane = (a.length * V + kThreads * kLoads - 1) / (kThreads * kLoads);
  const int plane2 = blockIdx.x / per_plane, first = (blockIdx.x - plane2 * per_plane) * kThreads * kLoads + threadIdx.x;
  const bool second = plane2 >= planes;
  const int bh = second ? plane2 - planes : plane2, nb = (a.c.S_max + a.c.block - 1) / a.c.block;
  const uint8_t* codes = reinterpret_cast<const uint8_t*>(second ? a.c.v8 : a.c.k8) + ((size_t)bh * a.c.S_max + a.start) * DH;
  const float* scales = (second ? a.c.v_scale : a.c.k_scale) + (size_t)bh * nb;
  __nv_bfloat16* out = (second ? a.v_out : a.k_out) + (size_t)bh * a.length * DH;
  const int end = a.seqlens ? (int)min((long long)a.length, max(0ll, (long long)a.seqlens[bh / a.c.Hk] + a.seqlen_add - a.start)) : a.length;
  uint4 w[kLoads];
  float f[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int at = first + i * kThreads, t = at / V;
    w[i] = make_uint4(0u, 0u, 0u, 0u);
    f[i] = 0.0f;
    if (t < end) {
      w[i] = __ldg(reinterpret_cast<const uint4*>(codes) + at);
      f[i] = __ldg(scales + (a.start + t) / a.c.block);
    }
  }
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int at = first + i * kThreads, t = at / V;
    if (t >= a.length) break;
    const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
    uint32_t o[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 p = decode2(x[e] & 0xffffu), q = decode2(x[e] >> 16);
      o[2 * e] = fsvd_rope::pack2(p.x * f[i], p.y * f[i]);
      o[2 * e + 1] = fsvd_rope::pack2(q.x * f[i], q.y * f[i]);
    }
    uint4* dst = reinterpret_cast<uint4*>(out) + 2 * (size_t)at;
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

// ------------------------------------------------------------------------------------------ host
static int check_cache(const fsvd_kv8* c) {
  if (!c || !c->k8 || !c->v8 || !c->k_scale || !c->v_scale) return fail(FSVD_ERR_ARG, "null cache");
  if (c->B < 1 || c->Hk < 1 || c->S_max < 1) return fail(FSVD_ERR_ARG, "bad cache sizes B=%d Hk=%d S_max=%d", c->B, c->Hk, c->S_max);
  if (c->Dh != 64 && c->Dh != 128) return fail(FSVD_ERR_UNSUPPORTED, "head_dim %d unsupported (64, 128)", c->Dh);
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
    return fail(FSVD_ERR_UNSUPPORTED, "block of %d tokens unsupported (16, 32, 64, 128)", c->block);
  if ((long long)c->B * c->Hk > (1 << 22)) return fail(FSVD_ERR_UNSUPPORTED, "B * Hk = %lld is beyond 2^22", (long long)c->B * c->Hk);
  if (c->S_max > (1 << 30)) return fail(FSVD_ERR_UNSUPPORTED, "S_max = %d is beyond 2^30", c->S_max);
  if (!aligned16(c->k8) || !aligned16(c->v8)) return fail(FSVD_ERR_ALIGN, "the cache must be 16-byte aligned");
  return 0;
}
static int check_rotary(const double* inv_freq, int R, int Dh) {
  if (!inv_freq) return 0;
  if (R < 2 || R > Dh || R % 2) return fail(FSVD_ERR_ARG, "rotary_dim %d must be even, 2..%d", R, Dh);
  return 0;
}

constexpr int kMaxCtas = 3;   // attention CTAs of an SM, at most

struct Kv8Ws {
  size_t counters, part, total;
};
static Kv8Ws ws_layout(long long B, long long H, long long Hk, long long Dh) {
  Kv8Ws w;
  w.counters = 256;   // behind the status word (fsvd_workspace_status)
  w.part = w.counters + (size_t)((B * Hk * 4 + 255) / 256 * 256);
  w.total = w.part + (size_t)kMaxCtas * sm_count() * 2 * (H / Hk) * (Dh + fsvd_kv8_attn::kPad) * 4;
  return w;
}

// Descriptor of the codes: B * Hk planes of S_max rows of Dh bytes, read in boxes of kBox rows under the swizzle of a row.
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<EncodeFn>(p) : nullptr;
  }();
  return fn;
}
static int encode(CUtensorMap* map, const void* codes, const fsvd_kv8& c) {
  const EncodeFn enc = encode_fn();
  if (!enc) return fail(FSVD_ERR_CUDA, "cuTensorMapEncodeTiled is not available in this driver");
  const cuuint64_t dims[3] = {(cuuint64_t)c.Dh, (cuuint64_t)c.S_max, (cuuint64_t)c.B * c.Hk};
  const cuuint64_t strides[2] = {(cuuint64_t)c.Dh, (cuuint64_t)c.S_max * c.Dh};
  const cuuint32_t box[3] = {(cuuint32_t)c.Dh, (cuuint32_t)fsvd_kv8_attn::kBox, 1}, es[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(codes), dims, strides, box, es,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, c.Dh == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : fail(FSVD_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
}

template <int DH, int GP>
static int launch_attn(const CUtensorMap& km, const CUtensorMap& vm, const fsvd_kv8_attn::Args& a, void* stream) {
  using S = fsvd_kv8_attn::Shape<DH, GP>;
  static_assert(S::kCtas <= kMaxCtas);
  const long long tiles = (long long)a.B * a.Hk * ((a.S_max + fsvd_kv8_attn::kTile - 1) / fsvd_kv8_attn::kTile);
  const unsigned grid = (unsigned)std::min<long long>(tiles, (long long)S::kCtas * sm_count());
  return launch(fsvd_kv8_attn::attn_kernel<DH, GP>, dim3(grid), S::kThreads, S::kSmem, stream, km, vm, a);
}
template <int DH>
static int launch_attn(const CUtensorMap& km, const CUtensorMap& vm, const fsvd_kv8_attn::Args& a, void* stream) {
  if (a.G == 1) return launch_attn<DH, 1>(km, vm, a, stream);
  if (a.G == 2) return launch_attn<DH, 2>(km, vm, a, stream);
  if (a.G <= 4) return launch_attn<DH, 4>(km, vm, a, stream);
  if (a.G <= 8) return launch_attn<DH, 8>(km, vm, a, stream);
  return launch_attn<DH, 16>(km, vm, a, stream);
}

template <int DH, int BLOCK>
static int launch_append(const AppendArgs& a, size_t smem, unsigned grid, void* stream) {
  if (a.rot.R % 16 == 0) return launch(append_kernel<DH, BLOCK, true>, dim3(grid), kThreads, smem, stream, a);
  return launch(append_kernel<DH, BLOCK, false>, dim3(grid), kThreads, smem, stream, a);
}
template <int DH>
static int launch_append(const AppendArgs& a, size_t smem, unsigned grid, void* stream) {
  switch (a.c.block) {
    case 16: return launch_append<DH, 16>(a, smem, grid, stream);
    case 32: return launch_append<DH, 32>(a, smem, grid, stream);
    case 64: return launch_append<DH, 64>(a, smem, grid, stream);
    default: return launch_append<DH, 128>(a, smem, grid, stream);
  }
}

}  // namespace fsvd_kv8_impl

using namespace fsvd_kv8_impl;

extern "C" {

int fsvd_rope_qk(const void* q, long long q_stride, const void* k, long long k_stride, const int* positions,
                 const double* inv_freq, int rotary_dim, int interleaved, float rope_scale, void* q_out, void* k_out, int T,
                 int H, int Hk, int Dh, int dtype, void* stream) {
  if (!q || !positions || !inv_freq || !q_out || (k != nullptr) != (k_out != nullptr)) return fail(FSVD_ERR_ARG, "null argument");
  if (dtype != FSVD_DTYPE_BF16 && dtype != FSVD_DTYPE_F32) return fail(FSVD_ERR_ARG, "bad dtype %d", dtype);
  if (T < 0 || H < 1 || (k && Hk < 1)) return fail(FSVD_ERR_ARG, "bad sizes T=%d H=%d Hk=%d", T, H, Hk);
  if (Dh < 16 || Dh > 256 || Dh % 16) return fail(FSVD_ERR_UNSUPPORTED, "head_dim %d unsupported (multiples of 16 up to 256)", Dh);
  if (int e = check_rotary(inv_freq, rotary_dim, Dh)) return e;
  const int es = dtype == FSVD_DTYPE_F32 ? 4 : 2;
  if (!k) Hk = 0;
  if (q_stride < 0 || k_stride < 0) return fail(FSVD_ERR_ARG, "negative stride");
  if (!aligned16(q) || !aligned16(k) || !aligned16(q_out) || !aligned16(k_out) || q_stride * es % 16 || (k && k_stride * es % 16))
    return fail(FSVD_ERR_ALIGN, "rows must start on 16-byte boundaries");
  if (T == 0) return 0;
  RopeArgs a;
  a.q = q; a.k = k; a.q_out = q_out; a.k_out = k_out;
  a.q_stride = q_stride; a.k_stride = k_stride; a.positions = positions;
  a.rot = Rotary{inv_freq, rotary_dim, interleaved != 0, rope_scale};
  a.T = T; a.H = H; a.Hk = Hk; a.Dh = Dh;
  // One wave of four CTAs per SM, up to 32 tokens each; a few tokens are shared out by heads.
  a.tokens = std::min(32, (T + 4 * sm_count() - 1) / (4 * sm_count()));
  const int ctas = (T + a.tokens - 1) / a.tokens, splits = std::max(1, std::min({2 * sm_count() / ctas, (H + Hk) * (Dh / 16) / kThreads, 8}));
  a.heads = (H + Hk + splits - 1) / splits;
  const dim3 grid((T + a.tokens - 1) / a.tokens, (H + Hk + a.heads - 1) / a.heads);
  const size_t smem = (size_t)a.tokens * (rotary_dim / 2) * sizeof(float2);
  const bool wide = rotary_dim % 16 == 0;
  if (dtype == FSVD_DTYPE_F32)
    return wide ? launch(rope_kernel<float, true>, grid, kThreads, smem, stream, a)
                : launch(rope_kernel<float, false>, grid, kThreads, smem, stream, a);
  return wide ? launch(rope_kernel<__nv_bfloat16, true>, grid, kThreads, smem, stream, a)
              : launch(rope_kernel<__nv_bfloat16, false>, grid, kThreads, smem, stream, a);
}

size_t fsvd_kv8_workspace_bytes(int B, int H, int Hk, int Dh, int S_max) {
  if (B < 1 || H < 1 || Hk < 1 || (Dh != 64 && Dh != 128) || S_max < 1) return 0;
  return ws_layout(B, H, Hk, Dh).total;
}

int fsvd_kv8_append(const fsvd_kv8* cache, const void* k, const void* v, long long kv_batch_stride, long long kv_token_stride,
                    const int* cache_seqlens, const int* new_lens, const void* q, long long q_batch_stride,
                    long long q_token_stride, void* q_out, const double* inv_freq, int rotary_dim, int interleaved,
                    float rope_scale, int H, int L, void* ws, size_t ws_bytes, void* stream) {
  if (int e = check_cache(cache)) return e;
  if (!k || !v || !cache_seqlens || (q != nullptr) != (q_out != nullptr)) return fail(FSVD_ERR_ARG, "null argument");
  if (q && !inv_freq) return fail(FSVD_ERR_ARG, "queries are passed to be rotated: inv_freq is missing");
  if (int e = check_rotary(inv_freq, rotary_dim, cache->Dh)) return e;
  if (L < 0 || (q && H < 1)) return fail(FSVD_ERR_ARG, "bad sizes L=%d H=%d", L, H);
  if (kv_batch_stride < 0 || kv_token_stride < 0 || q_batch_stride < 0 || q_token_stride < 0) return fail(FSVD_ERR_ARG, "negative stride");
  if (!aligned16(k) || !aligned16(v) || !aligned16(q) || !aligned16(q_out) || kv_batch_stride % 8 || kv_token_stride % 8 ||
      (q && (q_batch_stride % 8 || q_token_stride % 8)))
    return fail(FSVD_ERR_ALIGN, "rows must start on 16-byte boundaries");
  if (!ws || ws_bytes < 256) return fail(FSVD_ERR_WORKSPACE, "no workspace");
  if (!aligned16(ws)) return fail(FSVD_ERR_ALIGN, "workspace is not 16-byte aligned");
  if (L == 0) return 0;
  AppendArgs a;
  a.c = *cache;
  a.k = reinterpret_cast<const __nv_bfloat16*>(k);
  a.v = reinterpret_cast<const __nv_bfloat16*>(v);
  a.q = reinterpret_cast<const __nv_bfloat16*>(q);
  a.q_out = reinterpret_cast<__nv_bfloat16*>(q_out);
  a.kv_batch = kv_batch_stride; a.kv_token = kv_token_stride; a.q_batch = q_batch_stride; a.q_token = q_token_stride;
  a.seqlens = cache_seqlens; a.new_lens = new_lens;
  a.status = &reinterpret_cast<SyncState*>(ws)->status;
  a.rot = Rotary{inv_freq, inv_freq ? rotary_dim : 0, interleaved != 0, rope_scale};
  a.H = q ? H : 0; a.L = L;
  const int BLOCK = cache->block;
  a.nblk = (int)(((long long)L + BLOCK - 2) / BLOCK + 1);
  // Heads of a CTA share the table of angles: with rotation as few groups as still give every SM two CTAs.
  a.groups = cache->Hk;
  if (inv_freq)
    while (a.groups % 2 == 0 && (long long)cache->B * a.nblk * (a.groups / 2) >= 2ll * sm_count()) a.groups /= 2;
  const long long grid = (long long)cache->B * a.nblk * a.groups;
  if (grid > 0x7fffffffll) return fail(FSVD_ERR_UNSUPPORTED, "too many tokens for one call");
  const int tile = std::min(BLOCK, L);
  const size_t smem = (size_t)(a.rot.R / 2) * (tile * sizeof(float4) + (tile > 8 ? (8 + (tile + 7) / 8) * sizeof(double2) : 0));
  return cache->Dh == 64 ? launch_append<64>(a, smem, (unsigned)grid, stream) : launch_append<128>(a, smem, (unsigned)grid, stream);
}

int fsvd_kv8_load(const fsvd_kv8* cache, int start, int length, const int* cache_seqlens, int seqlen_add, void* k_out,
                  void* v_out, void* stream) {
  if (int e = check_cache(cache)) return e;
  if (!k_out || !v_out) return fail(FSVD_ERR_ARG, "null argument");
  if (start < 0 || length < 0 || (long long)start + length > cache->S_max)
    return fail(FSVD_ERR_ARG, "positions %d + %d are outside the cache (%d)", start, length, cache->S_max);
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(FSVD_ERR_ALIGN, "outputs must be 16-byte aligned");
  if (length == 0) return 0;
  LoadArgs a = {*cache, start, length, seqlen_add, cache_seqlens, reinterpret_cast<__nv_bfloat16*>(k_out),
                reinterpret_cast<__nv_bfloat16*>(v_out)};
  const long long grid = 2ll * cache->B * cache->Hk * (((long long)length * (cache->Dh / 16) + kThreads * kLoads - 1) / (kThreads * kLoads));
  if (grid > 0x7fffffffll) return fail(FSVD_ERR_UNSUPPORTED, "too many tokens for one call");
  return cache->Dh == 64 ? launch(load_kernel<64>, dim3((unsigned)grid), kThreads, 0, stream, a)
                         : launch(load_kernel<128>, dim3((unsigned)grid), kThreads, 0, stream, a);
}

int fsvd_flash_decode_kv8(const fsvd_kv8* cache, const void* q, const int* cache_seqlens, int seqlen_add, void* out, int H,
                          float scale, void* ws, size_t ws_bytes, void* stream) {
  if (int e = check_cache(cache)) return e;
  if (!q || !cache_seqlens || !out) return fail(FSVD_ERR_ARG, "null argument");
  if (H < 1 || H % cache->Hk) return fail(FSVD_ERR_ARG, "H=%d not a multiple of Hk=%d", H, cache->Hk);
  const int G = H / cache->Hk;
  if (G > fsvd_kv8_attn::kMaxGroup)
    return fail(FSVD_ERR_UNSUPPORTED, "H/Hk=%d unsupported (1..%d)", G, fsvd_kv8_attn::kMaxGroup);
  if (!aligned16(q) || !aligned16(out)) return fail(FSVD_ERR_ALIGN, "q and out must be 16-byte aligned");
  const Kv8Ws L = ws_layout(cache->B, H, cache->Hk, cache->Dh);
  if (!ws) return fail(FSVD_ERR_WORKSPACE, "null workspace");
  if (!aligned16(ws)) return fail(FSVD_ERR_ALIGN, "workspace is not 16-byte aligned");
  if (ws_bytes < L.total) return fail(FSVD_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", ws_bytes, L.total);
  CUtensorMap km, vm;
  if (int e = encode(&km, cache->k8, *cache)) return e;
  if (int e = encode(&vm, cache->v8, *cache)) return e;
  fsvd_kv8_attn::Args a;
  a.k_scale = cache->k_scale;
  a.v_scale = cache->v_scale;
  a.q = reinterpret_cast<const __nv_bfloat16*>(q);
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.seqlens = cache_seqlens;
  a.part = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + L.part);
  a.counters = reinterpret_cast<int*>(reinterpret_cast<char*>(ws) + L.counters);
  a.status = &reinterpret_cast<SyncState*>(ws)->status;
  a.wait_limit = fsvd_tile_wait_limit();
  a.B = cache->B; a.Hk = cache->Hk; a.S_max = cache->S_max;
  a.block_log2 = cache->block == 16 ? 4 : cache->block == 32 ? 5 : cache->block == 64 ? 6 : 7;
  a.nb = (cache->S_max + cache->block - 1) / cache->block;
  a.G = G; a.seqlen_add = seqlen_add;
  a.scale = scale > 0.0f ? scale : 1.0f / sqrtf((float)cache->Dh);
  return cache->Dh == 64 ? launch_attn<64>(km, vm, a, stream) : launch_attn<128>(km, vm, a, stream);
}

}  // extern "C"

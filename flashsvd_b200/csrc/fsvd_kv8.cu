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
#include <type_traits>
#include <atomic>

#include "../../include/flashsvd_b200.h"
#include "fsvd_kv8_attn.cuh"
#include "fsvd_rope.cuh"
#include "fsvd_smem.h"
#include "fsvd_stage.h"
#include "fsvd_tile.h"

namespace fsvd_kv8_impl {

using fsvd::DS_CACHE_FULL;
using fsvd::DS_OK;
using fsvd::SyncState;
using fsvd_rope::Form;
using fsvd_rope::kSingle;
using fsvd_rope::kTogether;
using fsvd_rope::kVectors;
using fsvd_rope::Rotary;

static int fail(int code, const char* fmt, ...) {
  char msg[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  if (code == FSVD_ERR_CUDA) cudaGetLastError();   // (off the thread: no later check of the caller's reports it again)
  fsvd_tile_set_error(code, msg);
  return code;
}
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }

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
template <auto KERNEL, typename... Args>
static int launch(dim3 grid, int threads, size_t smem, void* stream, const Args&... args) {
  // Above the 48 KB that a kernel has by itself its limit is raised, to all that there is: another thread's launch of another
  // size finds it as it needs it.
  cudaError_t e = cudaSuccess;
  if (smem > 48 * 1024) {
    static fsvd_tile::SmemLimit limit;
    e = limit.raise(KERNEL);
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
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, KERNEL, args...);
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
  bool on32;                         // all rows begin on boundaries of 32 bytes
};
constexpr int kRopeTokens = 32;
constexpr int kMaxHeads = 1 << 16;

// A CTA turns `tokens` rows of heads; its threads go through the (token, head, unit) list in steps of kThreads, several units
// at a time so that their loads are under way together.
template <typename T, Form FORM>
__global__ void __launch_bounds__(kThreads, 4) rope_kernel(const RopeArgs a) {
  constexpr int N = 2;                              // units at a time
  extern __shared__ __align__(16) float2 table[];   // per token: cosine and sine of the pairs, in slots (below)
  const int half = a.rot.R >> 1, tid = threadIdx.x, R = a.rot.R, inter = a.rot.interleaved;
  const int t0 = blockIdx.x * a.tokens, nt = min(a.tokens, a.T - t0);
  // Two neighbouring pairs of a unit share 16 bytes; neighbouring units lie next to each other, so that the lanes of a warp
  // read from different banks.
  const int units = (half + 7) / 8, row_slots = 8 * units;
  auto slot_of = [&](int two, int unit) { return two * units + unit; };
  pdl_begin();
  for (int i = tid; i < nt * half; i += kThreads) {
    double c, s;
    const int t = i / half, p = i - t * half;
    fsvd_rope::angle(a.positions[t0 + t], a.rot.inv_freq[p], a.rot.scale, c, s);
    table[t * row_slots + 2 * slot_of((p & 7) >> 1, p >> 3) + (p & 1)] = make_float2((float)c, (float)s);
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
        fsvd_rope::load_unit<FORM>(src, unit[k], R, inter, x[k], y[k]);
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
        const float4* cs = reinterpret_cast<const float4*>(table + token[k] * row_slots);
        // (pairs that are not rotated are copied: an infinity times a sine of zero is no number)
        if (8 * unit[k] < half) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float4 two = cs[slot_of(e >> 1, unit[k])];
            if (FORM != kSingle || 8 * unit[k] + e < half) turn(e, two.x, two.y);
            if (FORM != kSingle || 8 * unit[k] + e + 1 < half) turn(e + 1, two.z, two.w);
          }
        }
        fsvd_rope::store_unit<FORM>(dst[k], unit[k], R, inter, x[k], y[k]);
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
  bool on32;   // all rows of k, v and q begin on boundaries of 32 bytes
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

// A bf16 number as fp64 by its bits, finite ones only (the conversion instruction runs at an eighth of the rate; a zero
// comes out as 2^-127, which no code can tell from it).
__device__ __forceinline__ double wide(float x) {
  const uint32_t b = __float_as_uint(x);
  return __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), 0);
}

__device__ __forceinline__ uint32_t turn_key(uint32_t w, double2 cs) {
  const float fx = __uint_as_float(w << 16), fy = __uint_as_float(w & 0xffff0000u);
  double x = wide(fx), y = wide(fy);
  if ((w & 0x7f80u) == 0x7f80u) x = (double)fx;
  if ((w & 0x7f800000u) == 0x7f800000u) y = (double)fy;
  return fsvd_rope::pack2((float)(x * cs.x - y * cs.y), (float)(y * cs.x + x * cs.y));
}
__device__ __forceinline__ uint32_t turn_query(uint32_t w, float c, float s) {
  const float x = __uint_as_float(w << 16), y = __uint_as_float(w & 0xffff0000u);
  return fsvd_rope::pack2(x * c - y * s, y * c + x * s);
}

// Scales and codes of one thread's share of a tile: eight packed pairs of bf16 numbers (a in the low half).
struct Share {
  uint32_t top = 0;   // largest magnitude, as the bits of a bf16 number
  bool odd = false;   // something is not finite
};
__device__ __forceinline__ void largest(const uint32_t (&w)[8], Share& s) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  s.top = max(m & 0xffffu, m >> 16);
  if (s.top >= 0x7f80u) {   // the finite ones alone
    s.odd = true;
    s.top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t x = w[i] & 0x7fffu, y = (w[i] >> 16) & 0x7fffu;
      if (x < 0x7f80u) s.top = max(s.top, x);
      if (y < 0x7f80u) s.top = max(s.top, y);
    }
  }
}
__device__ __noinline__ uint32_t careful_codes(uint32_t w, float inv) {
  float x = __uint_as_float(w << 16) * inv, y = __uint_as_float(w & 0xffff0000u) * inv;
  if (inv <= 0x1p-120f) {   // 256 * 2^120 is no 32-bit number any more
    x = fabsf(x) > 240.0f && isfinite(x) ? copysignf(240.0f, x) : x;
    y = fabsf(y) > 240.0f && isfinite(y) ? copysignf(240.0f, y) : y;
  }
  return code2(x, y);
}
// Code pairs of one row, times inv (a power of two).
__device__ __forceinline__ void codes_of(const uint32_t (&w)[8], float inv, bool odd, uint32_t (&cd)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    cd[i] = __nv_cvt_float2_to_fp8x2(make_float2(__uint_as_float(w[i] << 16) * inv, __uint_as_float(w[i] & 0xffff0000u) * inv),
                                     __NV_SATFINITE, __NV_E4M3);
  if (odd || inv <= 0x1p-120f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) cd[i] = careful_codes(w[i], inv);
  }
}
template <Form FORM>
__device__ __forceinline__ void store_codes(uint8_t* dst, const uint32_t (&cd)[8], int u, int R, int inter) {
  const int half = R >> 1;
  if constexpr (FORM != kSingle) {
    const bool split = !inter && 16 * u < R;
    const uint32_t a03 = __byte_perm(cd[0] | (cd[1] << 16), cd[2] | (cd[3] << 16), 0x6420);
    const uint32_t a47 = __byte_perm(cd[4] | (cd[5] << 16), cd[6] | (cd[7] << 16), 0x6420);
    const uint32_t b03 = __byte_perm(cd[0] | (cd[1] << 16), cd[2] | (cd[3] << 16), 0x7531);
    const uint32_t b47 = __byte_perm(cd[4] | (cd[5] << 16), cd[6] | (cd[7] << 16), 0x7531);
    const uint2 first = split ? make_uint2(a03, a47) : make_uint2(cd[0] | (cd[1] << 16), cd[2] | (cd[3] << 16));
    const uint2 second = split ? make_uint2(b03, b47) : make_uint2(cd[4] | (cd[5] << 16), cd[6] | (cd[7] << 16));
    if (split) {
      *reinterpret_cast<uint2*>(dst + 8 * u) = first;
      *reinterpret_cast<uint2*>(dst + 8 * u + half) = second;
    } else {
      *reinterpret_cast<uint4*>(dst + 16 * u) = make_uint4(first.x, first.y, second.x, second.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int2 at = fsvd_rope::pair_at(8 * u + i, R, inter);
      dst[at.x] = (uint8_t)(cd[i] & 0xffu);
      dst[at.y] = (uint8_t)(cd[i] >> 8);
    }
  }
}

// Four codes at a larger scale: times f = old scale / new scale.
__device__ __forceinline__ uint32_t rescaled(uint32_t x, float f) {
  const float2 p = decode2(x & 0xffffu), q = decode2(x >> 16);
  return code2(p.x * f, p.y * f) | (code2(q.x * f, q.y * f) << 16);
}

// One CTA per (sequence, block of the cache, group of kv heads): a tile of at most BLOCK tokens x DH of a head sits in
// registers (bf16) between the maximum and the rounding, so that each input is read once and each code written once.  Keys
// are turned in 64 bits, then rounded to 32 and 16: a rotated key falls on the same side of a rounding border as in
// exact arithmetic.
// A thread to a unit of the tile.  CTAS of them to an SM: 512 threads of 128 registers, where a thread has its reads of the
// table under way together, or 1024 of 64 (MANY), which overlap better once there is much to do.
template <int DH, int BLOCK> constexpr int kAppendThreads = BLOCK * DH / 16;
template <int DH, int BLOCK, bool MANY> constexpr int kAppendCtas = std::max(1, (MANY ? 1024 : 512) / kAppendThreads<DH, BLOCK>);
template <int DH, int BLOCK, Form FORM, bool MANY>
__global__ void __launch_bounds__(kAppendThreads<DH, BLOCK>, kAppendCtas<DH, BLOCK, MANY>) append_kernel(const AppendArgs a) {
  constexpr int kThreads = kAppendThreads<DH, BLOCK>, U = DH / 16;
  extern __shared__ double2 tab[];   // per token: cosine and sine of the pairs
  __shared__ uint32_t red[2][2][kThreads / 32];
  const int tid = threadIdx.x, u = tid % U, t = tid / U;   // this thread's unit and token of the tile
  int idx = blockIdx.x;
  const int grp = idx % a.groups;
  idx /= a.groups;
  const int j = idx % a.nblk, b = idx / a.nblk;
  pdl_begin();
  const int start = max(a.seqlens[b], 0);
  const int count = a.new_lens ? min(max(a.new_lens[b], 0), a.L) : a.L;
  const long long end_ll = (long long)start + count;
  const int end = (int)min(end_ll, (long long)a.c.S_max);
  if (count > 0 && end_ll > a.c.S_max && j == 0 && grp == 0 && tid == 0) atomicCAS(a.status, (int)DS_OK, (int)DS_CACHE_FULL);
  const int blk = start / BLOCK + j;
  const long long blk0 = (long long)blk * BLOCK;
  if (blk0 >= end_ll) return;
  const long long lo = max((long long)start, blk0);   // position of this tile's first new token (behind 2^31 for a length near it)
  const int from = (int)(lo - start);                 // and its place among the call's
  // (queries of tokens beyond the cache are rotated too: their range is not cut at the capacity)
  const int nq = (int)(min(end_ll, blk0 + BLOCK) - lo), n = (int)max(0ll, min((long long)end, blk0 + BLOCK) - lo);
  const int R = a.rot.R, half = R >> 1, inter = a.rot.interleaved;
  // pair p of a token sits in slot (p % 8) * units + p / 8: the lanes of a warp, a unit of eight pairs each, read neighbours
  const int units = (half + 7) / 8, slots = 8 * units;
  const int Hk = a.c.Hk, nb = (a.c.S_max + BLOCK - 1) / BLOCK;
  const int hk0 = (int)((long long)Hk * grp / a.groups), hk1 = (int)((long long)Hk * (grp + 1) / a.groups);
  uint32_t kreg[8], vreg[8];   // packed pairs (a, b)
  auto fetch = [&](int hk) {
#pragma unroll
    for (int i = 0; i < 8; ++i) kreg[i] = vreg[i] = 0u;
    if (t < n) {
      const size_t off = (size_t)b * a.kv_batch + (size_t)(from + t) * a.kv_token + (size_t)hk * DH;
      fsvd_rope::load_pairs<FORM>(a.k + off, u, R, inter, kreg);
      fsvd_rope::load_pairs<FORM>(a.v + off, u, R, inter, vreg);
    }
  };
  if (n > 0 && hk0 < hk1) fetch(hk0);   // (the first head is under way while the angles are formed)
  if (R) {
    // Cosines and sines of the tile's tokens.  More than a few: of every eighth token and of steps 0..7, and the products of
    // those (64 tokens: 16 evaluations a pair instead of 64).
    auto pair_of = [&](int slot) { return slot % units * 8 + slot / units; };
    const int coarse = (nq + 7) / 8;
    double2* steps = nq <= 8 ? tab : tab + min(BLOCK, a.L) * slots;   // [8 + coarse][slots]
    for (int i = tid; i < (nq <= 8 ? nq : 8 + coarse) * slots; i += kThreads) {
      const int k = i / slots, p = pair_of(i - k * slots);
      if (p >= half) continue;
      const bool step = nq > 8 && k < 8;
      double c, s;
      fsvd_rope::angle((double)(step ? k : nq <= 8 ? lo + k : lo + 8 * (k - 8)), a.rot.inv_freq[p], step ? 1.0 : a.rot.scale, c, s);
      steps[i] = make_double2(c, s);
    }
    __syncthreads();
    if (nq > 8) {
      for (int s0 = tid % 32; s0 < slots; s0 += 32)
        for (int k = tid / 32; k < nq; k += kThreads / 32) {
          const double2 x = steps[(8 + (k >> 3)) * slots + s0], y = steps[(k & 7) * slots + s0];
          tab[k * slots + s0] = make_double2(x.x * y.x - x.y * y.y, x.y * y.x + x.x * y.y);
        }
      __syncthreads();
    }
  }
  const bool turns = 8 * u < half;
  const double2* my_tab = tab + u;   // pair i of this unit: my_tab[token * slots + i * units]
  const bool held = start > blk0;   // the block holds tokens already
  int parity = 0;
  for (int hk = hk0; hk < hk1 && n > 0; ++hk, parity ^= 1) {
    const size_t si = ((size_t)b * Hk + hk) * nb + blk;
    const float kold = held ? a.c.k_scale[si] : 0.0f, vold = held ? a.c.v_scale[si] : 0.0f;
    if (turns && t < n) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (FORM == kSingle && 8 * u + i >= half) break;
        kreg[i] = turn_key(kreg[i], my_tab[t * slots + i * units]);
      }
    }
    Share ks, vs;
    largest(kreg, ks);
    largest(vreg, vs);
    const uint32_t kwarp = __reduce_max_sync(0xffffffffu, ks.top), vwarp = __reduce_max_sync(0xffffffffu, vs.top);
    if ((tid & 31) == 0) {
      red[parity][0][tid >> 5] = kwarp;
      red[parity][1][tid >> 5] = vwarp;
    }
    __syncthreads();   // (two halves of `red` in turn: the next head writes the other one)
    uint32_t kbits = 0, vbits = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      kbits = max(kbits, red[parity][0][w]);
      vbits = max(vbits, red[parity][1][w]);
    }
    const float kscale = fmaxf(kold, two_to(scale_exponent(__uint_as_float(kbits << 16))));
    const float vscale = fmaxf(vold, two_to(scale_exponent(__uint_as_float(vbits << 16))));
    const size_t base = (((size_t)b * Hk + hk) * a.c.S_max + (size_t)blk0) * DH;
    uint8_t* kc = reinterpret_cast<uint8_t*>(a.c.k8) + base;
    uint8_t* vc = reinterpret_cast<uint8_t*>(a.c.v8) + base;
    if (held) {   // a larger scale: round what the block holds once more
      const int old_bytes = (int)(start - blk0) * DH;
      for (int which = 0; which < 2; ++which) {
        const float was = which ? vold : kold, now = which ? vscale : kscale;
        if (!(now > was)) continue;
        uint32_t* w = reinterpret_cast<uint32_t*>(which ? vc : kc);
        const float f = was / now;
        for (int i = tid; i < old_bytes / 4; i += kThreads) w[i] = rescaled(w[i], f);
      }
    }
    const float ki = 1.0f / kscale, vi = 1.0f / vscale;
    if (t < n) {
      const size_t row = (size_t)(lo - blk0 + t) * DH;
      uint32_t cd[8];   // codes of the pairs: low byte a, high byte b
      codes_of(kreg, ki, ks.odd, cd);
      store_codes<FORM>(kc + row, cd, u, R, inter);
      codes_of(vreg, vi, vs.odd, cd);
      store_codes<FORM>(vc + row, cd, u, R, inter);
    }
    if (tid == 0) {
      a.c.k_scale[si] = kscale;
      a.c.v_scale[si] = vscale;
    }
    if (hk + 1 < hk1) fetch(hk + 1);
  }
  if (!a.q || t >= nq) return;
  // queries: a thread keeps its token's cosines and sines while it goes through the heads, several at a time
  constexpr int kHeads = MANY ? 2 : 4;
  const int h0 = (int)((long long)a.H * grp / a.groups), h1 = (int)((long long)a.H * (grp + 1) / a.groups);
  float c[8], s[8];
  if (turns) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = FORM != kSingle || 8 * u + i < half;
      const double2 cs = my_tab[t * slots + (in ? i * units : 0)];
      c[i] = (float)cs.x;
      s[i] = (float)cs.y;
    }
  }
  const size_t tok = (size_t)(from + t);
  const __nv_bfloat16* src = a.q + (size_t)b * a.q_batch + tok * a.q_token;
  __nv_bfloat16* dst = a.q_out + ((size_t)b * a.L + tok) * a.H * DH;
  auto turn_heads = [&](auto many, int h) {
    constexpr int N = decltype(many)::value;
    uint32_t w[N][8];
#pragma unroll
    for (int k = 0; k < N; ++k) fsvd_rope::load_pairs<FORM>(src + (size_t)(h + k) * DH, u, R, inter, w[k]);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (FORM == kSingle && 8 * u + i >= half) break;
          w[k][i] = turn_query(w[k][i], c[i], s[i]);
        }
      }
      fsvd_rope::store_pairs<FORM>(dst + (size_t)(h + k) * DH, u, R, inter, w[k]);
    }
  };
  int h = h0;
  for (; h + kHeads <= h1; h += kHeads) turn_heads(std::integral_constant<int, kHeads>{}, h);
  for (; h < h1; ++h) turn_heads(std::integral_constant<int, 1>{}, h);
}

// A single token per sequence: the rows of a CTA are heads, not tokens, so that every thread has a share (the kernel above
// would leave all rows but one idle: a step of 128 sequences with 32 heads took 32.2 us, here 5.0; of 8 sequences 4.4 and 3.8).
// Almost all of a small step is latency: one load, one sine in 64 bits (about 1500 clocks), one store.
template <int DH, Form FORM>
__global__ void __launch_bounds__(kThreads) append_step_kernel(const AppendArgs a) {
  constexpr int U = DH / 16;
  __shared__ double2 tab[DH / 2];   // pair p in slot (p % 8) * units + p / 8
  const int tid = threadIdx.x, u = tid % U, lane = tid & 31;
  const int grp = blockIdx.x % a.groups, b = blockIdx.x / a.groups;
  const int R = a.rot.R, half = R >> 1, inter = a.rot.interleaved, units = (half + 7) / 8, BLOCK = a.c.block;
  const int Hk = a.c.Hk, nb = (a.c.S_max + BLOCK - 1) / BLOCK;
  const int hk = (int)((long long)Hk * grp / a.groups) + tid / U, h = (int)((long long)a.H * grp / a.groups) + tid / U;
  const bool has_q = h < (int)((long long)a.H * (grp + 1) / a.groups);
  pdl_begin();
  if (a.new_lens && a.new_lens[b] <= 0) return;
  const int start = max(a.seqlens[b], 0);
  if (start >= a.c.S_max && grp == 0 && tid == 0) atomicCAS(a.status, (int)DS_OK, (int)DS_CACHE_FULL);
  const bool has_kv = start < a.c.S_max && hk < (int)((long long)Hk * (grp + 1) / a.groups);
  const int blk = start / BLOCK, old = start - blk * BLOCK;   // tokens that the block holds already
  const size_t si = ((size_t)b * Hk + hk) * nb + blk;
  uint32_t kw[8], vw[8], qw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) kw[i] = vw[i] = 0u;
  float kold = 0.0f, vold = 0.0f;
  if (has_kv) {
    const size_t off = (size_t)b * a.kv_batch + (size_t)hk * DH;
    fsvd_rope::load_pairs<FORM>(a.k + off, u, R, inter, kw);
    fsvd_rope::load_pairs<FORM>(a.v + off, u, R, inter, vw);
    if (old) {
      kold = a.c.k_scale[si];
      vold = a.c.v_scale[si];
    }
  }
  if (has_q) fsvd_rope::load_pairs<FORM>(a.q + (size_t)b * a.q_batch + (size_t)h * DH, u, R, inter, qw);
  if (tid < half) {
    double c, s;
    fsvd_rope::angle(start, a.rot.inv_freq[tid], a.rot.scale, c, s);
    tab[(tid & 7) * units + (tid >> 3)] = make_double2(c, s);
  }
  __syncthreads();
  if (8 * u < half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (FORM == kSingle && 8 * u + i >= half) break;
      const double2 cs = tab[i * units + u];
      if (has_kv) kw[i] = turn_key(kw[i], cs);
      if (has_q) qw[i] = turn_query(qw[i], (float)cs.x, (float)cs.y);
    }
  }
  if (has_q) fsvd_rope::store_pairs<FORM>(a.q_out + ((size_t)b * a.H + h) * DH, u, R, inter, qw);
  Share ks, vs;
  largest(kw, ks);
  largest(vw, vs);
  uint32_t kbits = ks.top, vbits = vs.top;
#pragma unroll
  for (int d = 1; d < U; d *= 2) {
    kbits = max(kbits, __shfl_xor_sync(0xffffffffu, kbits, d));
    vbits = max(vbits, __shfl_xor_sync(0xffffffffu, vbits, d));
  }
  const float kscale = fmaxf(kold, two_to(scale_exponent(__uint_as_float(kbits << 16))));
  const float vscale = fmaxf(vold, two_to(scale_exponent(__uint_as_float(vbits << 16))));
  const size_t base = (((size_t)b * Hk + hk) * a.c.S_max + (size_t)blk * BLOCK) * DH;
  __syncwarp();   // (a row's lanes have read its scales)
  if (has_kv) {
    uint32_t cd[8];
    codes_of(kw, 1.0f / kscale, ks.odd, cd);
    store_codes<FORM>(reinterpret_cast<uint8_t*>(a.c.k8) + base + (size_t)old * DH, cd, u, R, inter);
    codes_of(vw, 1.0f / vscale, vs.odd, cd);
    store_codes<FORM>(reinterpret_cast<uint8_t*>(a.c.v8) + base + (size_t)old * DH, cd, u, R, inter);
    if (u == 0) {
      a.c.k_scale[si] = kscale;
      a.c.v_scale[si] = vscale;
    }
  }
  // A larger scale: round what the block holds once more, a warp together for each of its heads.
  for (int which = 0; which < 2; ++which) {
    const float was = which ? vold : kold, now = which ? vscale : kscale;
    for (uint32_t grown = __ballot_sync(0xffffffffu, has_kv && old && u == 0 && now > was); grown; grown &= grown - 1) {
      const int from = __ffs(grown) - 1;
      const float f = __shfl_sync(0xffffffffu, was / now, from);
      uint8_t* codes = reinterpret_cast<uint8_t*>(which ? a.c.v8 : a.c.k8) + __shfl_sync(0xffffffffu, base, from);
      uint4* p = reinterpret_cast<uint4*>(codes);
      for (int i = lane; i < old * DH / 16; i += 128) {
        uint4 x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + 32 * e < old * DH / 16) x[e] = p[i + 32 * e];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + 32 * e < old * DH / 16)
            p[i + 32 * e] = make_uint4(rescaled(x[e].x, f), rescaled(x[e].y, f), rescaled(x[e].z, f), rescaled(x[e].w, f));
      }
    }
  }
}

// ------------------------------------------------------------------------------------------ read-back
struct LoadArgs {
  fsvd_kv8 c;
  int start, length, seqlen_add;
  const int* seqlens;
  __nv_bfloat16 *k_out, *v_out;
  bool on32;   // which begin on boundaries of 32 bytes
};

// A thread reads back one sixteen-byte piece, counted through all planes (a sequence's head, keys or values): a short plane
// leaves no thread idle, and many small CTAs hide the way from memory better than several pieces of a thread do (8 x 191
// tokens with 32 heads of 128: 7.2 us, with two pieces 8.3, with four 10.4; 6.7 with stores of 32 bytes).
template <int DH>
__global__ void __launch_bounds__(kThreads) load_kernel(const LoadArgs a) {
  constexpr int V = DH / 16;   // pieces of a row
  pdl_begin();
  const unsigned planes = (unsigned)(a.c.B * a.c.Hk), pieces = (unsigned)a.length * V, nb = (a.c.S_max + a.c.block - 1) / a.c.block;
  const unsigned long long first = (unsigned long long)blockIdx.x * kThreads;
  const unsigned plane0 = (first >> 32) ? (unsigned)(first / pieces) : (unsigned)first / pieces;
  const unsigned off = (unsigned)(first - (unsigned long long)plane0 * pieces) + threadIdx.x, up = off / pieces;
  const unsigned at = off - up * pieces, plane = plane0 + up;
  if (plane >= 2 * planes) return;
  const bool second = plane >= planes;
  const unsigned bh = second ? plane - planes : plane;
  const int t = a.start + (int)(at / V);
  uint4 w = make_uint4(0u, 0u, 0u, 0u);
  float f = 0.0f;
  if (!a.seqlens || t < (long long)a.seqlens[bh / (unsigned)a.c.Hk] + a.seqlen_add) {
    const uint8_t* codes = reinterpret_cast<const uint8_t*>(second ? a.c.v8 : a.c.k8) + ((size_t)bh * a.c.S_max + a.start) * DH;
    w = __ldg(reinterpret_cast<const uint4*>(codes) + at);
    f = __ldg((second ? a.c.v_scale : a.c.k_scale) + (size_t)bh * nb + t / a.c.block);
  }
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
  uint32_t o[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 p = decode2(x[e] & 0xffffu), q = decode2(x[e] >> 16);
    o[2 * e] = fsvd_rope::pack2(p.x * f, p.y * f);
    o[2 * e + 1] = fsvd_rope::pack2(q.x * f, q.y * f);
  }
  uint4* dst = reinterpret_cast<uint4*>(second ? a.v_out : a.k_out) + 2 * ((size_t)bh * pieces + at);
  if (a.on32) {
    fsvd_rope::store32(dst, o);
  } else {
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
// The counters' place and number depend on the device alone: what a call of other sizes leaves in its partial sums is never
// read as a counter.
static Kv8Ws ws_layout(long long H, long long Hk, long long Dh) {
  Kv8Ws w;
  const size_t ctas = (size_t)kMaxCtas * sm_count();
  w.counters = 256;   // behind the status word (fsvd_workspace_status)
  w.part = w.counters + (ctas * 4 + 255) / 256 * 256;
  w.total = w.part + ctas * 2 * (H / Hk) * (Dh + fsvd_kv8_attn::kPad) * 4;
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
  return launch<fsvd_kv8_attn::attn_kernel<DH, GP>>(dim3(grid), S::kThreads, S::kSmem, stream, km, vm, a);
}
template <int DH>
static int launch_attn(const CUtensorMap& km, const CUtensorMap& vm, const fsvd_kv8_attn::Args& a, void* stream) {
  if (a.G == 1) return launch_attn<DH, 1>(km, vm, a, stream);
  if (a.G == 2) return launch_attn<DH, 2>(km, vm, a, stream);
  if (a.G <= 4) return launch_attn<DH, 4>(km, vm, a, stream);
  if (a.G <= 8) return launch_attn<DH, 8>(km, vm, a, stream);
  return launch_attn<DH, 16>(km, vm, a, stream);
}

static int launch_rope(RopeArgs& a, int dtype, void* stream) {
  // One wave of four CTAs per SM, up to 32 tokens each; a few tokens are shared out by heads.
  const int all = a.H + a.Hk;
  const long long T = a.T;
  a.tokens = (int)std::min<long long>(kRopeTokens, (T + 4 * sm_count() - 1) / (4 * sm_count()));
  const int ctas = (int)((T + a.tokens - 1) / a.tokens), splits = std::max(1, std::min({2 * sm_count() / ctas, all * (a.Dh / 16) / kThreads, 8}));
  a.heads = (all + splits - 1) / splits;
  const dim3 grid(ctas, (all + a.heads - 1) / a.heads);
  const size_t smem = (size_t)a.tokens * ((a.rot.R / 2 + 7) / 8 * 8) * sizeof(float2);
  const Form form = a.rot.R % 16 ? kSingle : dtype == FSVD_DTYPE_BF16 && a.rot.interleaved && a.on32 ? kTogether : kVectors;
  if (dtype == FSVD_DTYPE_F32)
    return form == kSingle ? launch<rope_kernel<float, kSingle>>(grid, kThreads, smem, stream, a)
                           : launch<rope_kernel<float, kVectors>>(grid, kThreads, smem, stream, a);
  return form == kSingle    ? launch<rope_kernel<__nv_bfloat16, kSingle>>(grid, kThreads, smem, stream, a)
         : form == kVectors ? launch<rope_kernel<__nv_bfloat16, kVectors>>(grid, kThreads, smem, stream, a)
                            : launch<rope_kernel<__nv_bfloat16, kTogether>>(grid, kThreads, smem, stream, a);
}

static Form form_of(const AppendArgs& a) {
  return a.rot.R % 16 ? kSingle : a.on32 && (a.rot.interleaved || !a.rot.R) ? kTogether : kVectors;
}
template <int DH, int BLOCK, Form FORM, bool MANY>
static int launch_append(AppendArgs a, void* stream) {
  // Heads of a CTA share the table of angles.  Of the groupings by halves the one with the least waves x (planes of a CTA +
  // kTable), the table being worth about as much as four planes (keys, values or queries of a head).  Beside as few groups
  // as give each SM two CTAs, then: 1024 tokens with 32 heads of 128 15.1 us (19.7), 2 x 1024 with 16 heads of 64 9.3 (12.6).
  constexpr int kTable = 4;
  const long long tiles = (long long)a.c.B * ((a.L + BLOCK - 1) / BLOCK), fit = (long long)kAppendCtas<DH, BLOCK, MANY> * sm_count();
  auto cost = [&](int g) {
    return (tiles * g + fit - 1) / fit * (2 * ((a.c.Hk + g - 1) / g) + (a.H + g - 1) / g + (a.rot.R ? kTable : 0));
  };
  a.groups = std::max(a.H, a.c.Hk);
  for (int g = a.groups; g > 1 && g % 2 == 0; g /= 2)
    if (cost(g / 2) < cost(a.groups)) a.groups = g / 2;
  const long long grid = (long long)a.c.B * a.nblk * a.groups;
  if (grid > 0x7fffffffll) return fail(FSVD_ERR_UNSUPPORTED, "too many tokens for one call");
  const int tile = std::min(BLOCK, a.L);
  const size_t smem = (size_t)((a.rot.R / 2 + 7) / 8 * 8) * (tile + (tile > 8 ? 8 + (tile + 7) / 8 : 0)) * sizeof(double2);
  return launch<append_kernel<DH, BLOCK, FORM, MANY>>(dim3((unsigned)grid), kAppendThreads<DH, BLOCK>, smem, stream, a);
}
template <int DH, int BLOCK, Form FORM>
static int launch_append(const AppendArgs& a, void* stream) {
  // Rows (a head's token of keys, values or queries) of an SM from which 1024 threads are ahead; us at 512 and 1024 threads,
  // heads of 128: 512 tokens with 32 heads (331 rows) 9.8 and 10.7, 1024 (662) 14.6 and 15.2, 2041 (1320) 27.7 and 25.7, 4096
  // with 32 and 8 (1328) 22.5 and 21.3, 4 x 1024 with 64 and 8 in blocks of 32 (2213) 32.1 and 30.8.  Without rotation there
  // is no table to wait for: 2041 tokens 18.4 and 13.4.  Heads of 64: 2 x 2000 with 32 heads (2595) 25.9 and 27.0.
  if constexpr (kAppendThreads<DH, BLOCK> >= 1024) {
    return launch_append<DH, BLOCK, FORM, true>(a, stream);
  } else if constexpr (DH == 64 || FORM == kSingle) {
    return launch_append<DH, BLOCK, FORM, false>(a, stream);
  } else {
    const bool many = !a.rot.R || (long long)a.c.B * a.L * (2 * a.c.Hk + a.H) >= 1024ll * sm_count();
    return many ? launch_append<DH, BLOCK, FORM, true>(a, stream) : launch_append<DH, BLOCK, FORM, false>(a, stream);
  }
}
template <int DH, int BLOCK>
static int launch_append(const AppendArgs& a, void* stream) {
  const Form form = form_of(a);
  return form == kSingle    ? launch_append<DH, BLOCK, kSingle>(a, stream)
         : form == kVectors ? launch_append<DH, BLOCK, kVectors>(a, stream)
                            : launch_append<DH, BLOCK, kTogether>(a, stream);
}
template <int DH>
static int launch_append(const AppendArgs& given, void* stream) {
  AppendArgs a = given;
  if (a.L == 1) {
    constexpr int rows = kThreads / (DH / 16);
    a.groups = (std::max(a.H, a.c.Hk) + rows - 1) / rows;
    const long long grid = (long long)a.c.B * a.groups;
    if (grid > 0x7fffffffll) return fail(FSVD_ERR_UNSUPPORTED, "too many heads for one call");
    const Form form = form_of(a);
    return form == kSingle    ? launch<append_step_kernel<DH, kSingle>>(dim3((unsigned)grid), kThreads, 0, stream, a)
           : form == kVectors ? launch<append_step_kernel<DH, kVectors>>(dim3((unsigned)grid), kThreads, 0, stream, a)
                              : launch<append_step_kernel<DH, kTogether>>(dim3((unsigned)grid), kThreads, 0, stream, a);
  }
  switch (a.c.block) {
    case 16: return launch_append<DH, 16>(a, stream);
    case 32: return launch_append<DH, 32>(a, stream);
    case 64: return launch_append<DH, 64>(a, stream);
    default: return launch_append<DH, 128>(a, stream);
  }
}

}  // namespace fsvd_kv8_impl

using namespace fsvd_kv8_impl;

extern "C" {

int fsvd_rope_qk(const void* q, long long q_stride, const void* k, long long k_stride, const int* positions,
                 const double* inv_freq, int rotary_dim, int interleaved, double rope_scale, void* q_out, void* k_out, int T,
                 int H, int Hk, int Dh, int dtype, void* stream) {
  if (!q || !positions || !inv_freq || !q_out || (k != nullptr) != (k_out != nullptr)) return fail(FSVD_ERR_ARG, "null argument");
  if (dtype != FSVD_DTYPE_BF16 && dtype != FSVD_DTYPE_F32) return fail(FSVD_ERR_ARG, "bad dtype %d", dtype);
  if (T < 0 || H < 1 || (k && Hk < 1)) return fail(FSVD_ERR_ARG, "bad sizes T=%d H=%d Hk=%d", T, H, Hk);
  if (H > kMaxHeads || Hk > kMaxHeads) return fail(FSVD_ERR_UNSUPPORTED, "more than %d heads", kMaxHeads);
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
  a.on32 = aligned32(q) && aligned32(k) && aligned32(q_out) && aligned32(k_out) && q_stride * es % 32 == 0 && k_stride * es % 32 == 0;
  return launch_rope(a, dtype, stream);
}

size_t fsvd_kv8_workspace_bytes(int B, int H, int Hk, int Dh, int S_max) {
  if (B < 1 || H < 1 || Hk < 1 || (Dh != 64 && Dh != 128) || S_max < 1) return 0;
  return ws_layout(H, Hk, Dh).total;
}

int fsvd_kv8_append(const fsvd_kv8* cache, const void* k, const void* v, long long kv_batch_stride, long long kv_token_stride,
                    const int* cache_seqlens, const int* new_lens, const void* q, long long q_batch_stride,
                    long long q_token_stride, void* q_out, const double* inv_freq, int rotary_dim, int interleaved,
                    double rope_scale, int H, int L, void* ws, size_t ws_bytes, void* stream) {
  if (int e = check_cache(cache)) return e;
  if (!k || !v || !cache_seqlens || (q != nullptr) != (q_out != nullptr)) return fail(FSVD_ERR_ARG, "null argument");
  if (q && !inv_freq) return fail(FSVD_ERR_ARG, "queries are passed to be rotated: inv_freq is missing");
  if (int e = check_rotary(inv_freq, rotary_dim, cache->Dh)) return e;
  if (L < 0 || (q && H < 1)) return fail(FSVD_ERR_ARG, "bad sizes L=%d H=%d", L, H);
  if (q && H > kMaxHeads) return fail(FSVD_ERR_UNSUPPORTED, "more than %d heads", kMaxHeads);
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
  a.on32 = aligned32(k) && aligned32(v) && aligned32(q) && aligned32(q_out) && kv_batch_stride % 16 == 0 && kv_token_stride % 16 == 0 &&
           q_batch_stride % 16 == 0 && q_token_stride % 16 == 0;
  const int BLOCK = cache->block;
  a.nblk = (int)(((long long)L + BLOCK - 2) / BLOCK + 1);
  if ((long long)cache->B * L > 0x7fffffffll) return fail(FSVD_ERR_UNSUPPORTED, "too many tokens for one call");
  return cache->Dh == 64 ? launch_append<64>(a, stream) : launch_append<128>(a, stream);
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
                reinterpret_cast<__nv_bfloat16*>(v_out), aligned32(k_out) && aligned32(v_out)};
  const long long pieces = (long long)length * (cache->Dh / 16);
  const long long grid = (2ll * cache->B * cache->Hk * pieces + kThreads - 1) / kThreads;
  if (grid > 0x7fffffffll || pieces > 0x7fffffffll) return fail(FSVD_ERR_UNSUPPORTED, "too many tokens for one call");
  return cache->Dh == 64 ? launch<load_kernel<64>>(dim3((unsigned)grid), kThreads, 0, stream, a)
                         : launch<load_kernel<128>>(dim3((unsigned)grid), kThreads, 0, stream, a);
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
  const Kv8Ws L = ws_layout(H, cache->Hk, cache->Dh);
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

// Rotary positions: the arithmetic that fsvd_rope_qk and fsvd_kv8_append share.
//
// A head of Dh dimensions is Dh / 2 pairs: pair p < R / 2 turns by position * inv_freq[p] and is made of dimensions
// (p, p + R / 2), or (2 p, 2 p + 1) when interleaved; the pairs behind them, (R + 2 j, R + 2 j + 1), stay.  A thread
// owns a unit of eight consecutive pairs of a row: it reads all 16 numbers before it writes any, so that a row can be
// rotated in place.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

namespace fsvd_rope {

// How a thread reads its unit: sixteen numbers one by one (R no multiple of 16), two vectors of eight, or one of sixteen
// (bf16; interleaved, or no rotation; rows on boundaries of 32 bytes).
enum Form { kSingle, kVectors, kTogether };

struct Rotary {
  const double* inv_freq;   // [R / 2], radians per position
  int R, interleaved;
  double scale;
};

// Sine and cosine of position * f, f in radians per position.  The angle is formed and reduced in 64 bits: in 32, a
// position of 10^5 leaves the fastest pair 0.004 radians off.
__device__ __forceinline__ void angle(double position, double f, double scale, double& c, double& s) {
  const double turns = position * (f * 0.15915494309189533577);   // 1 / (2 pi)
  sincospi(2.0 * (turns - rint(turns)), &s, &c);
  c *= scale;
  s *= scale;
}

// Offsets of the two numbers of pair p within the row.
__device__ __forceinline__ int2 pair_at(int p, int R, int interleaved) {
  const int half = R >> 1;
  if (p >= half || interleaved) return make_int2(2 * p, 2 * p + 1);   // (behind the rotated part: R + 2 (p - R / 2))
  return make_int2(p, p + half);
}

__device__ __forceinline__ void widen(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) { widen(*reinterpret_cast<const uint4*>(p), f); }
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ float num(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float num(float x) { return x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }

// 32 bytes on a boundary of 32.  Where a thread's share of a row lies together, two accesses of 16 bytes would each touch every
// other half of the warp's sectors.
__device__ __forceinline__ void load32(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// The eight pairs of unit u as (a[i], b[i]).
template <Form FORM, typename T>
__device__ __forceinline__ void load_unit(const T* row, int u, int R, int interleaved, float (&a)[8], float (&b)[8]) {
  if constexpr (FORM != kSingle) {
    const bool split = !interleaved && 16 * u < R;   // (16 u = twice the first pair)
    if constexpr (FORM == kTogether) {
      uint32_t w[8];
      load32(row + 16 * u, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] = __uint_as_float(w[i] << 16);
        b[i] = __uint_as_float(w[i] & 0xffff0000u);
      }
      return;
    }
    float x[8], y[8];
    load8(row + (split ? 8 * u : 16 * u), x);
    load8(row + (split ? 8 * u + (R >> 1) : 16 * u + 8), y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float lo = i < 4 ? x[(2 * i) & 7] : y[(2 * i) & 7], hi = i < 4 ? x[(2 * i + 1) & 7] : y[(2 * i + 1) & 7];
      a[i] = split ? x[i] : lo;
      b[i] = split ? y[i] : hi;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int2 at = pair_at(8 * u + i, R, interleaved);
      a[i] = num(row[at.x]);
      b[i] = num(row[at.y]);
    }
  }
}
template <Form FORM, typename T>
__device__ __forceinline__ void store_unit(T* row, int u, int R, int interleaved, const float (&a)[8], const float (&b)[8]) {
  if constexpr (FORM != kSingle) {
    const bool split = !interleaved && 16 * u < R;
    if constexpr (FORM == kTogether) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = pack2(a[i], b[i]);
      store32(row + 16 * u, w);
      return;
    }
    float x[8], y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float lo = (i & 1) ? b[i >> 1] : a[i >> 1], hi = (i & 1) ? b[4 + (i >> 1)] : a[4 + (i >> 1)];
      x[i] = split ? a[i] : lo;
      y[i] = split ? b[i] : hi;
    }
    store8(row + (split ? 8 * u : 16 * u), x);
    store8(row + (split ? 8 * u + (R >> 1) : 16 * u + 8), y);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int2 at = pair_at(8 * u + i, R, interleaved);
      put(row + at.x, a[i]);
      put(row + at.y, b[i]);
    }
  }
}

// The same for bf16 rows as packed pairs: a in the low half of a word, b in the high one.
template <Form FORM>
__device__ __forceinline__ void load_pairs(const __nv_bfloat16* row, int u, int R, int interleaved, uint32_t (&w)[8]) {
  if constexpr (FORM != kSingle) {
    const bool split = !interleaved && 16 * u < R;
    if constexpr (FORM == kTogether) {
      load32(row + 16 * u, w);
      return;
    }
    const uint4 x = *reinterpret_cast<const uint4*>(row + (split ? 8 * u : 16 * u));
    const uint4 y = *reinterpret_cast<const uint4*>(row + (split ? 8 * u + (R >> 1) : 16 * u + 8));
    const uint32_t p[4] = {x.x, x.y, x.z, x.w}, q[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[2 * i] = split ? __byte_perm(p[i], q[i], 0x5410) : i < 2 ? p[2 * i] : q[2 * i - 4];
      w[2 * i + 1] = split ? __byte_perm(p[i], q[i], 0x7632) : i < 2 ? p[2 * i + 1] : q[2 * i - 3];
    }
  } else {
    const uint16_t* r = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int2 at = pair_at(8 * u + i, R, interleaved);
      w[i] = (uint32_t)r[at.x] | ((uint32_t)r[at.y] << 16);
    }
  }
}
template <Form FORM>
__device__ __forceinline__ void store_pairs(__nv_bfloat16* row, int u, int R, int interleaved, const uint32_t (&w)[8]) {
  if constexpr (FORM != kSingle) {
    const bool split = !interleaved && 16 * u < R;
    if constexpr (FORM == kTogether) {
      store32(row + 16 * u, w);
      return;
    }
    uint32_t p[4], q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = split ? __byte_perm(w[2 * i], w[2 * i + 1], 0x5410) : w[i];
      q[i] = split ? __byte_perm(w[2 * i], w[2 * i + 1], 0x7632) : w[4 + i];
    }
    *reinterpret_cast<uint4*>(row + (split ? 8 * u : 16 * u)) = make_uint4(p[0], p[1], p[2], p[3]);
    *reinterpret_cast<uint4*>(row + (split ? 8 * u + (R >> 1) : 16 * u + 8)) = make_uint4(q[0], q[1], q[2], q[3]);
  } else {
    uint16_t* r = reinterpret_cast<uint16_t*>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int2 at = pair_at(8 * u + i, R, interleaved);
      r[at.x] = (uint16_t)(w[i] & 0xffffu);
      r[at.y] = (uint16_t)(w[i] >> 16);
    }
  }
}

}  // namespace fsvd_rope

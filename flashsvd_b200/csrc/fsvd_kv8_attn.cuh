// Single-query attention over the 8-bit cache on the tensor cores, without widening a code.
//
//   s_t = scale ks(t) q . k8_t,   out = sum_t softmax(s)_t vs(t) v8_t
//
// tcgen05.mma kind::f8f6f4 multiplies e4m3 by e4m3 exactly and adds in 32 bits, so the codes go from TMA to the tensor
// core as they lie in memory.  What is not e4m3 is written as a sum of e4m3 numbers and takes a column of the small
// operand each: a query row is q0 + q1 / 16 + q2 / 256 (a bf16 number has 8 bits, an e4m3 number 4: nothing is lost of the
// numbers above 2^-17 of the row's largest, less than 2^-25 of it below), a weight is eight digits of base 16, which keep all 24 bits of an fp32 number down to 2^-16 and reach
// to 2^-39 of the largest (`digits_of`).  A tile is 128 tokens: S^T [128 tokens, 4 G] = K8 . q^T, then
// O^T [Dh, 8 G] = V8^T . w^T, where V8^T is the tile as it lies, read along its other axis.  Scales are applied to the
// scores in 32 bits: the exponent of a weight is s log2(e) + log2(vs), so that the weight carries its value's scale, and the
// denominator divides it out.  (A token whose scale is 2^kSpan below the largest has its weight formed with a larger one, so
// that it does not leave the 32-bit range, and multiplied down for the product.)  Maxima are whole numbers: a change of them
// rounds nothing.
//
// A thread of the four softmax warps owns a token of S^T and a dimension of O^T; one more thread issues the copies, one
// the products.  O^T is read back after every tile and summed in registers, where a new maximum rescales it.  The
// maximum that weights refer to is one that was, and is renewed when a score passes it by more than the room that the
// digits are given (2^2): nearly every tile then needs one vote of the four warps instead of a maximum per head.
//
// The tiles of all (sequence, kv head) pairs form one list that is cut into equal parts, one per CTA, whatever the
// lengths are; a pair that more than one CTA works on is merged, in the order of its parts, by the CTA that finishes it.
#pragma once
#include <cuda.h>
#include <cuda_fp8.h>

#include "fsvd_tc.cuh"

namespace fsvd_kv8_attn {

using namespace fsvd_tile;

constexpr int kTile = 128;      // tokens
constexpr int kBox = 32;        // tokens of a TMA box: a short last tile is fetched in as many as it needs
constexpr int kSoft = 128;      // threads of a softmax group
constexpr int kDigits = 8;      // e4m3 numbers of a weight
constexpr int kParts = 4;       // columns of a query: three e4m3 numbers, and one that nobody reads
constexpr int kMaxGroup = 16;
constexpr int kPad = 4;         // floats behind a head's partial sums
constexpr int kRoom = 2;        // log2 of how far a weight may pass the largest one when the maximum was renewed
constexpr float kSpan = 60.0f, kSlack = 30.0f;   // binades below the largest value's scale when it was renewed, and above it
constexpr float kUnit = 1.0f / (1 << (7 - kRoom));   // of the sums that the digits give (`digits_of`)

struct Args {
  const float *k_scale, *v_scale;
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const int* seqlens;
  float* part;       // [CTAs][2][G][Dh + kPad]: partial sums, maximum, denominator
  int* counters;     // [CTAs], zero between launches: of the pair that begins in a CTA and goes on in the next one
  int* status;
  long long wait_limit;
  int B, Hk, S_max, block_log2, nb, G, seqlen_add;
  float scale;
};

template <int DH, int GP>
struct Shape {
  // Heads are shared out to groups of four softmax warps, four heads each: with 8 heads in one group (and weights of four
  // numbers) a tile took 1.4 times as long as its bytes.
  static constexpr int kGroups = GP > 4 ? GP / 4 : 1, kHeads = GP / kGroups;
  static constexpr int kThreads = kSoft * kGroups + 64;
  // CTAs of an SM, and tiles that a CTA has under way.  32 sequences x 32 heads of 128 x 2048 tokens: two CTAs of three tiles
  // 84 us, three of two 94; heads of 64, 128 ragged sequences: three CTAs of four tiles 44 us, two of six 50.
  static constexpr int kCtas = GP > 8 ? 1 : DH == 64 && GP <= 4 ? 3 : 2;
  static constexpr int kStages = GP > 8 ? 5 * (128 / DH) : DH == 128 ? 3 : GP <= 4 ? 4 : 6;
  static constexpr int kNq = kParts * GP < 16 ? 16 : kParts * GP;       // columns of S
  static constexpr int kNw = kDigits * GP < 16 ? 16 : kDigits * GP;     // columns of O
  static constexpr int kUsed = 2 * (kNq + kNw), kCols = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
  static_assert(kCols * kCtas <= 512, "tensor memory of an SM");
  static constexpr int kHalf = kTile * DH;                              // bytes of a K or V tile
  static constexpr int kQ = kNq * DH < 1024 ? 1024 : kNq * DH, kW = kNw * kTile;
  // The weights take the place of the tile's keys, which nobody reads once there are scores.
  static constexpr bool kOver = kW <= kHalf;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * 2 * kHalf + 2 * kQ + (kOver ? 0 : 2 * kW);
};

__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// e4m3 x e4m3 -> fp32, M = 128, N columns; both operands along their rows (K-major) or along their columns (transposed)
__device__ __forceinline__ uint32_t idesc_f8(int N, bool transposed) {
  return (1u << 4) | ((transposed ? 3u : 0u) << 15) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
// Operand of rows of ROW bytes (64 or 128) under the swizzle of that span; eight rows are 8 ROW bytes.  The stride
// between spans is zero: a transposed operand of 64 rows repeats them as rows 64..127 (which nobody reads).
template <int ROW>
__device__ __forceinline__ uint64_t desc_f8(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)(8 * ROW >> 4) << 32) | (1ull << 46) | ((ROW == 128 ? 2ull : 4ull) << 61);
}
// The weights: 128 rows (tokens) of N bytes (columns), read along the columns; rows of 32, 64 and 128 bytes under the
// swizzle of that span.
template <int N>
__device__ __forceinline__ uint64_t desc_weights(uint32_t addr) {
  const uint64_t at = (uint64_t)((addr >> 4) & 0x3fffu) | (1ull << 46);
  return N == 16 ? at | (8ull << 16) | (8ull << 32)
                 : at | ((uint64_t)(8 * N >> 4) << 32) | ((N == 32 ? 6ull : N == 64 ? 4ull : 2ull) << 61);
}
// Where 16-byte piece c of row r of them lies.
template <int N>
__device__ __forceinline__ uint32_t weights_at(int r, int c) {
  const int x = N == 32 ? (r >> 2) & 1 : N == 64 ? (r >> 1) & 3 : N == 128 ? r & 7 : 0;
  return (uint32_t)(r * N + ((c ^ x) << 4));
}
// byte c of row r of such an operand
template <int ROW>
__device__ __forceinline__ uint32_t swizzled(int r, int c) {
  const int x = ROW == 128 ? (r & 7) : ((r >> 1) & 3);
  return (uint32_t)(r * ROW + (((c >> 4) ^ x) << 4) + (c & 15));
}
__device__ __forceinline__ void tma_box_3d(uint32_t dst, const void* tmap, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Barriers: of the threads of one softmax group (its number), of all softmax threads.
__device__ __forceinline__ void group_sync(int group) { asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory"); }
__device__ __forceinline__ void soft_sync(int threads) { asm volatile("bar.sync 8, %0;" ::"r"(threads) : "memory"); }
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}

// N consecutive columns of this thread's lane.
template <int N>
__device__ __forceinline__ void tm_ld(uint32_t taddr, float* v);
template <>
__device__ __forceinline__ void tm_ld<2>(uint32_t taddr, float* v) {
  uint32_t r[2];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1])
               : "r"(taddr) : "memory");
#pragma unroll
  for (int i = 0; i < 2; ++i) v[i] = __uint_as_float(r[i]);
}
template <>
__device__ __forceinline__ void tm_ld<4>(uint32_t taddr, float* v) {
  uint32_t r[4];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr) : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
}
template <>
__device__ __forceinline__ void tm_ld<8>(uint32_t taddr, float* v) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr) : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
template <>
__device__ __forceinline__ void tm_ld<16>(uint32_t taddr, float* v) {
  uint32_t r[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr) : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
template <>
__device__ __forceinline__ void tm_ld<32>(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(taddr) : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
template <>
__device__ __forceinline__ void tm_ld<64>(uint32_t taddr, float* v) {
  tm_ld<32>(taddr, v);
  tm_ld<32>(taddr + 32, v + 32);
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// x 2^-up, for a whole `up` whose power alone may leave the 32-bit range
__device__ __forceinline__ float lowered(float x, float up) {
  const float half = truncf(0.5f * up);
  return x * ex2(-half) * ex2(half - up);
}
// Whether any thread of a softmax group says so.
__device__ __forceinline__ bool group_any(bool x, int group) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)x), "r"(group + 1)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ uint32_t prmt(uint32_t x, uint32_t y, uint32_t selector) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(y), "r"(selector));
  return r;
}
// A weight 0 <= u < 2^(kRoom + 1) as eight e4m3 numbers d_i 2^s, d_i the digits 0..15 of a 32-bit whole number W with
// W 2^s = u 2^(35 - kRoom): sum over i of 16^(i - 7) d_i 2^s = u / kUnit.  All of d 2^s with s = -6..4 are e4m3 numbers, so s
// follows the weight for ten binades, in which W is the significand with eight zeros behind it; below them s stays and W
// loses a bit per binade: nothing of the 24 down to 2^(kRoom - 18), less than 2^(kRoom - 41) in all.  A CTA goes through
// about 2^23 tokens at most (the card's memory in equal parts): what is cut off stays below 2^-15 of the largest value.
// Digits become codes by a table in registers: a selector of 0..7 takes a byte, one with the upper bit set takes the
// byte's sign, which is zero; the upper half of the table is asked for the digits with that bit turned.
__device__ __forceinline__ void digits_of(float u, uint32_t& low, uint32_t& high) {
  const uint32_t bits = __float_as_uint(u);
  const int up = (int)(bits >> 23) - (127 + kRoom - 10);
  const uint32_t w = __funnelshift_rc((bits << 8) | 0x80000000u, 0u, (uint32_t)max(-up, 0)), v = w ^ 0x88888888u;
  const uint32_t more = (uint32_t)max(up, 0) * 0x08080808u;   // 2^s = 2^-6 2^up; a zero stays one
  const uint32_t t0 = 0x14100800u + (more & 0xffffff00u), t1 = 0x1e1c1a18u + more, t2 = 0x23222120u + more, t3 = 0x27262524u + more;
  low = prmt(t0, t1, w) | prmt(t2, t3, v);
  high = prmt(t0, t1, w >> 16) | prmt(t2, t3, v >> 16);
}
// Two fp32 numbers -> their nearest e4m3 codes (x in the low byte), and what the codes stand for.
__device__ __forceinline__ uint32_t to_codes(float x, float y, float& dx, float& dy) {
  const uint32_t c = __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)c, __NV_E4M3);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  dx = f.x;
  dy = f.y;
  return c;
}

// The part of the list of tiles that a CTA works on, as runs of tiles of one (sequence, kv head).
struct Cursor {
  const int* seqlens;
  int add, S_max, Hk, B;
  int b, hk, tiles, n;       // sequence, kv head, the sequence's tiles and positions
  int tile, left;            // next tile, tiles left for this CTA
  __device__ __forceinline__ int positions(int i) const {
    return (int)min(max((long long)seqlens[i] + add, 0ll), (long long)S_max);
  }
  __device__ __forceinline__ void enter() {
    n = positions(b);
    tiles = (n + kTile - 1) / kTile;
  }
  // tiles of the current run
  __device__ __forceinline__ int run() const { return min(left, tiles - tile); }
  __device__ __forceinline__ void next(int done) {
    left -= done;
    tile += done;
    if (tile == tiles && left > 0) {
      tile = 0;
      if (++hk == Hk) {
        hk = 0;
        do {
          ++b;
          enter();
        } while (tiles == 0);
      }
    }
  }
};

template <int DH, int GP>
__global__ void __launch_bounds__(Shape<DH, GP>::kThreads, Shape<DH, GP>::kCtas) attn_kernel(const __grid_constant__ CUtensorMap kmap,
                                                                             const __grid_constant__ CUtensorMap vmap,
                                                                             const Args a) {
  using S = Shape<DH, GP>;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) unsigned long long kv_full[S::kStages], kv_empty[S::kStages], s_full[2], w_full[2], o_full[2], q_full[2];
  __shared__ uint32_t tmem_slot;
  __shared__ float qfac[2][GP], red2[2][4][GP], wtop[2][S::kGroups][4];
  __shared__ float2 wmax[2][4][GP];
  __shared__ int start_b, start_hk, start_tile, start_n, last_sh, giveup_sh;
  __shared__ int per_sh, total_sh, base_sh;
  struct Part { int bh, tiles, list; };   // of a pair: which, its tiles, where they begin in the list
  __shared__ Part part_of[2];
  constexpr int NG = S::kGroups, GH = S::kHeads, kCopy = 4 * NG, kMma = kCopy + 1;   // (warps)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = a.G;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* qs = smem + S::kStages * 2 * S::kHalf;
  auto weights = [&](int j) {   // of tile j
    return S::kOver ? smem + (j % S::kStages) * 2 * S::kHalf : qs + 2 * S::kQ + (j & 1) * S::kW;
  };
  volatile int* giveup = &giveup_sh;

  if (tid == 0) {
    giveup_sh = 0;
    part_of[0].tiles = part_of[1].tiles = 0;
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(smem_u32(&kv_full[i]), 1);
      mbar_init(smem_u32(&kv_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&w_full[i]), kSoft * NG);
      mbar_init(smem_u32(&o_full[i]), 1);
      mbar_init(smem_u32(&q_full[i]), kSoft * NG);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kCopy && lane < 2)
    asm volatile("prefetch.tensormap [%0];" ::"l"(lane ? reinterpret_cast<uint64_t>(&vmap) : reinterpret_cast<uint64_t>(&kmap)) : "memory");
  if (warp == kMma) tc_alloc(smem_u32(&tmem_slot), S::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();   // (the kernel behind this one must not take the tensor memory first)
  pdl_wait();

  // where this CTA's part of the list begins: every sequence has Hk * tiles entries
  Cursor cur;
  cur.seqlens = a.seqlens; cur.add = a.seqlen_add; cur.S_max = a.S_max; cur.Hk = a.Hk; cur.B = a.B;
  if (warp == 0) {
    auto entries = [&](int i, int& n, int& t) -> int {   // of sequence i
      n = i < a.B ? cur.positions(i) : 0;
      t = (n + kTile - 1) / kTile;
      return t * a.Hk;   // (a list of 2^31 tiles would stand for more memory than there is)
    };
    auto prefix = [&](int x) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      return x;
    };
    int n, t;
    const int x0 = entries(lane, n, t), inc0 = prefix(x0);   // the first 32 sequences, often all
    int total = __shfl_sync(0xffffffffu, inc0, 31);
    for (int b0 = 32; b0 < a.B; b0 += 32) {
      int n1, t1;
      total += __reduce_add_sync(0xffffffffu, entries(b0 + lane, n1, t1));
    }
    const int grid = gridDim.x, per = (total + grid - 1) / grid, w0 = per * blockIdx.x;
    int before = 0, x = x0, inc = inc0;
    for (int b0 = 0; w0 < total;) {
      const bool mine = w0 >= before + inc - x && w0 < before + inc;
      if (mine) {
        const int off = w0 - (before + inc - x);
        start_b = b0 + lane;
        start_hk = off / t;
        start_tile = off - off / t * t;
        start_n = n;
        base_sh = before + inc - x;   // list index of the sequence's first tile
      }
      b0 += 32;
      if (__any_sync(0xffffffffu, mine) || b0 >= a.B) break;
      before += __shfl_sync(0xffffffffu, inc, 31);
      x = entries(b0 + lane, n, t);
      inc = prefix(x);
    }
    if (lane == 0) {
      total_sh = total;
      per_sh = per;
    }
  }
  __syncthreads();
  const uint32_t tmem = tmem_slot;
  const int per = per_sh;
  cur.left = max(0, min(per, total_sh - per * (int)blockIdx.x));
  if (cur.left > 0) {
    cur.b = start_b; cur.hk = start_hk; cur.tile = start_tile; cur.n = start_n;
    cur.tiles = (cur.n + kTile - 1) / kTile;
  }

  if (warp == kCopy) {   // ---- copies
    if (lane == 0 && cur.left > 0) {
      int j = 0;
      while (cur.left > 0) {
        const int run = cur.run(), plane = cur.b * a.Hk + cur.hk;
        for (int t = cur.tile; t < cur.tile + run; ++t, ++j) {
          const int st = j % S::kStages;
          if (j >= S::kStages) wait_bar(smem_u32(&kv_empty[st]), (j / S::kStages - 1) & 1, giveup, a.status, a.wait_limit, DS_COPY_TIMEOUT);
          if (*giveup) break;
          const int boxes = min(kTile, cur.n - t * kTile + kBox - 1) / kBox;
          const uint32_t dst = smem_u32(smem + st * 2 * S::kHalf), bar = smem_u32(&kv_full[st]);
          mbar_expect_tx(bar, (uint32_t)boxes * 2 * kBox * DH);
          for (int i = 0; i < boxes; ++i) tma_box_3d(dst + i * kBox * DH, &kmap, 0, t * kTile + i * kBox, plane, bar);
          for (int i = 0; i < boxes; ++i) tma_box_3d(dst + S::kHalf + i * kBox * DH, &vmap, 0, t * kTile + i * kBox, plane, bar);
        }
        if (*giveup) break;
        cur.next(run);
      }
      // nothing may be on its way to this CTA's shared memory when it ends: the releases of the last stages, and
      // after a wait that ran out the copies into them
      for (int i = max(0, j - S::kStages); i < j; ++i) {
        const uint32_t full = smem_u32(&kv_full[i % S::kStages]);
        const long long c0 = clock64();
        while (!mbar_try_wait(full, (i / S::kStages) & 1) && clock64() - c0 < a.wait_limit) {
        }
        wait_bar(smem_u32(&kv_empty[i % S::kStages]), (i / S::kStages) & 1, giveup, a.status, a.wait_limit, DS_COPY_TIMEOUT);
      }
    }
  } else if (warp == kMma) {   // ---- products
    if (lane == 0 && cur.left > 0) {
      const uint32_t iq = idesc_f8(S::kNq, false), iw = idesc_f8(S::kNw, true);
      const int n = cur.left;
      int seg = 0, in_run = cur.run();
      auto weigh = [&](int j) {   // O(j) = V8^T . w^T
        const int st = j % S::kStages, buf = j & 1;
        wait_bar(smem_u32(&w_full[buf]), (j >> 1) & 1, giveup, a.status, a.wait_limit, DS_BARRIER_TIMEOUT);
        tc_fence_after();
        const uint32_t v = smem_u32(smem + st * 2 * S::kHalf + S::kHalf), w = smem_u32(weights(j));
#pragma unroll
        for (int k = 0; k < kTile / 32; ++k)
          mma_f8(tmem + 2 * S::kNq + buf * S::kNw, desc_f8<DH>(v + 32 * DH * k), desc_weights<S::kNw>(w + 32 * S::kNw * k), iw, k > 0);
        tc_commit(smem_u32(&o_full[buf]));
        tc_commit(smem_u32(&kv_empty[st]));
      };
      for (int j = 0; j < n; ++j) {
        if (in_run == 0) {
          ++seg;
          cur.next(cur.run());
          in_run = cur.run();
        }
        --in_run;
        const int st = j % S::kStages, buf = j & 1;
        wait_bar(smem_u32(&q_full[seg & 1]), (seg >> 1) & 1, giveup, a.status, a.wait_limit, DS_BARRIER_TIMEOUT);
        wait_bar(smem_u32(&kv_full[st]), (j / S::kStages) & 1, giveup, a.status, a.wait_limit, DS_COPY_TIMEOUT);
        if (*giveup) break;
        tc_fence_after();
        const uint32_t k8 = smem_u32(smem + st * 2 * S::kHalf), q8 = smem_u32(qs + (seg & 1) * S::kQ);
#pragma unroll
        for (int k = 0; k < DH / 32; ++k) mma_f8(tmem + buf * S::kNq, desc_f8<DH>(k8 + 32 * k), desc_f8<DH>(q8 + 32 * k), iq, k > 0);
        tc_commit(smem_u32(&s_full[buf]));
        if (j > 0) weigh(j - 1);
      }
      if (!*giveup) weigh(n - 1);
    }
  } else {   // ---- softmax
    // The query rows of a pair as q0 + q1 / 16 + q2 / 256, scaled to a largest magnitude in [128, 256): fetched while the pair before is
    // begun, written when its first tile is through.
    const int group = warp >> 2, tl = tid & (kSoft - 1), wl = warp & 3;   // thread and warp within the group
    const int head0 = group * GH;                                          // its heads
    constexpr int D = DH / 32;   // numbers of a lane; a warp takes a row
    static_assert(GP <= 4 * NG);
    uint32_t rows[D / 2];
    auto fetch_q = [&](int b, int hk) {
      if (warp < G) {
        const __nv_bfloat16* row = a.q + (((size_t)b * a.Hk + hk) * G + warp) * DH + lane * D;
        if constexpr (D == 4) {
          const uint2 w = *reinterpret_cast<const uint2*>(row);
          rows[0] = w.x;
          rows[D / 2 - 1] = w.y;
        } else {
          rows[0] = *reinterpret_cast<const uint32_t*>(row);
        }
      }
    };
    auto build_q = [&](int which) {
      if (warp < G) {
        const int g = warp;
        uint8_t* dst = qs + which * S::kQ;
        float x[D], top = 0.0f;
        bool fine = true;
#pragma unroll
        for (int e = 0; e < D; ++e) {
          x[e] = __uint_as_float((e & 1) ? rows[e / 2] & 0xffff0000u : rows[e / 2] << 16);
          top = fmaxf(top, fabsf(x[e]));
          fine = fine && isfinite(x[e]);
        }
        top = warp_max(top);
        fine = __all_sync(0xffffffffu, fine);
        const int e2 = (int)(__float_as_uint(top) >> 23) - 127;          // top in [2^e2, 2^(e2 + 1))
        const int up = fine ? min(max(7 - e2, -120), 120) : 0;
        const float f = __uint_as_float((uint32_t)(up + 127) << 23);
        uint32_t c[3] = {0, 0, 0};
#pragma unroll
        for (int e = 0; e < D; e += 2) {
          float x0 = x[e] * f, x1 = x[e + 1] * f;
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            float d0, d1;
            c[i] |= to_codes(x0, x1, d0, d1) << (8 * e);
            x0 = (x0 - d0) * 16.0f;
            x1 = (x1 - d1) * 16.0f;
          }
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          if (!fine) c[i] = 0x7f7f7f7fu;   // a query that is not finite gives no number
          uint8_t* p = dst + swizzled<DH>(g / GH * kParts * GH + i * GH + g % GH, lane * D);
          if constexpr (D == 4) *reinterpret_cast<uint32_t*>(p) = c[i];
          else *reinterpret_cast<uint16_t*>(p) = (uint16_t)c[i];
        }
        if (lane == 0) qfac[which][g] = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - up) << 23);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(smem_u32(&q_full[which]));
    };
    const uint32_t lanes = (uint32_t)(wl * 32) << 16;
    const bool owns = tl < DH;   // a dimension of the result
    int seq_base = cur.left > 0 ? base_sh : 0;
    int j = 0, seg = 0;
    // The pair that is ending: its last product runs while the first tile of the next pair goes through the softmax.
    float acc[GH], l_end[GH], m_end[GH], c_end[GH];
    int bh_end = 0, run_end = 0, tiles_end = 0, seg_end = 0, list_end = 0;
    bool pending = false;
#pragma unroll
    for (int g = 0; g < GH; ++g) acc[g] = 0.0f;
    auto collect = [&](int jj, const float (&c)[GH]) {   // acc = acc c + O(jj)
      const int buf = jj & 1;
      wait_bar(smem_u32(&o_full[buf]), (jj >> 1) & 1, giveup, a.status, a.wait_limit, DS_BARRIER_TIMEOUT);
      tc_fence_after();
      if (wl * 32 < DH) {
        constexpr int N = GH < 2 ? GH : 2;   // heads at a time
#pragma unroll
        for (int g0 = 0; g0 < GH; g0 += N) {
          float o[kDigits * N];
          tm_ld<kDigits * N>(tmem + 2 * S::kNq + buf * S::kNw + (head0 + g0) * kDigits + lanes, o);
#pragma unroll
          for (int g = 0; g < N; ++g) {
            float sum = o[g * kDigits];
#pragma unroll
            for (int d = 1; d < kDigits; ++d) sum = fmaf(sum, 0.0625f, o[g * kDigits + d]);
            acc[g0 + g] = fmaf(acc[g0 + g], c[g0 + g], sum);
          }
        }
      }
    };
    auto finalise = [&](int last) {
      float (&red)[4][GP] = red2[seg_end & 1];
      collect(last, c_end);
      // denominators
#pragma unroll
      for (int g = 0; g < GH; ++g) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l_end[g] += __shfl_xor_sync(0xffffffffu, l_end[g], o);
        if (lane == 0) red[wl][head0 + g] = l_end[g];
      }
      group_sync(group);
#pragma unroll
      for (int g = 0; g < GH; ++g) l_end[g] = (red[0][head0 + g] + red[1][head0 + g]) + (red[2][head0 + g] + red[3][head0 + g]);
      __nv_bfloat16* out = a.out + ((size_t)bh_end * G + head0) * DH + tl;
      constexpr int rec = DH + kPad;
      if (run_end == tiles_end) {
        if (owns) {
#pragma unroll
          for (int g = 0; g < GH; ++g)
            if (head0 + g < G) out[g * DH] = __float2bfloat16_rn(acc[g] * kUnit / l_end[g]);
        }
      } else {
        float* rp = a.part + ((size_t)blockIdx.x * 2 + (seg_end > 0)) * G * rec + head0 * rec;
#pragma unroll
        for (int g = 0; g < GH; ++g)
          if (head0 + g < G) {
            if (owns) rp[g * rec + tl] = acc[g] * kUnit;
            if (tl == 0) *reinterpret_cast<float2*>(rp + g * rec + DH) = make_float2(m_end[g], l_end[g]);
          }
        if (tid == 0) part_of[seg_end > 0] = Part{bh_end, tiles_end, list_end};
      }
#pragma unroll
      for (int g = 0; g < GH; ++g) acc[g] = 0.0f;
    };
    if (cur.left > 0) {
      fetch_q(cur.b, cur.hk);
      build_q(0);
      soft_sync(kSoft * NG);
    }
    while (cur.left > 0) {
      const int run = cur.run(), first = cur.tile, bh = cur.b * a.Hk + cur.hk, n = cur.n, ntiles = cur.tiles, hk = cur.hk;
      cur.next(run);
      const bool more = cur.left > 0;   // (`cur` is the next pair from here on)
      if (more) fetch_q(cur.b, cur.hk);
      const int list0 = seq_base + hk * ntiles;   // list index of the pair's first tile
      const float* ksc = a.k_scale + (size_t)bh * a.nb;
      const float* vsc = a.v_scale + (size_t)bh * a.nb;
      float m[GH], l[GH], corr[GH], qf[GH];   // (acc: the sums divided by kUnit)
      float vmax = 0.0f, floor = -INFINITY;           // largest log2(vs), and the least that weights are formed with
#pragma unroll
      for (int g = 0; g < GH; ++g) m[g] = l[g] = qf[g] = 0.0f;
      float ks = 0.0f, vs = 1.0f;
      auto scales = [&](int t) {
        const int at = t * kTile + tl;
        ks = at < n ? ksc[at >> a.block_log2] : 0.0f;
        vs = at < n ? vsc[at >> a.block_log2] : 1.0f;
      };
      scales(first);
      for (int i = 0; i < run; ++i, ++j) {
        const int t = first + i, buf = j & 1;
        const bool valid = t * kTile + tl < n;
        const float kf = ks, lv = __log2f(vs);
        if (i + 1 < run) scales(t + 1);
        wait_bar(smem_u32(&s_full[buf]), (j >> 1) & 1, giveup, a.status, a.wait_limit, DS_BARRIER_TIMEOUT);
        tc_fence_after();
        if (i == 0) {   // (this product was issued when every warp had written its factors: before it nothing orders them)
#pragma unroll
          for (int g = 0; g < GH; ++g) qf[g] = qfac[seg & 1][head0 + g];
        }
        float s[kParts * GH], e[GH];
        tm_ld<kParts * GH>(tmem + buf * S::kNq + group * kParts * GH + lanes, s);
        float used = fmaxf(lv, floor);
        bool higher = i == 0 || (valid && lv > vmax + kSlack);
#pragma unroll
        for (int g = 0; g < GH; ++g) {
          s[g] = fmaf(fmaf(s[2 * GH + g], 0.0625f, s[GH + g]), 0.0625f, s[g]);
          e[g] = fmaf(s[g], kf * qf[g], used - m[g]);
          higher = higher || (valid && head0 + g < G && e[g] > (float)kRoom);
        }
        if (!valid && group == 0) {   // the last tile: a row behind the end may hold anything
          uint4* row = reinterpret_cast<uint4*>(smem + (j % S::kStages) * 2 * S::kHalf + S::kHalf + tl * DH);
#pragma unroll
          for (int x = 0; x < DH / 16; ++x) row[(x + tl) % (DH / 16)] = make_uint4(0u, 0u, 0u, 0u);   // (neighbours in other banks)
        }
        float prev[GH];   // rescaling of the tile before, which is collected below
#pragma unroll
        for (int g = 0; g < GH; ++g) {
          prev[g] = corr[g];
          corr[g] = 1.0f;
        }
        if (group_any(higher, group)) {
#pragma unroll
          for (int g = 0; g < GH; ++g) {
            const float top = warp_max(valid ? e[g] : -INFINITY), score = warp_max(valid ? e[g] - used : -INFINITY);
            if (lane == 0) wmax[buf][wl][head0 + g] = make_float2(top, score);
          }
          const float vtop = warp_max(valid ? lv : -INFINITY);
          if (lane == 0) wtop[buf][group][wl] = vtop;
          group_sync(group);
          const float v4 = fmaxf(fmaxf(wtop[buf][group][0], wtop[buf][group][1]), fmaxf(wtop[buf][group][2], wtop[buf][group][3]));
          vmax = i == 0 ? v4 : fmaxf(vmax, v4);
          floor = vmax - kSpan;
          used = fmaxf(lv, floor);
#pragma unroll
          for (int g = 0; g < GH; ++g) {
            float2 top = wmax[buf][0][head0 + g];
#pragma unroll
            for (int w = 1; w < 4; ++w) {
              const float2 y = wmax[buf][w][head0 + g];
              top.x = fmaxf(top.x, y.x);
              top.y = fmaxf(top.y, y.y);
            }
            // (the first tile's maximum may be below zero; where nothing is above -infinity there is nothing to refer to)
            const float most = ceilf(fmaxf(top.x, top.y + floor)), up = most > -INFINITY ? (i == 0 ? most : fmaxf(most, 0.0f)) : 0.0f;
            if (i > 0) {   // (before it there are no sums)
              corr[g] = ex2(-up);
              l[g] = lowered(l[g], up);
            }
            m[g] += up;
            e[g] = fmaf(s[g], kf * qf[g], used - m[g]);
          }
        }
        const float inv = valid ? ex2(-used) : 0.0f, down = ex2(lv - used);
#pragma unroll
        for (int g = 0; g < GH; ++g) {
          e[g] = valid ? ex2(e[g]) : 0.0f;   // at most 2^kRoom
          l[g] = fmaf(e[g], inv, l[g]);
          e[g] *= down;
        }
        {
          uint8_t* dst = weights(j);
          if constexpr (GH == 1) {
            uint2 c;
            digits_of(e[0], c.x, c.y);
            *reinterpret_cast<uint2*>(dst + tl * S::kNw) = c;
          } else {
#pragma unroll
            for (int g = 0; g < GH; g += 2) {   // two heads to a piece
              uint4 c;
              digits_of(e[g], c.x, c.y);
              digits_of(e[g + 1], c.z, c.w);
              *reinterpret_cast<uint4*>(dst + weights_at<S::kNw>(tl, (head0 + g) / 2)) = c;
            }
          }
        }
        tc_fence_before();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(smem_u32(&w_full[buf]));
        if (i == 0 && more) build_q((seg + 1) & 1);   // (the products of the pair before the last are done with that buffer)
        if (i > 0) {
          collect(j - 1, prev);
        } else if (pending) {
          finalise(j - 1);
          pending = false;
        }
      }
      if (hk == a.Hk - 1 && first + run == ntiles) seq_base += a.Hk * ntiles;
#pragma unroll
      for (int g = 0; g < GH; ++g) {
        l_end[g] = l[g];
        m_end[g] = m[g];
        c_end[g] = corr[g];
      }
      bh_end = bh; run_end = run; tiles_end = ntiles; seg_end = seg; list_end = list0;
      if (more) pending = true;
      else finalise(j - 1);
      ++seg;
    }
    // The pairs that this CTA has worked on a part of (its first and its last one): whoever finishes a pair merges its parts,
    // in their order.
    soft_sync(kSoft * NG);   // (the release below covers what the barrier orders in front of it)
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
      const Part pt = part_of[which];
      if (pt.tiles == 0) continue;
      constexpr int rec = DH + kPad;
      const int c0 = pt.list / per, c1 = (pt.list + pt.tiles - 1) / per;   // the CTAs of this pair
      if (tid == 0) {
        int arrived;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(arrived) : "l"(a.counters + c0) : "memory");
        last_sh = arrived == c1 - c0;
      }
      soft_sync(kSoft * NG);
      if (last_sh) {
        // CTA c's part is its first one if it starts inside the pair's tiles, else its last
        auto record = [&](int c) { return a.part + ((size_t)c * 2 + (per * c < pt.list)) * G * rec; };
        __nv_bfloat16* out = a.out + (size_t)pt.bh * G * DH;
        // Four dimensions to a thread, which goes through the parts eight at a time with a running maximum; where there are many
        // parts and fewer dimensions than threads, the parts are shared out too.
        constexpr int kBatch = 8;
        const int items = G * (DH / 4), shares = c1 - c0 >= kBatch ? max(1, kSoft / items) : 1;
        float4* sums = reinterpret_cast<float4*>(smem);   // (no tile is on its way any more; at most 128 of each)
        float2* tops = reinterpret_cast<float2*>(smem + kSoft * sizeof(float4));
        static_assert(S::kHalf >= kSoft * (int)(sizeof(float4) + sizeof(float2)));
        auto store = [&](int item, const float4& o, float den) {
          *reinterpret_cast<uint2*>(out + item / (DH / 4) * DH + item % (DH / 4) * 4) =
              make_uint2(pack_bf16(o.x / den, o.y / den), pack_bf16(o.z / den, o.w / den));
        };
        for (int x = tid; x < items * shares; x += kSoft * NG) {
          const int item = x % items, share = x / items, g = item / (DH / 4), d = item % (DH / 4) * 4;
          float top = -INFINITY, den = 0.0f;
          float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int cb = c0 + share; cb <= c1; cb += kBatch * shares) {
            float2 ml[kBatch];
            float4 v[kBatch];
#pragma unroll
            for (int c = 0; c < kBatch; ++c) {
              const float* r = record(min(cb + c * shares, c1)) + g * rec;
              ml[c] = __ldcg(reinterpret_cast<const float2*>(r + DH));
              v[c] = __ldcg(reinterpret_cast<const float4*>(r + d));
            }
            float mn = top;
#pragma unroll
            for (int c = 0; c < kBatch; ++c) mn = fmaxf(mn, cb + c * shares <= c1 ? ml[c].x : -INFINITY);
            const float gone = top > -INFINITY ? mn - top : 0.0f, f0 = ex2(-gone);
            top = mn;
            den = lowered(den, gone);
            o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
#pragma unroll
            for (int c = 0; c < kBatch; ++c)
              if (cb + c * shares <= c1) {
                const float f = ex2(ml[c].x - mn);
                den += lowered(ml[c].y, mn - ml[c].x);
                o.x = fmaf(f, v[c].x, o.x); o.y = fmaf(f, v[c].y, o.y); o.z = fmaf(f, v[c].z, o.z); o.w = fmaf(f, v[c].w, o.w);
              }
          }
          if (shares == 1) {
            store(item, o, den);
          } else {
            sums[x] = o;
            tops[x] = make_float2(top, den);
          }
        }
        if (shares > 1) {
          soft_sync(kSoft * NG);
          if (tid < items) {
            float top = tops[tid].x;
            for (int x = 1; x < shares; ++x) top = fmaxf(top, tops[tid + x * items].x);
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float den = 0.0f;
            for (int x = 0; x < shares; ++x) {
              const float2 ml = tops[tid + x * items];
              const float4 v = sums[tid + x * items];
              const float f = ex2(ml.x - top);
              den += ml.x > -INFINITY ? lowered(ml.y, top - ml.x) : ml.y;
              o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
            }
            store(tid, o, den);
          }
        }
        if (tid == 0) a.counters[c0] = 0;
      }
      soft_sync(kSoft * NG);
    }
    // sequences without positions
    for (int i = blockIdx.x; i < a.B; i += gridDim.x)
      if (cur.positions(i) == 0)
        for (int x = tid; x < a.Hk * G * DH / 8; x += kSoft * NG)
          reinterpret_cast<uint4*>(a.out + (size_t)i * a.Hk * G * DH)[x] = make_uint4(0u, 0u, 0u, 0u);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMma) tc_dealloc(tmem, S::kCols);
}

}  // namespace fsvd_kv8_attn

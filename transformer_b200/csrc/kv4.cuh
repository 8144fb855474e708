// kv4.cuh — kernels of the 4-bit paged KV cache (sm_100a): append with the
// rotary positions applied on the way, read-back, and attention.
//
// Format.  A position's row of one kv head is cut into groups of 16 dims.  A
// group's scale s is the smallest number >= amax / 7 with 5 exponent and 3
// mantissa bits (its byte b is the half with the bits b << 7), at most 9216;
// x is held as clamp(round-to-nearest-even(x / s), -7, 7), plus 8, in a
// nibble.  A held value is s (4 significant bits) times a whole number below
// 8: at most 7 significant bits, exact in bf16 and, with s <= 9216, in half.
//
// Page of 16 positions of one kv head, 18 d bytes, h < d / 64, g < 8, t < 4,
// p, q, e < 2, G < 4:
//   K codes  [h][g][t][e][8 B]        position 8e + g, dims 64h + 16t ..+15
//   K scales [h][g][t][e]             the same position and dims
//   V codes  [h][g][t][p][q][e][2 B]  position 8p + 2t + e, dims 64h + 8g + 4q ..+3
//   V scales [h][G][t][p][e]          position 8p + 2t + e, dims 64h + 16G ..+15
// so that lane 4g + t of a warp finds its A fragments of m16n8k16 (positions x
// dims for K, dims x positions for V) in 16 contiguous bytes per 64 dims.  The
// smallest store is the two bytes of four dims of one position: rows of one
// page can be appended by different threads without a read-modify-write.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <type_traits>

#include "b2d_ptx.cuh"
#include "kv4.h"

namespace b2d {

// ---- page addressing ---------------------------------------------------------
__device__ __forceinline__ int kv4_unit(int h, int g, int t) { return (h * 8 + g) * 4 + t; }
__device__ __forceinline__ int kv4_k_code(int grp, int r) {  // 8 bytes: 16 dims of slot r
  return kv4_unit(grp >> 2, r & 7, grp & 3) * 16 + (r >> 3) * 8;
}
__device__ __forceinline__ int kv4_k_scale(int d, int grp, int r) {
  return 8 * d + kv4_unit(grp >> 2, r & 7, grp & 3) * 2 + (r >> 3);
}
__device__ __forceinline__ int kv4_v_code(int d, int quad, int r) {  // 2 bytes: dims 4 quad .. of slot r
  const int h = quad >> 4, g = (quad >> 1) & 7, q = quad & 1;
  return 9 * d + ((kv4_unit(h, g, (r & 7) >> 1) * 2 + (r >> 3)) * 2 + q) * 4 + (r & 1) * 2;
}
__device__ __forceinline__ int kv4_v_scale(int d, int grp, int r) {
  return 17 * d + ((grp * 4 + ((r & 7) >> 1)) * 2 + (r >> 3)) * 2 + (r & 1);
}
__device__ __forceinline__ float kv4_scale_value(uint32_t byte) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(byte << 7)));
}
__device__ __forceinline__ void kv4_error(uint32_t* status, uint32_t code) {
  if (status != nullptr) atomicCAS(status, 0u, code);
}
constexpr uint32_t kKv4BadPos = 0x202u, kKv4BadTable = 0x203u, kKv4Timeout = 0x10Du;

// Whether the pool has the block that a table's entry names.
__device__ __forceinline__ bool kv4_named(const Kv4Cache& c, int blk) { return blk >= 0 && blk < c.num_blocks; }
// The page of position `pos` of the sequence with table row `sid`, or null
// (status set) when the table does not name one.
__device__ __forceinline__ uint8_t* kv4_page(const Kv4Cache& c, int sid, int pos, int g) {
  const int pg = pos / kKv4Page;
  if (sid < 0 || sid >= c.table_rows || pg >= c.bps) {
    kv4_error(c.status, kKv4BadTable);
    return nullptr;
  }
  const int blk = __ldg(c.table + sid * c.table_ld + pg);
  if (!kv4_named(c, blk)) {
    kv4_error(c.status, kKv4BadTable);
    return nullptr;
  }
  return c.pool + (static_cast<int64_t>(blk) * c.n_kv + g) * kv4_page_bytes(c.d);
}

// ---- element access ------------------------------------------------------------
template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

// 8 elements from / to p; vec: p is 16-byte aligned.
template <class T>
struct __align__(16) Eight {
  T v[8];
};
template <class T>
__device__ __forceinline__ Eight<T> load8(const T* p, bool vec) {
  Eight<T> x;
  if (vec) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4*>(x.v)[i] = reinterpret_cast<const uint4*>(p)[i];  // (not the read-only path: q may be q_out)
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = p[i];
  }
  return x;
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float* x, bool vec) {
  if (vec) {
    __align__(16) T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = from_f32<T>(x[i]);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_f32<T>(x[i]);
  }
}
// 8 values as four pairs of halves to p (all types hold them exactly).
template <class T>
__device__ __forceinline__ void put8(T* p, const uint32_t (&h)[4], bool vec) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
  store8(p, x, vec);
}
template <>
__device__ __forceinline__ void put8(__half* p, const uint32_t (&h)[4], bool vec) {
  if (vec) {
    *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __ushort_as_half(static_cast<unsigned short>(h[i >> 1] >> (16 * (i & 1))));
  }
}
__device__ __forceinline__ bool aligned16(const void* p, int64_t stride_a, int64_t stride_b, int size) {
  return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride_a * size) |
           static_cast<uintptr_t>(stride_b * size)) & 15u) == 0;
}

// ---- quantisation ----------------------------------------------------------------
// x c + y s as hi + lo: the products' rounding errors by fma, the sum's by the
// two-sum, so hi + lo is the exact rotation to about 2^-47 of its terms.
// Explicit roundings: a contracted fma here would break the error terms.
__device__ __forceinline__ void rotate_pair(float x, float c, float y, float s, float& hi, float& lo) {
  const float p1 = __fmul_rn(x, c), e1 = __fmaf_rn(x, c, -p1);
  const float p2 = __fmul_rn(y, s), e2 = __fmaf_rn(y, s, -p2);
  const float sum = __fadd_rn(p1, p2), b = __fsub_rn(sum, p1);
  const float err = __fadd_rn(__fadd_rn(__fsub_rn(p1, __fsub_rn(sum, b)), __fsub_rn(p2, b)), __fadd_rn(e1, e2));
  hi = __fadd_rn(sum, err);
  lo = __fsub_rn(err, __fsub_rn(hi, sum));
  if (!(fabsf(sum) < INFINITY)) {  // infinities and NaN as the plain sum has them
    hi = sum;
    lo = 0.f;
  }
}

// Scale byte of a group whose largest magnitude is m: rounding up an estimate
// just below m / 7 gives the byte or the one under it, and 7 s, exact in
// float32, says which.  (A part below m's last bit can only matter where 7 s = m.)
__device__ __forceinline__ uint32_t kv4_scale_byte(float m) {
  const float q = m * 0.14285711f;  // (1 - 2^-22) / 7, rounded down
  const uint32_t normal = ((__float_as_uint(q) + 0xFFFFFu) >> 20) - (112u << 3);
  const uint32_t small = static_cast<uint32_t>(ceilf(q * 131072.f));  // below 2^-14: multiples of 2^-17
  uint32_t b = min(q >= 6.103515625e-05f ? normal : small, static_cast<uint32_t>(kKv4MaxByte));
  if (7.f * kv4_scale_value(b) < m && b < kKv4MaxByte) ++b;
  return b;
}

// Code (1..15) of hi + lo under scale s > 0, whatever they are: the quotient may
// be one off next to a half; the remainder hi - n s is exact (s has 4 bits, n
// few) and settles it, ties by the low part, then to even.
__device__ __noinline__ uint32_t kv4_code_any(float hi, float lo, float s) {
  float n = rintf(__fdiv_rn(hi, s));
  const float r = __fmaf_rn(-n, s, hi), half = 0.5f * s;
  const bool odd = (__float2int_rn(n) & 1) != 0;
  if (r > half || (r == half && (lo > 0.f || (lo == 0.f && odd)))) n += 1.f;
  else if (r < -half || (r == -half && (lo < 0.f || (lo == 0.f && odd)))) n -= 1.f;
  n = fminf(fmaxf(n, -7.f), 7.f);
  if (hi != hi) n = 0.f;  // NaN is held as 0
  return static_cast<uint32_t>(__float2int_rn(n) + 8);
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
// Half a group: this lane's 8 values as hi + lo, the other half in lane ^ 1.
// Returns the group's scale byte and the lane's 8 nibbles (dim i in nibble i).
// few (the same for both lanes): lo is zero and hi has at most 11 significant bits.
// The whole warp takes part.
__device__ __forceinline__ uint32_t kv4_quantise(const float (&hi)[8], const float (&lo)[8], bool few,
                                                 uint32_t& codes) {
  float m = fabsf(hi[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(hi[i]));
  m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
  const uint32_t b = kv4_scale_byte(m);
  const float s = kv4_scale_value(b);
  // hi / s to the nearest whole number by adding 1.5 2^23 (and 8, the code's own
  // offset), from an estimate a little above and one a little below: where they
  // agree they are right.  Where not, the quotient is next to a half: with few
  // bits it is on it (others are 2^-12 off), and the even number holds.
  constexpr float kRound = 12582920.f;
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  const float above = inv * (1.f + 0x1p-20f), below = inv * (1.f - 0x1p-20f);
  uint32_t differ = 0u;
  codes = 0u;
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    const uint32_t t = __float_as_uint(__fmaf_rn(hi[i], above, kRound));
    const uint32_t u = __float_as_uint(__fmaf_rn(hi[i], below, kRound));
    differ |= t ^ u;
    codes = codes * 16u + ((t & 1u) ? u : t);
  }
  codes -= 0x4B400000u * 0x11111111u;  // each number's bits are 0x4B400000 + 8 + n
  // zero scales (a NaN's byte is 0) and capped ones, and what the low parts decide, are for below
  const bool sure = b - 1u < kKv4MaxByte - 1u && (few || (differ == 0u && 7.f * s != m));
  if (__all_sync(0xffffffffu, sure)) return b;
  m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(hi[i]));  // (NaN counts for nothing)
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
  uint32_t c = kv4_scale_byte(m);
  float t = kv4_scale_value(c);
  bool over = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) over = over || (hi[i] == m && lo[i] > 0.f) || (hi[i] == -m && lo[i] < 0.f);
  const uint32_t votes = __ballot_sync(0xffffffffu, over) >> (threadIdx.x & 30);
  if ((votes & 3u) && 7.f * t == m && c < kKv4MaxByte) t = kv4_scale_value(++c);
  if (!sure) {
    codes = c == 0u ? 0x88888888u : 0u;
    if (c != 0u) {
#pragma unroll
      for (int i = 0; i < 8; ++i) codes |= kv4_code_any(hi[i], lo[i], t) << (4 * i);
    }
  }
  return c;
}

// Four pairs of halves of a code word: nibbles (i, i + 4) for i = 0 .. 3, each
// times its scale.  (Bits put into the mantissa of a power of two make a float of
// a small whole number, the common way around a conversion.)  1024 + u (bits 0-3
// of a half's mantissa) less 1032, or 1024 + 16 u (bits 4-7) over 16 less 72, is
// u - 8 exactly; so is the product.
__device__ __forceinline__ void kv4_values(uint32_t w, uint32_t s, uint32_t (&v)[4]) {
  const uint32_t x = w >> 8;
  asm("{\n\t.reg .b32 a, b, c, d;\n\t"
      "lop3.b32 a, %4, 0x000F000F, 0x64006400, 0xEA;\n\t"
      "lop3.b32 b, %4, 0x00F000F0, 0x64006400, 0xEA;\n\t"
      "lop3.b32 c, %5, 0x000F000F, 0x64006400, 0xEA;\n\t"
      "lop3.b32 d, %5, 0x00F000F0, 0x64006400, 0xEA;\n\t"
      "sub.rn.f16x2 a, a, %7;\n\t"
      "fma.rn.f16x2 b, b, %8, %9;\n\t"
      "sub.rn.f16x2 c, c, %7;\n\t"
      "fma.rn.f16x2 d, d, %8, %9;\n\t"
      "mul.rn.f16x2 %0, a, %6;\n\t"
      "mul.rn.f16x2 %1, b, %6;\n\t"
      "mul.rn.f16x2 %2, c, %6;\n\t"
      "mul.rn.f16x2 %3, d, %6;\n\t}"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
      : "r"(w), "r"(x), "r"(s), "r"(0x64086408u), "r"(0x2C002C00u), "r"(0xD480D480u));
}

// A pair of scales for pairs of bf16 values, and -136 times it (17 times 8 times
// at most 4 bits: 8 bits, exact).  A scale's 8 bits lie in a bf16's as they do in
// a half's, with an exponent 112 less; below 2^-14 they are subnormal in both.
struct Kv4ScaleBf {
  uint32_t s, c;
};
__device__ __forceinline__ Kv4ScaleBf kv4_scales_bf(uint32_t w, uint32_t selector) {  // selector as in kv4_scales
  Kv4ScaleBf k;
  const uint32_t b = __byte_perm(w, 0u, selector) * 16u;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(k.s) : "r"(b), "r"(0x77807780u));    // 2^112
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(k.c) : "r"(k.s), "r"(0xC308C308u));  // -136
  return k;
}
// kv4_values as bf16: 128 + u times the scale less 136 times it, exact in one step.
__device__ __forceinline__ void kv4_values(uint32_t w, const Kv4ScaleBf& k, uint32_t (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("{\n\t.reg .b32 a;\n\t"
        "lop3.b32 a, %1, 0x000F000F, 0x43004300, 0xEA;\n\t"
        "fma.rn.bf16x2 %0, a, %2, %3;\n\t}"
        : "=r"(v[i])
        : "r"(w >> (4 * i)), "r"(k.s), "r"(k.c));
}

// ---- append ------------------------------------------------------------------------
// Thread = (8 dims, slice of the heads): a block on one row, d / 8 octets by its
// other threads' slices; a thread keeps its 8 dims' angles in registers over
// the heads it walks.  Reads and writes of rows are 16 bytes a lane, contiguous
// over a head.  blockIdx.x = row; gridDim.y = 1: a block takes the whole row;
// else blockIdx.y = a batch of query heads, one a thread, then K, then V.
// 10239 rows of 32 + 8 + 8 heads of 128 (224 MB): 80 us, 34 at the copy rate.
// No unit is full (47% of the issue slots, 29% of DRAM): a warp's chain of loads,
// rotation, codes and stores bounds it, and registers how many of them it has in
// flight (two query heads; rows of float32, as the engine's, already spill some
// 60 bytes a thread: 512 of 16 + 4 + 4 heads of 64 5.1 us, 0.7 at the copy rate).
constexpr int kKv4AppendThreads = 128;  // at most; one warp a row where there are many rows (see kv4.cu)

// How the first `rotary` dims of a head pair up.
enum Kv4Rope { kRopeNone, kRopeBlocks, kRopePairs, kRopeAny };  // none; i, i + half with half % 8 = 0; 2i, 2i + 1; else

// The angles of a thread's 8 dims from i0: out[i] = x[i] c[i] + partner[i] s[i].
template <int ROPE>
__device__ __forceinline__ void kv4_angles(const Kv4AppendArgs& a, int pos, int i0, float (&c)[8], float (&s)[8]) {
  const int half = a.rotary >> 1;
  const float* cr = a.cos + static_cast<int64_t>(pos) * half;
  const float* sr = a.sin + static_cast<int64_t>(pos) * half;
  const bool vec = ((reinterpret_cast<uintptr_t>(cr) | reinterpret_cast<uintptr_t>(sr)) & 15u) == 0;
  if (ROPE == kRopeBlocks && vec) {
    const int f = i0 < half ? i0 : i0 - half;
    const float sign = i0 < half ? -1.f : 1.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(cr + f) + k), y = __ldg(reinterpret_cast<const float4*>(sr + f) + k);
      c[4 * k] = x.x; c[4 * k + 1] = x.y; c[4 * k + 2] = x.z; c[4 * k + 3] = x.w;
      s[4 * k] = sign * y.x; s[4 * k + 1] = sign * y.y; s[4 * k + 2] = sign * y.z; s[4 * k + 3] = sign * y.w;
    }
  } else if (ROPE == kRopePairs && vec && (half & 3) == 0) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(cr + (i0 >> 1))), y = __ldg(reinterpret_cast<const float4*>(sr + (i0 >> 1)));
    c[0] = c[1] = x.x; c[2] = c[3] = x.y; c[4] = c[5] = x.z; c[6] = c[7] = x.w;
    s[0] = -y.x; s[1] = y.x; s[2] = -y.y; s[3] = y.y;
    s[4] = -y.z; s[5] = y.z; s[6] = -y.w; s[7] = y.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int dim = i0 + i;
      c[i] = 1.f;
      s[i] = 0.f;
      if (dim < a.rotary) {
        const int f = ROPE == kRopePairs ? dim >> 1 : dim < half ? dim : dim - half;
        const bool first = ROPE == kRopePairs ? (dim & 1) == 0 : dim < half;
        c[i] = __ldg(cr + f);
        s[i] = first ? -__ldg(sr + f) : __ldg(sr + f);
      }
    }
  }
}
// The partners of a head's 8 dims from i0, where they are elsewhere in the head.
template <int ROPE, class T>
__device__ __forceinline__ Eight<T> kv4_partners(const Kv4AppendArgs& a, const T* head, int i0, bool vec) {
  const int half = a.rotary >> 1;
  if (ROPE == kRopeBlocks) return load8(head + (i0 < half ? i0 + half : i0 - half), vec);
  Eight<T> y;
  if (ROPE == kRopeAny) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int dim = i0 + i;
      y.v[i] = head[dim < half ? dim + half : dim < a.rotary ? dim - half : dim];
    }
  }
  return y;
}

template <class T, class TQ, int ROPE>
__global__ void __launch_bounds__(kKv4AppendThreads, 6) kv4_append_kernel(
    const __grid_constant__ Kv4AppendArgs a) {
  pdl_wait();
  pdl_launch();
  const int oct_bits = a.c.d == 64 ? 3 : 4;  // d / 8 octets
  const int oct = threadIdx.x & ((1 << oct_bits) - 1), slice = threadIdx.x >> oct_bits, slices = blockDim.x >> oct_bits;
  const int64_t row = blockIdx.x;
  const int i0 = oct * 8, y = blockIdx.y;
  const int nq = a.q != nullptr ? a.n_heads : 0, q_batches = gridDim.y - 2;
  const bool all = gridDim.y == 1, do_k = all || y == q_batches, do_v = all || y == q_batches + 1;
  const bool turns = ROPE != kRopeNone && i0 < a.rotary;  // some of the thread's dims turn
  const bool part = ROPE != kRopeNone && i0 + 8 > a.rotary;  // but not all of them
  const bool kvec = aligned16(a.k, a.k_row, a.k_head, sizeof(T)), vvec = aligned16(a.v, a.v_row, a.v_head, sizeof(T));
  const int pos = __ldg(a.pos + row);
  const int sid = a.seq != nullptr ? __ldg(a.seq + row) : static_cast<int>(row);
  // Loops below are alike for all threads of the block (a thread without a head
  // goes along): the warp stays together.
  const T* k = static_cast<const T*>(a.k) + row * a.k_row + slice * a.k_head;
  const T* v = static_cast<const T*>(a.v) + row * a.v_row + slice * a.v_head;
  Eight<T> kx = {}, ky = {}, vx = {};
  auto fetch_k = [&](int g) {
    if (g < a.c.n_kv) {
      kx = load8(k + i0, kvec);
      if (turns) ky = kv4_partners<ROPE>(a, k, i0, kvec);
    }
  };
  if (do_k) fetch_k(slice);
  if (do_v && slice < a.c.n_kv) vx = load8(v + i0, vvec);
  if (pos < 0) return;  // idle row
  if (ROPE != kRopeNone && pos >= a.max_pos) {
    if (threadIdx.x == 0) kv4_error(a.c.status, kKv4BadPos);
    return;
  }
  uint8_t* page = kv4_page(a.c, sid, pos, slice);
  if (page == nullptr) return;  // (its query is skipped too)
  float c[8], s[8];
  if (turns) kv4_angles<ROPE>(a, pos, i0, c, s);

  if (all || y < q_batches) {
    const bool qvec = aligned16(a.q, a.q_row, a.q_head, sizeof(T)), ovec = aligned16(a.q_out, a.qo_row, a.qo_head, sizeof(TQ));
    const int h0 = all ? 0 : y * slices, h1 = all ? nq : min(nq, (y + 1) * slices);
    const T* q = static_cast<const T*>(a.q) + row * a.q_row + (h0 + slice) * a.q_head;
    TQ* o = static_cast<TQ*>(a.q_out) + row * a.qo_row + (h0 + slice) * a.qo_head + i0;
    const int64_t q_step = slices * a.q_head, o_step = slices * a.qo_head;
#pragma unroll 2
    for (int h = h0; h < h1; h += slices, q += q_step, o += o_step) {
      const bool mine = h + slice < h1;
      Eight<T> x = {}, p = {};
      if (mine) {
        x = load8(q + i0, qvec);
        if (turns) p = kv4_partners<ROPE>(a, q, i0, qvec);
      }
      float r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = to_f32(x.v[i]);
      if (turns) {
        float z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = ROPE == kRopePairs ? r[i ^ 1] : to_f32(p.v[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = fmaf(r[i], c[i], z[i] * s[i]);
        if (part) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i0 + i >= a.rotary) r[i] = to_f32(x.v[i]);
        }
      }
      __syncwarp();  // q_out may be q: a head's threads, all of one warp, have read their partners
      if (mine) store8(o, r, ovec);
    }
  }
  if (!do_k && !do_v) return;
  const int r = pos % kKv4Page, page_step = slices * kv4_page_bytes(a.c.d);
  if (do_k) {
    const int code_at = kv4_k_code(oct >> 1, r) + 4 * (oct & 1), scale_at = kv4_k_scale(a.c.d, oct >> 1, r);
    const bool few = sizeof(T) == 2 && !(ROPE != kRopeNone && (i0 & ~15) < a.rotary);  // (alike over a group)
    uint8_t* to = page;
    for (int g = slice; g - slice < a.c.n_kv; g += slices, to += page_step) {
      float hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hi[i] = to_f32(kx.v[i]);
        lo[i] = 0.f;
      }
      if (turns) {
        float z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = ROPE == kRopePairs ? hi[i ^ 1] : to_f32(ky.v[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) rotate_pair(hi[i], c[i], z[i], s[i], hi[i], lo[i]);
        if (part) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i0 + i >= a.rotary) {
              hi[i] = to_f32(kx.v[i]);
              lo[i] = 0.f;
            }
        }
      }
      k += slices * a.k_head;
      fetch_k(g + slices);
      uint32_t codes;
      const uint32_t b = kv4_quantise(hi, lo, few, codes);
      if (g < a.c.n_kv) {
        *reinterpret_cast<uint32_t*>(to + code_at) = codes;
        if ((oct & 1) == 0) to[scale_at] = static_cast<uint8_t>(b);
      }
    }
  }
  if (do_v) {
    const int code_at = kv4_v_code(a.c.d, 2 * oct, r), scale_at = kv4_v_scale(a.c.d, oct >> 1, r);
    for (int g = slice; g - slice < a.c.n_kv; g += slices, page += page_step) {
      float hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hi[i] = to_f32(vx.v[i]);
        lo[i] = 0.f;
      }
      v += slices * a.v_head;
      if (g + slices < a.c.n_kv) vx = load8(v + i0, vvec);
      uint32_t codes;
      const uint32_t b = kv4_quantise(hi, lo, sizeof(T) == 2, codes);
      if (g < a.c.n_kv) {
        uint16_t* to = reinterpret_cast<uint16_t*>(page + code_at);
        to[0] = static_cast<uint16_t>(codes);
        to[2] = static_cast<uint16_t>(codes >> 16);  // (the next quad's two bytes are 4 bytes on)
        if ((oct & 1) == 0) page[scale_at] = static_cast<uint8_t>(b);
      }
    }
  }
}

// ---- read --------------------------------------------------------------------------
// Rows out of the cache as values (zeros where the position is negative or the
// table names no page).  Block: 128 threads on one row; thread = 8 dims of a
// kv head's K or V.  10239 rows of 8 heads of 128 (54 MB): 14.8 us, 3.6 TB/s, of
// the 8.2 that the copy rate gives: position, table and page are loads that wait
// for one another, and a block has one row's.
template <class T>
__global__ void __launch_bounds__(128) kv4_read_kernel(const __grid_constant__ Kv4ReadArgs a) {
  pdl_wait();
  pdl_launch();
  const int octs = a.c.d >> 3, oct = threadIdx.x & (octs - 1);
  const int64_t row = blockIdx.x;
  const int pos = __ldg(a.pos + row), sid = a.seq != nullptr ? __ldg(a.seq + row) : static_cast<int>(row);
  const uint8_t* block = pos >= 0 ? kv4_page(a.c, sid, pos, 0) : nullptr;
  const int r = pos >= 0 ? pos % kKv4Page : 0, step = 128 / octs * gridDim.y;
  const bool kvec = (reinterpret_cast<uintptr_t>(a.k) & 15u) == 0, vvec = (reinterpret_cast<uintptr_t>(a.v) & 15u) == 0;
#pragma unroll 4
  for (int hh = threadIdx.x / octs + blockIdx.y * (128 / octs); hh < 2 * a.c.n_kv; hh += step) {
    const bool is_k = hh < a.c.n_kv;
    const int g = is_k ? hh : hh - a.c.n_kv;
    uint32_t p[4] = {0u, 0u, 0u, 0u};  // dims (0, 1), (2, 3), ..
    if (block != nullptr) {
      const uint8_t* page = block + g * kv4_page_bytes(a.c.d);
      uint32_t codes, b;
      if (is_k) {
        codes = *reinterpret_cast<const uint32_t*>(page + kv4_k_code(oct >> 1, r) + 4 * (oct & 1));
        b = page[kv4_k_scale(a.c.d, oct >> 1, r)];
      } else {
        const uint16_t* w = reinterpret_cast<const uint16_t*>(page + kv4_v_code(a.c.d, 2 * oct, r));
        codes = w[0] | (static_cast<uint32_t>(w[2]) << 16);  // (the next quad's two bytes are 4 bytes on)
        b = page[kv4_v_scale(a.c.d, oct >> 1, r)];
      }
      uint32_t v[4];
      kv4_values(codes, b * 0x00800080u, v);
      p[0] = __byte_perm(v[0], v[1], 0x5410);
      p[1] = __byte_perm(v[2], v[3], 0x5410);
      p[2] = __byte_perm(v[0], v[1], 0x7632);
      p[3] = __byte_perm(v[2], v[3], 0x7632);
    }
    T* out = static_cast<T*>(is_k ? a.k : a.v) + (row * a.c.n_kv + g) * a.c.d + 8 * oct;
    put8(out, p, is_k ? kvec : vvec);
  }
}

// ---- attention -----------------------------------------------------------------------
// S^T = K Q^T and O^T = V^T P^T on m16n8k16: the 16 positions of a page
// are the rows of the first product and the reduction of the second, the query
// columns (row of the sequence, head of the group) its 8 columns, so no
// fragment of the cache is wasted on absent queries.
//
// Both operands of both products are exact but for the probabilities: held
// values are exact in bf16 and in half, so S is formed in the queries' own type
// (as halves under a power of two per column, bf16 queries lost what lies 2^17
// below their row's largest, and a wave of 256 took 14.5 us, not 13.9) and O in
// half.  Probabilities keep 11 bits (as two halves they would double the second
// product; a result of 8 bits hides it, one of 11 is off by up to a third more):
// they carry a factor 2^15, so those down to 2^-29 of the row's largest are normal
// halves, and the sum they are divided by, of the unrounded ones, carries it too.
//
// An exponent is the difference of two scores first, then scaled: scaled scores
// apart, each rounded at its own size, would be off by more than the factor's room
// from 2^25 on.  (An instruction more a score: 45.9 us, not 45.6, on 131071
// positions; prompts' chunks 151, not 149.)
constexpr float kKv4POffset = 15.f;

// Scale pair from two bytes of w: selector 0x4i4j puts bytes j, i into the halves.
__device__ __forceinline__ uint32_t kv4_scales(uint32_t w, uint32_t selector) {
  return __byte_perm(w, 0u, selector) * 128u;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void mma_half(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_half_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {  // d = a b
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// The same on pairs of T, bf16 or half.
template <class T>
__device__ __forceinline__ void mma_scores(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                           uint32_t b0, uint32_t b1, bool first) {
  if constexpr (std::is_same<T, __half>::value) {
    if (first) mma_half_first(d, a0, a1, a2, a3, b0, b1);
    else mma_half(d, a0, a1, a2, a3, b0, b1);
  } else if (first) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
// A pair of scales for values of type T.
template <class T>
__device__ __forceinline__ auto kv4_scales_of(uint32_t w, uint32_t selector) {
  if constexpr (std::is_same<T, __half>::value) return kv4_scales(w, selector);
  else return kv4_scales_bf(w, selector);
}
template <class T>
__device__ __forceinline__ void load16(const T* p, uint32_t (&w)[8], bool in, bool vec) {  // 16 elements of 2 bytes
  if (!in) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0u;
  } else if (vec) {
    const uint4 x = *reinterpret_cast<const uint4*>(p), y = *reinterpret_cast<const uint4*>(p + 8);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    w[4] = y.x; w[5] = y.y; w[6] = y.z; w[7] = y.w;
  } else {
    const uint16_t* b = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = b[2 * i] | (static_cast<uint32_t>(b[2 * i + 1]) << 16);
  }
}
// A column's query fragments: f[h][2 s], f[h][2 s + 1] for k-step s, dims (s, s + 4)
// and (8 + s, 12 + s) of the lane's 16 at q + 64 h.
template <int NH, class T>
__device__ __forceinline__ void kv4_query(const T* q, bool in, bool vec, uint32_t (&f)[NH][8]) {
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    uint32_t w[8];
    load16(q + 64 * h, w, in, vec);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint32_t sel = s & 1 ? 0x7632 : 0x5410;  // the odd or even elements of two words
      f[h][2 * s] = __byte_perm(w[s >> 1], w[2 + (s >> 1)], sel);
      f[h][2 * s + 1] = __byte_perm(w[4 + (s >> 1)], w[6 + (s >> 1)], sel);
    }
  }
}

__device__ __forceinline__ float exp2_fast(float x) {  // 2^x (2 ulp), 0 at -infinity
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Where a CTA's work lies.
struct Kv4Tile {
  int seq, g, tile, split;
  int r0, rows, len;
  __device__ __forceinline__ int cols(const Kv4AttnArgs& a) const { return rows * a.group; }
};
__device__ __forceinline__ int kv4_row(const Kv4AttnArgs& a, int col) {  // col / group
  return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(col)) * a.group_inv >> 32);
}
// positions that column c sees
__device__ __forceinline__ int kv4_limit(const Kv4AttnArgs& a, const Kv4Tile& t, int c) {
  return t.rows == 1 ? t.len : min(t.len, max(0, t.len - t.rows + kv4_row(a, c) + 1));
}
// Tile of query columns and split of kv head g of sequence seq.
// False when the tile has no columns.  Bad inputs (lengths past the table or
// max_len, rows past n_rows or max_rows) leave rows or len 0 and set the status.
__device__ __forceinline__ bool kv4_tile(const Kv4AttnArgs& a, int seq, int g, int tile, int split, Kv4Tile& t) {
  t.seq = seq;
  t.g = g;
  t.tile = tile;
  t.split = split;
  t.len = __ldg(a.lens + t.seq) + a.len_add;
  t.r0 = t.seq;
  t.rows = 1;
  if (a.rows_of_one > 0) t.rows = a.rows_of_one;
  if (a.q_start != nullptr) {
    t.r0 = __ldg(a.q_start + t.seq);
    t.rows = __ldg(a.q_start + t.seq + 1) - t.r0;
    if (t.rows <= 0) return false;
    if (t.r0 < 0 || t.rows > a.max_rows || t.rows > a.n_rows - t.r0) {
      if (threadIdx.x == 0) kv4_error(a.c.status, kKv4BadPos);
      return false;
    }
  }
  if (t.tile * a.tile_cols >= t.cols(a)) return false;
  if (t.len > a.max_len) {
    if (threadIdx.x == 0) kv4_error(a.c.status, kKv4BadPos);
    t.len = 0;
  }
  if (t.len < 0) t.len = 0;
  return true;
}
// Pages that a tile's columns see.
__device__ __forceinline__ int kv4_tile_pages(const Kv4AttnArgs& a, const Kv4Tile& t) {
  const int last = min(t.cols(a), (t.tile + 1) * a.tile_cols) - 1;
  return (kv4_limit(a, t, last) + kKv4Page - 1) / kKv4Page;
}

// A row that sees a position of a block that the table does not name is zero: a
// share of it without those positions would look like an answer.  Its share of a
// column has an infinite maximum, next to which no other share counts, and a sum
// and o of zero (as an infinite score would not: its sum is NaN).
__device__ __forceinline__ float kv4_share(float m, float top, float scale_log2) {  // what a share counts for, 0 .. 1
  return m == top ? 1.f : exp2_fast((m - top) * scale_log2);
}
// A split's share of a column: d floats of o, then its maximum (of the scores
// before their scale) and sum.
__device__ __forceinline__ float* kv4_part(const Kv4AttnArgs& a, int seq, int g, int tile, int split, int col, int d) {
  const int64_t unit = (static_cast<int64_t>(seq) * a.c.n_kv + g) * a.tiles + tile;
  return a.part + ((unit * a.splits + split) * a.tile_cols + col) * (d + 4);
}

// Waits for a phase of an mbarrier: tries that sleep up to a microsecond each,
// at most kKv4Tries of them (0.2 s).  No timer and no call: either one in the
// loop made the compiler spill around every wait.
constexpr uint32_t kKv4Tries = 200000u;
__device__ __forceinline__ bool kv4_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t at = smem_addr(bar);
  uint32_t ok = 0u;
  for (uint32_t i = 0; i < kKv4Tries && !ok; ++i)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(at), "r"(parity), "r"(1000u) : "memory");
  return ok != 0u;
}
// The same without sleeping, for a warp that others wait for (a sleeping one was
// seen to wake up some 250 cycles late).
constexpr uint32_t kKv4Polls = 1u << 23;
__device__ __forceinline__ bool kv4_poll(uint64_t* bar, uint32_t parity) {
  const uint32_t at = smem_addr(bar);
  uint32_t ok = 0u;
  for (uint32_t i = 0; i < kKv4Polls && !ok; ++i)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(at), "r"(parity) : "memory");
  return ok != 0u;
}

// The pages of a warp's ring: kKv4Ahead + 1 steps of P pages.
constexpr int kKv4Ahead = 2;
constexpr __host__ __device__ int kv4_step_pages(int nh) { return nh == 1 ? 4 : 2; }
constexpr int kKv4Warps = 4;  // of a CTA (2: the same on a wave of 256; 1: slower everywhere)
template <int NH, int NB>
constexpr __host__ __device__ int kv4_attn_smem() {
  constexpr int W = kKv4Warps, ring = W * (kKv4Ahead + 1) * kv4_step_pages(NH) * kv4_page_bytes(64 * NH);
  constexpr int join = W * 8 * NB * (64 * NH + 2) * 4;  // reuses the ring
  return ring > join ? ring : join;
}

// One CTA of W warps per (sequence, kv head, tile of 8 NB query columns, split
// of the positions).  Warp w takes the split's pages w, w + W, ...; each runs
// its own online softmax, and the warps meet in shared memory at the end.
// A page's bytes are contiguous: each comes by one bulk copy into the warp's
// ring, kKv4Ahead steps ahead; a step takes P pages, so the running maximum
// and the rescaling of o are paid once for 16 P positions.
// One row of 32 heads over 8 of 128 dims on 131071 positions: 46 us with the join, 3.3
// TB/s; 32 such rows on 1001 to 16384: 93 us, 3.5 TB/s.  Bound by instructions, 386 a
// page of 2304 bytes, most of them turning codes to values, at 62% of the issue slots.
template <class T, int NH, int NB>
__global__ void __launch_bounds__(32 * kKv4Warps) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
  constexpr int W = kKv4Warps, D = 64 * NH, COLS = 8 * NB, P = kv4_step_pages(NH), PB = kv4_page_bytes(D), SLOTS = kKv4Ahead + 1;
  extern __shared__ __align__(16) uint8_t kv4_smem[];
  __shared__ uint64_t s_bar[W][SLOTS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  uint64_t* bar = s_bar[warp];
  if (lane == 0) {
    for (int i = 0; i < SLOTS; ++i) mbar_init(&bar[i], 1);
    fence_mbar_init();
  }
  __syncwarp();
  bool after = !a.early;  // the kernel before has ended
  if (after) pdl_wait();
  pdl_launch();
  Kv4Tile tl;
  // grid: x = sequence, y = kv head, z = tile + tiles * split
  const int split = a.tiles == 1 ? blockIdx.z : blockIdx.z / a.tiles;
  const bool work = kv4_tile(a, blockIdx.x, blockIdx.y, blockIdx.z - split * a.tiles, split, tl);
  const int pages = work ? kv4_tile_pages(a, tl) : 0;
  const int lo = split * a.split_pages, hi = min(pages, lo + a.split_pages);
  if (!work || (lo >= hi && split > 0)) {  // (the first split always answers)
    if (!after) pdl_wait();
    return;
  }
  const int c0 = tl.tile * COLS, cols = tl.cols(a);

  // ---- the warp's pages: the k-th is lo + warp + W k ----
  const int32_t* table = a.c.table + tl.seq * a.c.table_ld;
  const int n_mine = max(0, hi - lo - warp + W - 1) / W, steps = (n_mine + P - 1) / P;
  uint8_t* ring = kv4_smem + warp * (SLOTS * P * PB);
  const uint64_t pol = l2_policy_evict_first();
  // lane p < P: block of page p of a step (loaded one step before its copies go out)
  auto load_id = [&](int step) {
    const int k = step * P + lane;
    return lane < P && k < n_mine ? __ldg(table + lo + warp + W * k) : -1;
  };
  int fill = 0;  // the slot that the next step's copies fill
  int lost = INT_MAX;  // the warp's first position whose block the table does not name
  auto issue = [&](int step, int id) {
    if (step >= steps) return;
    const int slot = fill, n = min(P, n_mine - step * P);
    const bool good = kv4_named(a.c, id);
    const uint32_t in = __ballot_sync(0xffffffffu, lane < n && good);
    uint8_t* dst = ring + slot * P * PB;
    if (__popc(in) != n) {  // a page that the table does not name is read as zeros
      lost = min(lost, (lo + warp + W * (step * P + __ffs(~in) - 1)) * kKv4Page);
      for (int p = 0; p < n; ++p)
        if (!((in >> p) & 1u))
          for (int i = lane * 16; i < PB; i += 512) *reinterpret_cast<uint4*>(dst + p * PB + i) = make_uint4(0, 0, 0, 0);
      if (lane == 0) kv4_error(a.c.status, kKv4BadTable);
      fence_proxy_async_smem();  // before the slot's next copies
    }
    if (lane == 0) mbar_arrive_expect_tx(&bar[slot], static_cast<uint32_t>(__popc(in)) * PB);
    __syncwarp();
    if ((in >> lane) & 1u)
      bulk_g2s(dst + lane * PB, a.c.pool + (static_cast<int64_t>(id) * a.c.n_kv + tl.g) * PB, PB, &bar[slot], pol);
    fill = fill + 1 == SLOTS ? 0 : fill + 1;
  };
  bool waited = true;
  uint32_t phase = 0;  // bit i: the parity that slot i completes next
  auto wait = [&](int slot) {  // bounded; a wait that runs out sets the status
    uint64_t* b = &bar[slot];
    const uint32_t parity = (phase >> slot) & 1u;
    phase ^= 1u << slot;
    if (!kv4_wait(b, parity)) waited = false;
  };
  int id = load_id(0);
#pragma unroll
  for (int st = 0; st < kKv4Ahead; ++st) {
    const int next = load_id(st + 1);
    if (!after && st == steps - 1) {  // the sequence's last page may be in a warp's last step
      pdl_wait();
      after = true;
    }
    issue(st, id);
    id = next;
  }
  if (!after) pdl_wait();

  // query fragments: column gid of each block, dims 64h + 16 tig .. in the codes' order
  uint32_t qf[NB][NH][8];
  const float up = a.scale_log2;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int col = c0 + 8 * nb + gid;
    const bool in = col < cols;
    const int row = in && tl.rows > 1 ? kv4_row(a, col) : 0, head = in ? col - row * a.group : 0;
    const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(tl.r0 + row) * a.q_row +
                 static_cast<int64_t>(tl.g * a.group + head) * a.q_head + 16 * tig;
    kv4_query<NH>(q, in, aligned16(a.q, a.q_row, a.q_head, sizeof(T)), qf[nb]);
  }
  // columns 2 tig, 2 tig + 1 of each block: the positions they see
  int lim[NB][2];
  float m[NB][2], l[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = c0 + 8 * nb + 2 * tig + e;
      lim[nb][e] = col < cols ? kv4_limit(a, tl, col) : 0;
      m[nb][e] = -INFINITY;  // of the scores before their scale
      l[nb][e] = 0.f;
    }
  const int seen = kv4_limit(a, tl, min(cols, c0 + COLS) - 1);  // positions that any column sees
  float o[NB][4 * NH][4];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int j = 0; j < 4 * NH; ++j) o[nb][j][0] = o[nb][j][1] = o[nb][j][2] = o[nb][j][3] = 0.f;

  const int all_see = kv4_limit(a, tl, c0);  // positions that every column sees
  int slot = 0;
  for (int step = 0; step < steps; ++step, slot = slot + 1 == SLOTS ? 0 : slot + 1) {
    const int next = load_id(step + kKv4Ahead + 1);
    issue(step + kKv4Ahead, id);
    id = next;
    wait(slot);
    __syncwarp();
    const uint8_t* page0 = ring + slot * P * PB;
    const int n = min(P, n_mine - step * P);
    const int at0 = (lo + warp + W * step * P) * kKv4Page;  // page p of the step starts at at0 + 16 W p
    // No branch around the pages a last step lacks: their scores are masked and
    // their V scales dropped below, whatever the ring holds.
    float sc[P][NB][4];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint8_t* page = page0 + p * PB;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const uint4 kc = reinterpret_cast<const uint4*>(page)[h * 32 + lane];
        const uint32_t kb = reinterpret_cast<const uint16_t*>(page + 8 * D)[h * 32 + lane];
        const auto s0 = kv4_scales_of<T>(kb, 0x4040), s1 = kv4_scales_of<T>(kb, 0x4141);
        uint32_t k0[4], k1[4], k2[4], k3[4];
        kv4_values(kc.x, s0, k0);
        kv4_values(kc.z, s1, k1);
        kv4_values(kc.y, s0, k2);
        kv4_values(kc.w, s1, k3);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            mma_scores<T>(sc[p][nb], k0[s], k1[s], k2[s], k3[s], qf[nb][h][2 * s], qf[nb][h][2 * s + 1],
                          h == 0 && s == 0);
      }
    }
    // softmax of the step's positions: rows gid (c0, c1) and gid + 8 (c2, c3) of each page
    const bool whole = n == P && at0 + W * kKv4Page * (P - 1) + kKv4Page <= all_see;
    if (!whole) {
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int left = p < n ? lim[nb][e] - at0 - W * kKv4Page * p - gid : 0;  // > 0: row gid is seen
            if (left <= 0) sc[p][nb][e] = -INFINITY;
            if (left <= 8) sc[p][nb][2 + e] = -INFINITY;
          }
    }
    uint32_t pf[P][NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float al[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(sc[0][nb][e], sc[0][nb][2 + e]);
#pragma unroll
        for (int p = 1; p < P; ++p) mx = fmaxf(mx, fmaxf(sc[p][nb][e], sc[p][nb][2 + e]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(m[nb][e], mx), ref = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: all zero
        al[e] = exp2_fast((m[nb][e] - ref) * up);
        m[nb][e] = mn;
        float sum = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
          sc[p][nb][e] = exp2_fast(fmaf(sc[p][nb][e] - ref, up, kKv4POffset));
          sc[p][nb][2 + e] = exp2_fast(fmaf(sc[p][nb][2 + e] - ref, up, kKv4POffset));
          sum += sc[p][nb][e] + sc[p][nb][2 + e];
        }
        l[nb][e] = fmaf(l[nb][e], al[e], sum);
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        pf[p][nb][0] = transpose8x8(pack_half2(sc[p][nb][0], sc[p][nb][1]));
        pf[p][nb][1] = transpose8x8(pack_half2(sc[p][nb][2], sc[p][nb][3]));
      }
      if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {  // a maximum grew
#pragma unroll
        for (int j = 0; j < 4 * NH; ++j) {
          o[nb][j][0] *= al[0];
          o[nb][j][1] *= al[1];
          o[nb][j][2] *= al[0];
          o[nb][j][3] *= al[1];
        }
      }
    }
    // positions past the last one seen may never have been written: their V
    // scales are dropped, since 0 times an infinity or a NaN is not 0
    uint32_t keep[P];
#pragma unroll
    for (int p = 0; p < P; ++p) keep[p] = 0xFFFFFFFFu;
    if (!whole) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int left = p < n ? seen - at0 - W * kKv4Page * p : 0;
        keep[p] = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (2 * tig + 8 * (i >> 1) + (i & 1) < left) keep[p] |= 0xFFu << (8 * i);
      }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint8_t* page = page0 + p * PB;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const uint4 vc = reinterpret_cast<const uint4*>(page + 9 * D)[h * 32 + lane];
        const uint32_t vb = reinterpret_cast<const uint32_t*>(page + 17 * D)[(h * 4 + (gid >> 1)) * 4 + tig] & keep[p];
        const uint32_t s0 = kv4_scales(vb, 0x4140), s1 = kv4_scales(vb, 0x4342);
        // word (positions 2 tig, + 1 or 2 tig + 8, + 9; dims 0-3 or 4-7 of the lane's 8)
        uint32_t v0[4], v1[4], w0[4], w1[4];
        kv4_values(vc.x, s0, v0);
        kv4_values(vc.z, s1, w0);
        kv4_values(vc.y, s0, v1);
        kv4_values(vc.w, s1, w1);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {  // block j: dims 2j (row gid) and 2j + 1 (row gid + 8)
          mma_half(o[nb][4 * h], v0[0], v0[1], w0[0], w0[1], pf[p][nb][0], pf[p][nb][1]);
          mma_half(o[nb][4 * h + 1], v0[2], v0[3], w0[2], w0[3], pf[p][nb][0], pf[p][nb][1]);
          mma_half(o[nb][4 * h + 2], v1[0], v1[1], w1[0], w1[1], pf[p][nb][0], pf[p][nb][1]);
          mma_half(o[nb][4 * h + 3], v1[2], v1[3], w1[2], w1[3], pf[p][nb][0], pf[p][nb][1]);
        }
      }
    }
    __syncwarp();  // every lane is done with the step's pages before they are refilled
  }
  if (!__all_sync(0xffffffffu, waited)) {
    // a wait ran out: the result means nothing; wait once more for what is in flight
    if (lane == 0) kv4_error(a.c.status, kKv4Timeout);
    for (int i = 0; i < SLOTS; ++i)
      if (i < steps) {
        phase ^= 1u << i;  // the slot's last phase once more
        wait(i);
      }
  }
  // ---- the result: column 2 tig + e of each block, dims 64h + 8 gid .. in this lane ----
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], 4);
      l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], 8);
      l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], 16);
    }
  if (lost != INT_MAX) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (lost < lim[nb][e]) {
          m[nb][e] = INFINITY;
          l[nb][e] = 0.f;
#pragma unroll
          for (int j = 0; j < 4 * NH; ++j) o[nb][j][e] = o[nb][j][2 + e] = 0.f;
        }
  }
  const bool ovec = aligned16(a.out, a.o_row, a.o_head, sizeof(T));
  // 8 dims from d0 of column c (of the sequence): final, or this split's share
  auto put = [&](int c, int d0, float (&r)[8], float M, float L) {
    if (a.splits == 1) {
      const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);  // a row that sees nothing: zeros (NaN stays NaN)
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] *= inv;
      const int row = tl.rows > 1 ? kv4_row(a, c) : 0;
      store8(static_cast<T*>(a.out) + static_cast<int64_t>(tl.r0 + row) * a.o_row +
                 static_cast<int64_t>(tl.g * a.group + c - row * a.group) * a.o_head + d0,
             r, ovec);
    } else {
      float* dst = kv4_part(a, tl.seq, tl.g, tl.tile, tl.split, c - c0, D);
      *reinterpret_cast<float4*>(dst + d0) = make_float4(r[0], r[1], r[2], r[3]);
      *reinterpret_cast<float4*>(dst + d0 + 4) = make_float4(r[4], r[5], r[6], r[7]);
      if (d0 == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(M, L);
    }
  };
  __syncthreads();  // the ring's memory becomes the warps' states
  float(*s_o)[COLS][D] = reinterpret_cast<float(*)[COLS][D]>(kv4_smem);
  float(*s_m)[COLS] = reinterpret_cast<float(*)[COLS]>(kv4_smem + sizeof(float) * W * COLS * D);
  float(*s_l)[COLS] = s_m + W;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = 8 * nb + 2 * tig + e;
      if (c0 + col >= cols) continue;
      if (gid == 0) {
        s_m[warp][col] = m[nb][e];
        s_l[warp][col] = l[nb][e];
      }
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        float4* dst = reinterpret_cast<float4*>(&s_o[warp][col][64 * h + 8 * gid]);
        dst[0] = make_float4(o[nb][4 * h][e], o[nb][4 * h][2 + e], o[nb][4 * h + 1][e], o[nb][4 * h + 1][2 + e]);
        dst[1] = make_float4(o[nb][4 * h + 2][e], o[nb][4 * h + 2][2 + e], o[nb][4 * h + 3][e], o[nb][4 * h + 3][2 + e]);
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < COLS * (D / 8); i += 32 * W) {
    const int col = i / (D / 8), d0 = i % (D / 8) * 8;
    if (c0 + col >= cols) break;
    float M = s_m[0][col], L = 0.f, r[8];
#pragma unroll
    for (int w = 1; w < W; ++w) M = fmaxf(M, s_m[w][col]);
#pragma unroll
    for (int k = 0; k < 8; ++k) r[k] = 0.f;
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = kv4_share(s_m[w][col], ref, up);
      L = fmaf(f, s_l[w][col], L);
      const float4 x = *reinterpret_cast<const float4*>(&s_o[w][col][d0]), y = *reinterpret_cast<const float4*>(&s_o[w][col][d0 + 4]);
      r[0] = fmaf(f, x.x, r[0]); r[1] = fmaf(f, x.y, r[1]); r[2] = fmaf(f, x.z, r[2]); r[3] = fmaf(f, x.w, r[3]);
      r[4] = fmaf(f, y.x, r[4]); r[5] = fmaf(f, y.y, r[5]); r[6] = fmaf(f, y.z, r[6]); r[7] = fmaf(f, y.w, r[7]);
    }
    put(c0 + col, d0, r, M, L);
  }
}

// Joins the splits of each column: a warp per column, 8 loads in flight a lane
// (a CTA per column with its warps on different splits: the same for 32 columns of
// 74 splits, and 82 us instead of 69 for 256 rows of 4 heads on 8192 positions).
template <class T, int NH>
__global__ void __launch_bounds__(128) kv4_join_kernel(const __grid_constant__ Kv4AttnArgs a) {
  constexpr int D = 64 * NH, PER = 2 * NH, DEEP = 8;
  pdl_wait();
  pdl_launch();
  // grid: x = sequence, y = kv head, z = 4 columns
  const int lane = threadIdx.x & 31;
  const int c = blockIdx.z * 4 + (threadIdx.x >> 5), tile = c / a.tile_cols;
  Kv4Tile tl;
  if (!kv4_tile(a, blockIdx.x, blockIdx.y, tile, 0, tl) || c >= tl.cols(a)) return;
  const int n = max(1, (kv4_tile_pages(a, tl) + a.split_pages - 1) / a.split_pages);
  const float* src = kv4_part(a, tl.seq, tl.g, tile, 0, c - tile * a.tile_cols, D);
  const int64_t step = static_cast<int64_t>(a.tile_cols) * (D + 4);
  float M = -INFINITY;
  for (int s = lane; s < n; s += 32) M = fmaxf(M, src[s * step + D]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f, r[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) r[k] = 0.f;
  for (int s0 = 0; s0 < n; s0 += DEEP) {
    float2 ml[DEEP], x[DEEP][NH];
#pragma unroll
    for (int i = 0; i < DEEP; ++i) {
      const int s = s0 + i;
      ml[i] = s < n ? *reinterpret_cast<const float2*>(src + s * step + D) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int h = 0; h < NH; ++h)
        x[i][h] = s < n ? *reinterpret_cast<const float2*>(src + s * step + 64 * h + 2 * lane) : make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < DEEP; ++i) {
      const float f = kv4_share(ml[i].x, ref, a.scale_log2);
      L = fmaf(f, ml[i].y, L);
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        r[2 * h] = fmaf(f, x[i][h].x, r[2 * h]);
        r[2 * h + 1] = fmaf(f, x[i][h].y, r[2 * h + 1]);
      }
    }
  }
  const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);
  const int row = kv4_row(a, c);
  T* out = static_cast<T*>(a.out) + static_cast<int64_t>(tl.r0 + row) * a.o_row +
           static_cast<int64_t>(tl.g * a.group + c - row * a.group) * a.o_head;
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int k = 0; k < 2; ++k) out[64 * h + 2 * lane + k] = from_f32<T>(r[2 * h + k] * inv);
}

}  // namespace b2d

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
constexpr uint32_t kKv4BadPos = 0x202u, kKv4BadTable = 0x203u;

// The page of position `pos` of the sequence with table row `sid`, or null
// (status set) when the table does not name one.
__device__ __forceinline__ uint8_t* kv4_page(const Kv4Cache& c, int sid, int pos, int g) {
  const int pg = pos / kKv4Page;
  if (sid < 0 || sid >= c.table_rows || pg >= c.bps) {
    kv4_error(c.status, kKv4BadTable);
    return nullptr;
  }
  const int blk = __ldg(c.table + sid * c.table_ld + pg);
  if (blk < 0 || blk >= c.num_blocks) {
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
__device__ __forceinline__ void load8(const T* p, float* x, bool vec) {
  if (vec) {
    __align__(16) T v[8];
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
  }
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

// Scale byte of a group whose largest magnitude is m + ml (ml: the low part).
// The quotient is rounded up, so rounding it up again to 4 bits gives the
// smallest scale s with 7 s >= m exactly; where 7 s = m the low part decides.
__device__ __forceinline__ uint32_t kv4_scale_byte(float m, float ml) {
  const float q = __fdiv_ru(m, 7.f);
  uint32_t b;
  if (q >= 6.103515625e-05f) {  // 2^-14: normal
    b = ((__float_as_uint(q) + 0xFFFFFu) >> 20) - (112u << 3);
  } else {
    b = static_cast<uint32_t>(ceilf(q * 131072.f));  // whole multiples of 2^-17 (exact product)
  }
  b = min(b, static_cast<uint32_t>(kKv4MaxByte));
  if (ml > 0.f && 7.f * kv4_scale_value(b) == m && b < kKv4MaxByte) ++b;
  return b;
}

// Code (1..15) of hi + lo under scale s > 0 (inv = 1 / s).  The quotient may be
// one off next to a half; the remainder hi - n s is exact (s has 4 bits, n few)
// and settles it, ties by the low part, then to even.
__device__ __forceinline__ uint32_t kv4_code(float hi, float lo, float s, float inv) {
  float n = rintf(__fmul_rn(hi, inv));
  const float r = __fmaf_rn(-n, s, hi), half = 0.5f * s;
  const bool odd = (__float2int_rn(n) & 1) != 0;
  if (r > half || (r == half && (lo > 0.f || (lo == 0.f && odd)))) n += 1.f;
  else if (r < -half || (r == -half && (lo < 0.f || (lo == 0.f && odd)))) n -= 1.f;
  n = fminf(fmaxf(n, -7.f), 7.f);
  if (hi != hi) n = 0.f;  // NaN is held as 0
  return static_cast<uint32_t>(__float2int_rn(n) + 8);
}

// One group: 16 values as hi + lo -> scale byte and 16 nibbles (dim i in nibble i).
__device__ __forceinline__ uint32_t kv4_quantise(const float (&hi)[16], const float (&lo)[16], uint2& codes) {
  float m = 0.f, ml = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float a = fabsf(hi[i]), l = hi[i] < 0.f ? -lo[i] : lo[i];
    if (a > m || (a == m && l > ml)) {
      m = a;
      ml = l;
    }
  }
  const uint32_t b = kv4_scale_byte(m, ml);
  codes = make_uint2(0x88888888u, 0x88888888u);
  if (b != 0) {
    const float s = kv4_scale_value(b), inv = __frcp_rn(s);
    codes = make_uint2(0u, 0u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      codes.x |= kv4_code(hi[i], lo[i], s, inv) << (4 * i);
      codes.y |= kv4_code(hi[8 + i], lo[8 + i], s, inv) << (4 * i);
    }
  }
  return b;
}

// ---- append ------------------------------------------------------------------------
// Thread = (group of 16 dims, slice of the heads): block of 128 threads, d / 16
// groups x 2048 / d slices; blockIdx.x = row, blockIdx.y = batch of heads.
// Heads are numbered q 0.., then k, then v; a thread keeps its 16 dims' angles
// in registers over the heads it walks.
constexpr int kKv4AppendThreads = 128;

template <class T, class TQ>
__global__ void __launch_bounds__(kKv4AppendThreads) kv4_append_kernel(const __grid_constant__ Kv4AppendArgs a,
                                                                       int heads_per_block) {
  pdl_wait();
  pdl_launch();
  const int groups = a.c.d >> 4;
  const int grp = threadIdx.x % groups, slice = threadIdx.x / groups, slices = kKv4AppendThreads / groups;
  const int row = blockIdx.x, i0 = grp * 16;
  const int nq = a.q != nullptr ? a.n_heads : 0, total = nq + 2 * a.c.n_kv;
  const int pos = a.pos[row];
  if (pos < 0) return;  // idle row
  const int sid = a.seq != nullptr ? a.seq[row] : row;
  if (a.cos != nullptr && pos >= a.max_pos) {
    if (threadIdx.x == 0) kv4_error(a.c.status, kKv4BadPos);
    return;
  }
  const int half = a.rotary >> 1;
  const bool rotate = a.cos != nullptr && i0 < a.rotary;
  const bool blocks = (half & 7) == 0;  // a block of 8 dims has its partners in one block of 8
  float c[16], s[16];  // out[i] = x[i] c[i] + partner[i] s[i]
  if (rotate) {
    const float* cr = a.cos + static_cast<int64_t>(pos) * half;
    const float* sr = a.sin + static_cast<int64_t>(pos) * half;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int dim = i0 + i;
      c[i] = 1.f;
      s[i] = 0.f;
      if (dim < a.rotary) {
        const int f = a.interleaved ? dim >> 1 : dim < half ? dim : dim - half;
        const bool first = a.interleaved ? (dim & 1) == 0 : dim < half;
        c[i] = __ldg(cr + f);
        s[i] = first ? -__ldg(sr + f) : __ldg(sr + f);
      }
    }
  }
  const bool qvec = aligned16(a.q, a.q_row, a.q_head, sizeof(T)), kvec = aligned16(a.k, a.k_row, a.k_head, sizeof(T));
  const bool vvec = aligned16(a.v, a.v_row, a.v_head, sizeof(T));
  const bool ovec = aligned16(a.q_out, a.qo_row, a.qo_head, sizeof(TQ));
  const int lo_h = blockIdx.y * heads_per_block, hi_h = min(total, lo_h + heads_per_block);
  for (int hh = lo_h + slice; hh < hi_h; hh += slices) {
    const int kind = hh < nq ? 0 : hh < nq + a.c.n_kv ? 1 : 2;  // q, k, v
    const int g = kind == 0 ? hh : kind == 1 ? hh - nq : hh - nq - a.c.n_kv;
    const T* x = kind == 0   ? static_cast<const T*>(a.q) + row * a.q_row + g * a.q_head
                 : kind == 1 ? static_cast<const T*>(a.k) + row * a.k_row + g * a.k_head
                             : static_cast<const T*>(a.v) + row * a.v_row + g * a.v_head;
    const bool vec = kind == 0 ? qvec : kind == 1 ? kvec : vvec;
    float hi[16], lo[16];
    load8(x + i0, hi, vec);
    load8(x + i0 + 8, hi + 8, vec);
#pragma unroll
    for (int i = 0; i < 16; ++i) lo[i] = 0.f;
    if (rotate && kind != 2) {
      float y[16];  // partners
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = hi[i ^ 1];
      } else if (blocks) {
#pragma unroll
        for (int b = 0; b < 16; b += 8) {
          const int dim = i0 + b;
          load8(x + (dim < half ? dim + half : dim < a.rotary ? dim - half : dim), y + b, vec);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int dim = i0 + i;
          y[i] = to_f32(x[dim < half ? dim + half : dim < a.rotary ? dim - half : dim]);
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (i0 + i >= a.rotary) continue;
        if (kind == 1) {
          rotate_pair(hi[i], c[i], y[i], s[i], hi[i], lo[i]);
        } else {
          hi[i] = fmaf(hi[i], c[i], y[i] * s[i]);
        }
      }
    }
    if (kind == 0) {
      // q_out may be q: the head's threads (one warp's) have read their partners
      __syncwarp(((1u << groups) - 1u) << ((threadIdx.x & 31) / groups * groups));
      TQ* o = static_cast<TQ*>(a.q_out) + row * a.qo_row + g * a.qo_head + i0;
      store8(o, hi, ovec);
      store8(o + 8, hi + 8, ovec);
      continue;
    }
    uint8_t* page = kv4_page(a.c, sid, pos, g);
    if (page == nullptr) continue;
    const int r = pos % kKv4Page;
    uint2 codes;
    const uint32_t b = kv4_quantise(hi, lo, codes);
    if (kind == 1) {
      *reinterpret_cast<uint2*>(page + kv4_k_code(grp, r)) = codes;
      page[kv4_k_scale(a.c.d, grp, r)] = static_cast<uint8_t>(b);
    } else {
      const uint32_t w[4] = {codes.x & 0xFFFFu, codes.x >> 16, codes.y & 0xFFFFu, codes.y >> 16};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint16_t*>(page + kv4_v_code(a.c.d, 4 * grp + i, r)) = static_cast<uint16_t>(w[i]);
      page[kv4_v_scale(a.c.d, grp, r)] = static_cast<uint8_t>(b);
    }
  }
}

// ---- read --------------------------------------------------------------------------
// Rows out of the cache as values (zeros where the position is negative or the
// table names no page).  Thread = (row, kv head, K or V, group).
template <class T>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4ReadArgs a) {
  const int groups = a.c.d >> 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t per_row = static_cast<int64_t>(a.c.n_kv) * 2 * groups;
  if (i >= a.n_rows * per_row) return;
  const int row = static_cast<int>(i / per_row), rest = static_cast<int>(i % per_row);
  const int g = rest / (2 * groups), kv = rest / groups % 2, grp = rest % groups;
  const int pos = a.pos[row];
  const uint8_t* page = nullptr;
  if (pos >= 0) page = kv4_page(a.c, a.seq != nullptr ? a.seq[row] : row, pos, g);
  float x[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) x[k] = 0.f;
  if (page != nullptr) {
    const int r = pos % kKv4Page;
    uint2 codes;
    uint32_t b;
    if (kv == 0) {
      codes = *reinterpret_cast<const uint2*>(page + kv4_k_code(grp, r));
      b = page[kv4_k_scale(a.c.d, grp, r)];
    } else {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = *reinterpret_cast<const uint16_t*>(page + kv4_v_code(a.c.d, 4 * grp + k, r));
      codes = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
      b = page[kv4_v_scale(a.c.d, grp, r)];
    }
    const float s = kv4_scale_value(b);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      x[k] = s * static_cast<float>(static_cast<int>((codes.x >> (4 * k)) & 15u) - 8);
      x[8 + k] = s * static_cast<float>(static_cast<int>((codes.y >> (4 * k)) & 15u) - 8);
    }
  }
  T* o = static_cast<T*>(kv == 0 ? a.k : a.v) + (static_cast<int64_t>(row) * a.c.n_kv + g) * a.c.d + grp * 16;
  const bool vec = (reinterpret_cast<uintptr_t>(o) & 15u) == 0;
  store8(o, x, vec);
  store8(o + 8, x + 8, vec);
}

// ---- attention -----------------------------------------------------------------------
// S^T = K Q^T and O^T = V^T P^T on m16n8k16: the 16 positions of a page are
// the rows of the first product and the reduction of the second, the query
// columns (row of the sequence, head of the group) its 8 columns, so no
// fragment of the cache is wasted on absent queries.  The held values are
// exact in the operands' type: a nibble becomes 128 + u (bf16) or 1024 + u
// (half) by one logic instruction, and value = scale * (u - 8).

// Operands in bf16: value = (128 + u) s - 136 s, one fma, exact: 136 s has at
// most 8 significant bits and the result at most 7.
struct Kv4Bf16 {
  using T = __nv_bfloat16;
  static constexpr float kPOffset = 0.f;
  // scale pair from the bytes b0 << 8 | b1 << 24: the byte's bits as a bf16 with a
  // tiny exponent (subnormal for b < 8), times 2^112
  static __device__ __forceinline__ uint32_t scale(uint32_t bytes) {
    uint32_t s;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(s) : "r"(bytes >> 4), "r"(0x77807780u));
    return s;
  }
  static __device__ __forceinline__ uint32_t offset(uint32_t s) {
    uint32_t c;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(s), "r"(0xC308C308u));  // -136
    return c;
  }
  static __device__ __forceinline__ uint32_t value(uint32_t w, uint32_t s, uint32_t c) {
    uint32_t v;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(v) : "r"((w & 0x000F000Fu) | 0x43004300u), "r"(s), "r"(c));
    return v;
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_bf16(d, a[0], a[1], a[2], a[3], b0, b1);
  }
};
// Operands in half: 1032 s may exceed the type, so the offset goes first:
// (1024 + u) - 1032, then times s, both exact.
// Probabilities carry a factor 2^15, so that those down to 2^-29 of the row's
// largest keep 11 bits; the sum carries it too.
struct Kv4Half {
  using T = __half;
  static constexpr float kPOffset = 15.f;
  static __device__ __forceinline__ uint32_t scale(uint32_t bytes) { return bytes >> 1; }
  static __device__ __forceinline__ uint32_t offset(uint32_t) { return 0u; }
  static __device__ __forceinline__ uint32_t value(uint32_t w, uint32_t s, uint32_t) {
    uint32_t v;
    asm("{\n\t.reg .b32 u;\n\tsub.rn.f16x2 u, %1, %2;\n\tmul.rn.f16x2 %0, u, %3;\n\t}"
        : "=r"(v) : "r"((w & 0x000F000Fu) | 0x64006400u), "r"(0x64086408u), "r"(s));
    return v;
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

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

constexpr int kKv4Warps = 4;

// Where a tile's work lies: sequence, kv head, tile of query columns, split.
struct Kv4Tile {
  int seq, g, tile, split;
  int r0, rows, len, group;
  __device__ __forceinline__ int cols() const { return rows * group; }
  // positions that column c sees
  __device__ __forceinline__ int limit(int c) const { return min(len, max(0, len - rows + c / group + 1)); }
};

// False when the tile has no columns.  Bad inputs (lengths past the table or
// max_len, rows past n_rows or max_rows) leave rows or len 0 and set the status.
__device__ __forceinline__ bool kv4_tile(const Kv4AttnArgs& a, int u, int cols_per_tile, Kv4Tile& t) {
  t.tile = u % a.tiles;
  u /= a.tiles;
  t.split = u % a.splits;
  u /= a.splits;
  t.g = u % a.c.n_kv;
  t.seq = u / a.c.n_kv;
  t.group = a.n_heads / a.c.n_kv;
  t.r0 = a.q_start != nullptr ? a.q_start[t.seq] : t.seq;
  t.rows = a.q_start != nullptr ? a.q_start[t.seq + 1] - t.r0 : 1;
  if (t.rows <= 0) return false;
  if (t.r0 < 0 || t.rows > a.max_rows || t.rows > a.n_rows - t.r0) {
    if (threadIdx.x == 0) kv4_error(a.c.status, kKv4BadPos);
    return false;
  }
  if (t.tile * cols_per_tile >= t.cols()) return false;
  t.len = a.lens[t.seq] + a.len_add;
  if (t.len > a.max_len) {
    if (threadIdx.x == 0) kv4_error(a.c.status, kKv4BadPos);
    t.len = 0;
  }
  if (t.len < 0) t.len = 0;
  return true;
}
// Pages that a tile's columns see, and the splits that have some of them.
__device__ __forceinline__ int kv4_tile_pages(const Kv4Tile& t, int cols_per_tile) {
  const int last = min(t.cols(), (t.tile + 1) * cols_per_tile) - 1;
  return (t.limit(last) + kKv4Page - 1) / kKv4Page;
}

// One CTA of 4 warps per (sequence, kv head, tile of 8 NB query columns, split
// of the positions).  Warp w takes the split's pages w, w + 4, ...; each runs
// its own online softmax, and the four meet in shared memory at the end.
template <class Op, int NH, int NB>
__global__ void __launch_bounds__(32 * kKv4Warps) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
  using T = typename Op::T;
  constexpr int D = 64 * NH, COLS = 8 * NB;
  __shared__ float s_o[kKv4Warps][COLS][D];
  __shared__ float s_m[kKv4Warps][COLS], s_l[kKv4Warps][COLS];
  pdl_wait();
  pdl_launch();
  Kv4Tile tl;
  if (!kv4_tile(a, blockIdx.x, COLS, tl)) return;
  const int pages = kv4_tile_pages(tl, COLS);
  const int lo = tl.split * a.split_pages, hi = min(pages, lo + a.split_pages);
  if (lo >= hi && tl.split > 0) return;  // (the first split always answers)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int c0 = tl.tile * COLS, cols = tl.cols();

  // query fragments: column gid of each block, dims 64h + 16 tig .. in the codes' order
  uint32_t qf[NB][NH][8];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int col = c0 + 8 * nb + gid;
    const bool in = col < cols;
    const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(tl.r0 + (in ? col / tl.group : 0)) * a.q_row +
                 static_cast<int64_t>(tl.g * tl.group + (in ? col % tl.group : 0)) * a.q_head + 16 * tig;
    const bool vec = aligned16(a.q, a.q_row, a.q_head, sizeof(T));
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      __align__(16) T x[16];
      if (!in) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = from_f32<T>(0.f);
      } else if (vec) {
        reinterpret_cast<uint4*>(x)[0] = *reinterpret_cast<const uint4*>(q + 64 * h);
        reinterpret_cast<uint4*>(x)[1] = *reinterpret_cast<const uint4*>(q + 64 * h + 8);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = q[64 * h + i];
      }
      const uint16_t* b = reinterpret_cast<const uint16_t*>(x);
#pragma unroll
      for (int s = 0; s < 4; ++s) {  // k-step s: dims (s, s + 4) and (8 + s, 12 + s) of the 16
        qf[nb][h][2 * s] = b[s] | (static_cast<uint32_t>(b[s + 4]) << 16);
        qf[nb][h][2 * s + 1] = b[8 + s] | (static_cast<uint32_t>(b[12 + s]) << 16);
      }
    }
  }
  // columns 2 tig, 2 tig + 1 of each block: the positions they see
  int lim[NB][2];
  float m[NB][2], l[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = c0 + 8 * nb + 2 * tig + e;
      lim[nb][e] = col < cols ? tl.limit(col) : 0;
      m[nb][e] = -INFINITY;
      l[nb][e] = 0.f;
    }
  const int seen = tl.limit(min(cols, c0 + COLS) - 1);  // positions that any column sees
  float o[NB][4 * NH][4];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int j = 0; j < 4 * NH; ++j) o[nb][j][0] = o[nb][j][1] = o[nb][j][2] = o[nb][j][3] = 0.f;

  const int32_t* table = a.c.table + tl.seq * a.c.table_ld;
  for (int pg = lo + warp; pg < hi; pg += kKv4Warps) {
    const int blk = __ldg(table + pg);
    if (blk < 0 || blk >= a.c.num_blocks) {
      if (lane == 0) kv4_error(a.c.status, kKv4BadTable);
      continue;
    }
    const uint8_t* page = a.c.pool + (static_cast<int64_t>(blk) * a.c.n_kv + tl.g) * kv4_page_bytes(D);
    float sc[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) sc[nb][0] = sc[nb][1] = sc[nb][2] = sc[nb][3] = 0.f;
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const uint4 kc = __ldg(reinterpret_cast<const uint4*>(page) + h * 32 + lane);
      const uint32_t kb = __ldg(reinterpret_cast<const uint16_t*>(page + 8 * D) + h * 32 + lane);
      const uint32_t s0 = Op::scale(__byte_perm(kb, 0u, 0x0404)), s1 = Op::scale(__byte_perm(kb, 0u, 0x1414));
      const uint32_t f0 = Op::offset(s0), f1 = Op::offset(s1);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint32_t k[4] = {Op::value(kc.x >> (4 * s), s0, f0), Op::value(kc.z >> (4 * s), s1, f1),
                               Op::value(kc.y >> (4 * s), s0, f0), Op::value(kc.w >> (4 * s), s1, f1)};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) Op::mma(sc[nb], k, qf[nb][h][2 * s], qf[nb][h][2 * s + 1]);
      }
    }
    // softmax of the page's 16 positions: rows gid (c0, c1) and gid + 8 (c2, c3)
    uint32_t pf[NB][2];
    const int p0 = pg * kKv4Page + gid;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float x[4], al[2];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = p0 + 8 * (i >> 1) < lim[nb][i & 1] ? sc[nb][i] * a.scale_log2 : -INFINITY;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(x[e], x[2 + e]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(m[nb][e], mx), ref = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: all zero
        al[e] = exp2_fast(m[nb][e] - ref);
        m[nb][e] = mn;
        x[e] = exp2_fast(x[e] - ref + Op::kPOffset);
        x[2 + e] = exp2_fast(x[2 + e] - ref + Op::kPOffset);
        l[nb][e] = fmaf(l[nb][e], al[e], x[e] + x[2 + e]);
      }
      pf[nb][0] = transpose8x8(Op::pack(x[0], x[1]));
      pf[nb][1] = transpose8x8(Op::pack(x[2], x[3]));
#pragma unroll
      for (int j = 0; j < 4 * NH; ++j) {
        o[nb][j][0] *= al[0];
        o[nb][j][1] *= al[1];
        o[nb][j][2] *= al[0];
        o[nb][j][3] *= al[1];
      }
    }
    // positions past the last one seen may never have been written: their V
    // scales are dropped, since 0 times an infinity or a NaN is not 0
    uint32_t keep = 0xFFFFFFFFu;
    const int left = seen - pg * kKv4Page;
    if (left < kKv4Page) {
      keep = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (2 * tig + 8 * (i >> 1) + (i & 1) < left) keep |= 0xFFu << (8 * i);
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const uint4 vc = __ldg(reinterpret_cast<const uint4*>(page + 9 * D) + h * 32 + lane);
      const uint32_t vb =
          __ldg(reinterpret_cast<const uint32_t*>(page + 17 * D) + (h * 4 + (gid >> 1)) * 4 + tig) & keep;
      const uint32_t s0 = Op::scale(__byte_perm(vb, 0u, 0x1404)), s1 = Op::scale(__byte_perm(vb, 0u, 0x3424));
      const uint32_t f0 = Op::offset(s0), f1 = Op::offset(s1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // dims 2j (row gid) and 2j + 1 (row gid + 8) of the lane's 8
        const uint32_t w0 = j < 2 ? vc.x : vc.y, w1 = j < 2 ? vc.z : vc.w;
        const int sh = 8 * (j & 1);
        const uint32_t v[4] = {Op::value(w0 >> sh, s0, f0), Op::value(w0 >> (sh + 4), s0, f0),
                               Op::value(w1 >> sh, s1, f1), Op::value(w1 >> (sh + 4), s1, f1)};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) Op::mma(o[nb][4 * h + j], v, pf[nb][0], pf[nb][1]);
      }
    }
  }

  // the warps' states to shared memory: column 2 tig + e, dims 64h + 8 gid ..
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float s = l[nb][e];
      s += __shfl_xor_sync(0xffffffffu, s, 4);
      s += __shfl_xor_sync(0xffffffffu, s, 8);
      s += __shfl_xor_sync(0xffffffffu, s, 16);
      const int col = 8 * nb + 2 * tig + e;
      if (gid == 0) {
        s_m[warp][col] = m[nb][e];
        s_l[warp][col] = s;
      }
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        float4* dst = reinterpret_cast<float4*>(&s_o[warp][col][64 * h + 8 * gid]);
        dst[0] = make_float4(o[nb][4 * h][e], o[nb][4 * h][2 + e], o[nb][4 * h + 1][e], o[nb][4 * h + 1][2 + e]);
        dst[1] = make_float4(o[nb][4 * h + 2][e], o[nb][4 * h + 2][2 + e], o[nb][4 * h + 3][e], o[nb][4 * h + 3][2 + e]);
      }
    }
  __syncthreads();
  const int64_t unit = (static_cast<int64_t>(tl.seq) * a.c.n_kv + tl.g) * a.tiles + tl.tile;
  const bool ovec = aligned16(a.out, a.o_row, a.o_head, sizeof(T));
  for (int i = threadIdx.x; i < COLS * (D / 8); i += 32 * kKv4Warps) {
    const int col = i / (D / 8), d0 = i % (D / 8) * 8;
    if (c0 + col >= cols) break;
    float M = s_m[0][col], L = 0.f, r[8];
#pragma unroll
    for (int w = 1; w < kKv4Warps; ++w) M = fmaxf(M, s_m[w][col]);
#pragma unroll
    for (int k = 0; k < 8; ++k) r[k] = 0.f;
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < kKv4Warps; ++w) {
      const float f = exp2_fast(s_m[w][col] - ref);
      L = fmaf(f, s_l[w][col], L);
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = fmaf(f, s_o[w][col][d0 + k], r[k]);
    }
    if (a.splits == 1) {
      const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);  // a row that sees nothing: zeros (NaN stays NaN)
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] *= inv;
      const int c = c0 + col;
      store8(static_cast<T*>(a.out) + static_cast<int64_t>(tl.r0 + c / tl.group) * a.o_row +
                 static_cast<int64_t>(tl.g * tl.group + c % tl.group) * a.o_head + d0,
             r, ovec);
    } else {
      float* dst = a.part + ((unit * a.splits + tl.split) * COLS + col) * (D + 4);
      *reinterpret_cast<float4*>(dst + d0) = make_float4(r[0], r[1], r[2], r[3]);
      *reinterpret_cast<float4*>(dst + d0 + 4) = make_float4(r[4], r[5], r[6], r[7]);
      if (d0 == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(M, L);
    }
  }
}

// Joins the splits of each column, in split order: one warp per column.
template <class Op, int NH, int NB>
__global__ void __launch_bounds__(256) kv4_join_kernel(const __grid_constant__ Kv4AttnArgs a) {
  using T = typename Op::T;
  constexpr int D = 64 * NH, COLS = 8 * NB, PER = D / 32;
  pdl_wait();
  pdl_launch();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, col = static_cast<int>(i % COLS);
  const int64_t unit = i / COLS;
  if (unit >= static_cast<int64_t>(a.n_seqs) * a.c.n_kv * a.tiles) return;
  Kv4Tile tl;
  // the unit's first split, in the numbering of the attention kernel's CTAs
  const int tile = static_cast<int>(unit % a.tiles);
  if (!kv4_tile(a, static_cast<int>((unit / a.tiles) * a.splits * a.tiles + tile), COLS, tl)) return;
  const int c = tl.tile * COLS + col;
  if (c >= tl.cols()) return;
  const int n = max(1, (kv4_tile_pages(tl, COLS) + a.split_pages - 1) / a.split_pages);
  const float* src = a.part + (unit * a.splits * COLS + col) * (D + 4);
  const int64_t step = static_cast<int64_t>(COLS) * (D + 4);
  float M = -INFINITY;
  for (int s = lane; s < n; s += 32) M = fmaxf(M, src[s * step + D]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f, r[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) r[k] = 0.f;
  for (int s = 0; s < n; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(src + s * step + D);
    const float f = exp2_fast(ml.x - ref);
    L = fmaf(f, ml.y, L);
#pragma unroll
    for (int k = 0; k < PER; ++k) r[k] = fmaf(f, src[s * step + lane + 32 * k], r[k]);
  }
  const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);
  T* out = static_cast<T*>(a.out) + static_cast<int64_t>(tl.r0 + c / tl.group) * a.o_row +
           static_cast<int64_t>(tl.g * tl.group + c % tl.group) * a.o_head;
#pragma unroll
  for (int k = 0; k < PER; ++k) out[lane + 32 * k] = from_f32<T>(r[k] * inv);
}

}  // namespace b2d

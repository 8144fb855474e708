// kv4_prompt.cuh — attention of many query columns over the 4-bit cache on the
// 5th-generation tensor cores (tcgen05, sm_100a).
//
// One CTA of 128 threads takes 128 query columns (row of the sequence, head of
// the group) of a (sequence, kv head) through tiles of 128 positions:
//   S = Q K^T   M = 128 columns, N = 128 positions, K = d; Q and K in shared memory
//   O += P V    M = 128 columns, N = d, K = 128 positions; P in tensor memory, V
//               in shared memory
// with the halves of kv4.cuh (held values, queries and scores exact, P with 11
// bits and a factor 2^10).  Thread r owns column r: lane r of tensor memory.
//
// The four warps turn two pages each from codes to halves, straight into the
// swizzled operands.  The orders are chosen so that a lane's fragments lie
// together (16 and 8 byte stores without bank conflicts): the dims of K and Q
// are permuted alike within each 16, the positions of a page alike in S, P and
// V, and the dims of V, which are O's columns, are put back on the way out.
// The first product runs while V is turned, the second while the next K is;
// the other CTA of the SM (two fit: 256 columns of tensor memory each) fills
// the waits.
//
// Column r's running maximum is only moved, and O rescaled, when the scores
// exceed it by 2^5 or more: P then stays below 2^15, and those down to 2^-24 of
// the largest keep their 11 bits.
#pragma once

#include <type_traits>

#include "kv4.cuh"
#include "tc_ptx.cuh"

namespace b2d {

constexpr int kKv4PromptCols = 128;  // query columns of a CTA
constexpr int kKv4PromptKeys = 128;  // positions of a tile
constexpr float kKv4PromptOffset = 10.f, kKv4PromptSlack = 5.f;  // (their sum: P below 2^15)
constexpr uint32_t kKv4PromptTmem = 256;  // columns: S (P over it) 128, O d
template <int NH>
constexpr __host__ __device__ int kv4_prompt_smem() {
  // Q, K, V tiles and 1 KB to align; at least 80 KB, so that no more than two CTAs
  // share an SM's tensor memory (a third would wait for it)
  constexpr int tiles = 3 * NH * 128 * 128 + 1024;
  return tiles > 80 * 1024 ? tiles : 80 * 1024;
}

// f16 x f16 -> f32, both operands K-major.
__host__ __device__ constexpr uint32_t idesc_f16_f32(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
// One thread: D[tmem] (+)= A[tmem] * B[smem]^T.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                              bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
// Whole warp: 32 consecutive columns of its 32 lanes, without waiting.
__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t* r) {
  tmem_store16(taddr, r);
  tmem_store16(taddr + 16, r + 16);
}

// Column k of a page's 16 in S, P and V's reduction <-> slot of the page: the
// four slots of a lane lie together.
__host__ __device__ constexpr int kv4_slot(int k) { return 8 * ((k >> 1) & 1) + 2 * (k >> 2) + (k & 1); }
// Row n of V's operand (column of O) within 64 dims: dim 8 g + i is row 8 i + perm(g).
__host__ __device__ constexpr int kv4_perm(int g) { return ((g << 1) & 7) | (g >> 2); }

// One page of this lane's fragments as it is loaded.
template <int NH>
struct Kv4Frag {
  uint4 code[NH];
  uint32_t scale[NH];
};

template <class T, int NH>
__global__ void __launch_bounds__(128) kv4_prompt_kernel(const __grid_constant__ Kv4AttnArgs a) {
  constexpr int D = 64 * NH, PB = kv4_page_bytes(D), PAGES = kKv4PromptKeys / kKv4Page;
  extern __shared__ uint8_t kv4_prompt_raw[];
  __shared__ uint64_t s_bar[2];  // S done, O done
  __shared__ uint32_t s_tmem;
  __shared__ volatile uint32_t s_fail;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
  uint8_t* sq = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(kv4_prompt_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sk = sq + NH * 128 * 128;  // [NH][128 rows][128 B] each
  uint8_t* sv = sk + NH * 128 * 128;  // [2][D rows][128 B]
  pdl_wait();
  Kv4Tile tl;
  const bool work = kv4_tile(a, blockIdx.z, tl);
  const int pages = work ? kv4_tile_pages(a, tl) : 0;
  const int lo = tl.split * a.split_pages, hi = min(pages, lo + a.split_pages);
  if (!work || (lo >= hi && tl.split > 0)) {  // (the first split always answers)
    pdl_launch();
    return;
  }
  if (warp == 0) tmem_alloc(&s_tmem, kKv4PromptTmem);
  if (tid == 0) {
    mbar_init(&s_bar[0], 1);
    mbar_init(&s_bar[1], 1);
    fence_mbar_init();
    s_fail = 0u;
  }
  const int c0 = tl.tile * kKv4PromptCols, cols = tl.cols(a), col = c0 + tid;
  const bool in = col < cols;
  const int row = in && tl.rows > 1 ? kv4_row(a, col) : 0, head = in ? col - row * a.group : 0;
  const int lim = in ? kv4_limit(a, tl, col) : 0;                          // positions this column sees
  const int seen = kv4_limit(a, tl, min(cols, c0 + kKv4PromptCols) - 1);   // that any does
  const int all_see = kv4_limit(a, tl, c0);                                // that all do

  // ---- the column's query: halves, dims in the codes' order, to row tid of sq ----
  float up = a.scale_log2;
  {
    const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(tl.r0 + row) * a.q_row +
                 static_cast<int64_t>(tl.g * a.group + head) * a.q_head;
    const bool vec = aligned16(a.q, a.q_row, a.q_head, sizeof(T));
    float down = 1.f;
    if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
      uint32_t top = 0;
#pragma unroll
      for (int b = 0; b < D / 16; ++b) {
        uint32_t w[8];
        load16(q + 16 * b, w, in, vec);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t x = w[i] & 0x7F807F80u;
          top = max(top, max(x, x << 16));
        }
      }
      top >>= 23;
      const int e = top == 0 ? 0 : min(static_cast<int>(top), 253) - 127;
      down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      up *= __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    }
#pragma unroll
    for (int b = 0; b < D / 16; ++b) {
      uint32_t w[8], f[8];
      load16(q + 16 * b, w, in, vec);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k) {  // pair s of block k: dims (8k + s, 8k + s + 4)
          const uint32_t x = w[4 * k + (s >> 1)], y = w[4 * k + 2 + (s >> 1)];
          if constexpr (std::is_same<T, __half>::value)
            f[4 * k + s] = __byte_perm(x, y, s & 1 ? 0x7632 : 0x5410);
          else
            f[4 * k + s] = s & 1 ? pack_half2(bf16_hi(x) * down, bf16_hi(y) * down)
                                 : pack_half2(bf16_lo(x) * down, bf16_lo(y) * down);
        }
      uint8_t* dst = sq + (b >> 2) * 16384 + tid * 128;
      const int c = (b & 3) * 2;
      *reinterpret_cast<uint4*>(dst + (((c) ^ (tid & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<uint4*>(dst + (((c + 1) ^ (tid & 7)) << 4)) = make_uint4(f[4], f[5], f[6], f[7]);
    }
  }

  // ---- pages: this warp's two of a tile, K or V part ----
  const int32_t* table = a.c.table + tl.seq * a.c.table_ld;
  const uint8_t* pool = a.c.pool + static_cast<int64_t>(tl.g) * PB;
  const int64_t block_bytes = static_cast<int64_t>(a.c.n_kv) * PB;
  auto page_at = [&](int pg) -> const uint8_t* {  // null: zeros (past the split, or not named by the table)
    if (pg >= hi) return nullptr;
    const int blk = __ldg(table + pg);
    if (blk < 0 || blk >= a.c.num_blocks) {
      if (lane == 0) kv4_error(a.c.status, kKv4BadTable);
      return nullptr;
    }
    return pool + blk * block_bytes;
  };
  Kv4Frag<NH> kf[2], vf[2];
  const uint8_t* next_page[2];
  auto load_k = [&]() {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        kf[p].code[h] = make_uint4(0u, 0u, 0u, 0u);
        kf[p].scale[h] = 0u;
        if (next_page[p] != nullptr) {
          kf[p].code[h] = __ldg(reinterpret_cast<const uint4*>(next_page[p]) + h * 32 + lane);
          kf[p].scale[h] = __ldg(reinterpret_cast<const uint16_t*>(next_page[p] + 8 * D) + h * 32 + lane);
        }
      }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        vf[p].code[h] = make_uint4(0u, 0u, 0u, 0u);
        vf[p].scale[h] = 0u;
        if (next_page[p] != nullptr) {
          vf[p].code[h] = __ldg(reinterpret_cast<const uint4*>(next_page[p] + 9 * D) + h * 32 + lane);
          vf[p].scale[h] = __ldg(reinterpret_cast<const uint32_t*>(next_page[p] + 17 * D) + (h * 4 + (gid >> 1)) * 4 + tig);
        }
      }
  };
  auto find = [&](int tile_page) {
#pragma unroll
    for (int p = 0; p < 2; ++p) next_page[p] = page_at(tile_page + 2 * warp + p);
  };
  // this lane's rows of the K tile: slots gid and gid + 8 of a page are its columns key, key + 2
  const int key = 4 * (gid >> 1) + (gid & 1);
  auto turn_k = [&]() {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int r = 16 * (2 * warp + p) + key;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const uint32_t s0 = kv4_scales(kf[p].scale[h], 0x4040), s1 = kv4_scales(kf[p].scale[h], 0x4141);
        uint32_t v[4];
        uint8_t* d0 = sk + h * 16384 + r * 128;
        uint8_t* d1 = d0 + 2 * 128;
        kv4_values(kf[p].code[h].x, s0, v);
        *reinterpret_cast<uint4*>(d0 + (((2 * tig) ^ (r & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        kv4_values(kf[p].code[h].y, s0, v);
        *reinterpret_cast<uint4*>(d0 + (((2 * tig + 1) ^ (r & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        kv4_values(kf[p].code[h].z, s1, v);
        *reinterpret_cast<uint4*>(d1 + (((2 * tig) ^ ((r + 2) & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        kv4_values(kf[p].code[h].w, s1, v);
        *reinterpret_cast<uint4*>(d1 + (((2 * tig + 1) ^ ((r + 2) & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
      }
    }
  };
  const int vrow = kv4_perm(gid);
  auto turn_v = [&](int tile_page) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int pg = 2 * warp + p;
      // slots past the last position seen may never have been written: no scale
      const int left = seen - (tile_page + pg) * kKv4Page;
      uint32_t keep = 0xFFFFFFFFu;
      if (left < kKv4Page) {
        keep = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (2 * tig + 8 * (i >> 1) + (i & 1) < left) keep |= 0xFFu << (8 * i);
      }
      uint8_t* dst = sv + (pg >> 2) * (D * 128) + vrow * 128 + ((((pg & 3) * 2 + (tig >> 1)) ^ vrow) << 4) + (tig & 1) * 8;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const uint32_t sc = vf[p].scale[h] & keep;
        const uint32_t s0 = kv4_scales(sc, 0x4140), s1 = kv4_scales(sc, 0x4342);
        uint32_t x[4], y[4];
        kv4_values(vf[p].code[h].x, s0, x);
        kv4_values(vf[p].code[h].z, s1, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint2*>(dst + (64 * h + 8 * i) * 128) = make_uint2(x[i], y[i]);
        kv4_values(vf[p].code[h].y, s0, x);
        kv4_values(vf[p].code[h].w, s1, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint2*>(dst + (64 * h + 32 + 8 * i) * 128) = make_uint2(x[i], y[i]);
      }
    }
  };
  // Bounded wait; one that runs out marks the CTA, which then issues no more.
  auto wait = [&](int which, uint32_t parity) {
    if (mbar_test(&s_bar[which], parity) || s_fail) return;
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t i = 1; !mbar_test(&s_bar[which], parity); ++i)
      if ((i & 255u) == 0 && (s_fail || globaltimer_ns() - t0 > kKv4WaitNs)) {
        s_fail = 1u;
        return;
      }
  };

  find(lo);
  load_k();
  load_v();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch();  // (every CTA that runs now holds its tensor memory)
  const uint32_t tmem = s_tmem, t_s = tmem, t_o = tmem + 128;
  const uint32_t t_lane = static_cast<uint32_t>(warp * 32) << 16;
  float m = -INFINITY, l = 0.f;  // maximum of the scores before their scale, as used; sum of p
  const int tiles = (hi - lo + PAGES - 1) / PAGES;

  for (int i = 0; i < tiles; ++i) {
    const int tile_page = lo + i * PAGES;
    turn_k();  // (the last S is done with sk)
    find(tile_page + PAGES);
    load_k();
    if (i > 0) wait(1, static_cast<uint32_t>(i - 1) & 1u);  // O: sv, and P's columns under S
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && !s_fail) {
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        tc_mma_bf16(t_s, sdesc_kmajor_sw128(smem_addr(sq + (k >> 2) * 16384 + (k & 3) * 32)),
                   sdesc_kmajor_sw128(smem_addr(sk + (k >> 2) * 16384 + (k & 3) * 32)), idesc_f16_f32(128, 128), k > 0);
      tc_commit(&s_bar[0]);
    }
    turn_v(tile_page);
    load_v();
    fence_proxy_async_smem();
    wait(0, static_cast<uint32_t>(i) & 1u);
    tc_fence_after();

    // ---- softmax of this column's 128 scores ----
    uint32_t s[128];
#pragma unroll
    for (int c = 0; c < 4; ++c) tmem_load32(t_s + t_lane + 32 * c, s + 32 * c);
    tmem_wait_ld();
    const int at = tile_page * kKv4Page;
    if (at + kKv4PromptKeys > all_see || tile_page + PAGES > hi) {
      const int left = min(lim, hi * kKv4Page) - at;
#pragma unroll
      for (int c = 0; c < 128; ++c)
        if (16 * (c >> 4) + kv4_slot(c & 15) >= left) s[c] = 0xFF800000u;  // -infinity
    }
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < 128; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(s[c]));
    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
    const bool grows = (top - m) * up > kKv4PromptSlack;  // (from -infinity too; not for a column that sees nothing)
    if (__any_sync(0xffffffffu, grows)) {
      const float mn = fmaxf(m, top);
      const float f = mn == -INFINITY ? 0.f : exp2_fast((m - mn) * up);
      m = mn;
      l *= f;
      if (i > 0) {
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_load32(t_o + t_lane + c, o);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
          tmem_store32(t_o + t_lane + c, o);
        }
      }
    }
    const float sub = fmaf(m == -INFINITY ? 0.f : -m, up, kKv4PromptOffset);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 128; c += 32) {
      uint32_t p[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float x = exp2_fast(fmaf(__uint_as_float(s[c + 2 * k]), up, sub));
        const float y = exp2_fast(fmaf(__uint_as_float(s[c + 2 * k + 1]), up, sub));
        sum[k & 3] += x + y;
        p[k] = pack_half2(x, y);
      }
      tmem_store16(t_s + t_lane + (c >> 1), p);
    }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    tmem_wait_st();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && !s_fail) {
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < kKv4PromptKeys / 16; ++k)
        tc_mma_f16_ts(t_o, t_s + 8 * k, sdesc_kmajor_sw128(smem_addr(sv + (k >> 2) * (D * 128) + (k & 3) * 32)),
                      idesc_f16_f32(128, D), i > 0 || k > 0);
      tc_commit(&s_bar[1]);
    }
  }
  if (tiles > 0) wait(1, static_cast<uint32_t>(tiles - 1) & 1u);
  tc_fence_after();

  // ---- the column's result ----
  const bool ovec = aligned16(a.out, a.o_row, a.o_head, sizeof(T));
  const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);  // a column that sees nothing: zeros (NaN stays NaN)
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    uint32_t o[64];
    if (tiles > 0) {
      tmem_load32(t_o + t_lane + 64 * h, o);
      tmem_load32(t_o + t_lane + 64 * h + 32, o + 32);
      tmem_wait_ld();
    } else {
#pragma unroll
      for (int k = 0; k < 64; ++k) o[k] = 0u;
    }
    if (!in) continue;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      float r[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = __uint_as_float(o[8 * k + kv4_perm(g)]);
      if (a.splits == 1) {
#pragma unroll
        for (int k = 0; k < 8; ++k) r[k] = l == 0.f ? 0.f : r[k] * inv;
        store8(static_cast<T*>(a.out) + static_cast<int64_t>(tl.r0 + row) * a.o_row +
                   static_cast<int64_t>(tl.g * a.group + head) * a.o_head + 64 * h + 8 * g,
               r, ovec);
      } else {
        float* dst = kv4_part(a, tl.seq, tl.g, tl.tile, tl.split, tid, D) + 64 * h + 8 * g;
        *reinterpret_cast<float4*>(dst) = make_float4(r[0], r[1], r[2], r[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(r[4], r[5], r[6], r[7]);
      }
    }
  }
  if (in && a.splits > 1)
    *reinterpret_cast<float2*>(kv4_part(a, tl.seq, tl.g, tl.tile, tl.split, tid, D) + D) = make_float2(m * up, l);
  if (s_fail) {
    if (tid == 0) kv4_error(a.c.status, kKv4Timeout);
    // what was issued may still be running: once more, for the last of each
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < kKv4WaitNs &&
           !(mbar_test(&s_bar[0], static_cast<uint32_t>(tiles - 1) & 1u) && mbar_test(&s_bar[1], static_cast<uint32_t>(tiles - 1) & 1u))) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, kKv4PromptTmem);
}

}  // namespace b2d

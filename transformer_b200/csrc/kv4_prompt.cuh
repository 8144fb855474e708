// kv4_prompt.cuh — attention of many query columns over the 4-bit cache on the
// 5th-generation tensor cores (tcgen05, sm_100a).
//
// One CTA takes one or two groups of 128 query columns (row of the sequence, head
// of the group) of a (sequence, kv head) through tiles of 64 positions; for each
// group
//   S = Q K^T   M = 128 columns, N = 64 positions, K = d; Q and K in shared memory
//   O += P V    M = 128 columns, N = d, K = 64 positions; P in tensor memory, V in
//               shared memory
// with the operands of kv4.cuh (held values and queries exact, S in the queries'
// type, P with 11 bits and a factor 2^10).  Its warps have parts, which meet only
// on mbarriers (for two groups):
//   warps 0-7    softmax: thread r owns column r, lane r % 128 of its group's
//                tensor memory
//   warps 8-11   turn K's codes to values, a page of each tile, straight into the
//                swizzled operand
//   warps 12-15  V's
//   warps 16-17  issue a group's products
// K, V and S (with P over it) have two buffers each: S of the next tile is made
// during the softmax of this one, O of the last one too.  One CTA to an SM.
//
// 4 chunks of 128 to 512 rows on 2049 to 8191 positions, 32 heads over 8 of 128
// dims (125 GFLOP): 153 us, 816 TFLOP/s; 288 tiles of equal length 151 us, 950.
// What bounds the latter: per tile and group the softmax has 512 cycles of
// exponentials on a quarter SM, next to 280 of its other instructions and as many
// for the codes; both products take 512 of the tensor cores (before differences
// and waits were made safe, 147 us: without the exponentials 130, without the codes
// 141, without most of the products 145).  The 4 chunks lose another 20% to the
// longest columns' end.  Measured on the same case when it took 147: two CTAs to
// an SM of one group, 205; four warps for K and V
// together, 166; all 64 scores held at once, 155; one pass with the last
// maximum that is repeated when that was too small, 158; waits that poll, 147.
// Before the longest came first, 274: tiles of 128 positions with one buffer 296
// to 318; all warps sharing softmax and codes 329.
//
// The orders are chosen so that a lane's fragments lie together (16 and 8 byte
// stores without bank conflicts): the dims of K and Q are permuted alike within
// each 16, the positions of a page alike in S, P and V, and the dims of V, which
// are O's columns, are put back on the way out.
//
// The softmax is the published online one (Milakov and Gimelshein, 2018) with a
// maximum that may lag, as others have published since: it is only moved, and O
// rescaled, when scores exceed it by 2^5 or more.  P then stays below 2^15, and
// those down to 2^-24 of the largest keep their 11 bits.
#pragma once

#include <climits>

#include "kv4.cuh"
#include "tc_ptx.cuh"

namespace b2d {

constexpr int kKv4PromptCols = 128;  // query columns of a group; a CTA has one or two
constexpr int kKv4PromptKeys = 64;   // positions of a tile
template <int NG>
constexpr __host__ __device__ int kv4_prompt_threads() {
  return 32 * (4 * NG + 4 + 4 + 2);
}
constexpr float kKv4PromptOffset = 10.f, kKv4PromptSlack = 5.f;  // (their sum: P below 2^15)
constexpr uint32_t kKv4PromptTmem = 256;  // columns of a group: S (P over it) 2 x 64, O d
template <int NH, int NG>
constexpr __host__ __device__ int kv4_prompt_smem() {
  // Q, K, V tiles and 1 KB to align; at least so much that no more groups than two
  // share an SM's tensor memory (a third would wait for it)
  constexpr int tiles = (NG + 2) * NH * 128 * 128 + 1024, least = (NG == 1 ? 80 : 120) * 1024;
  return tiles > least ? tiles : least;
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
// Two floats at once.
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ float2 floats_of(uint64_t x) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(x));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return d;
}
__device__ __forceinline__ bool elect_one() {  // of a whole warp: true in one lane
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
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
__device__ __forceinline__ void tmem_load16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15])
      : "r"(taddr));
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

// The sequence that is rank-th from the longest (equal lengths in their order):
// the longest tiles start first, so that short ones fill the end (4 chunks as
// above: 205 us, and 274 in the sequences' order).  Whole warp.  More than 32 sequences stay in
// their order: with so many tiles the last ones are a small part.
__device__ __forceinline__ int kv4_seq_of_rank(const Kv4AttnArgs& a, int rank) {
  if (a.n_seqs > 32 || a.n_seqs == 1) return rank;
  const int lane = threadIdx.x & 31;
  const int len = lane < a.n_seqs ? __ldg(a.lens + lane) : INT_MIN;
  int before = 0;
  for (int i = 0; i < a.n_seqs; ++i) {
    const int other = __shfl_sync(0xffffffffu, len, i);
    before += other > len || (other == len && i < lane);
  }
  return __ffs(__ballot_sync(0xffffffffu, lane < a.n_seqs && before == rank)) - 1;
}

// Grid: x = (rank * kv heads + kv head) * tiles + tile from the last, y = split.
template <class T, int NH, int NG>
__global__ void __launch_bounds__(kv4_prompt_threads<NG>(), 1) kv4_prompt_kernel(const __grid_constant__ Kv4AttnArgs a) {
  constexpr int D = 64 * NH, PB = kv4_page_bytes(D), PAGES = kKv4PromptKeys / kKv4Page;
  extern __shared__ uint8_t kv4_prompt_raw[];
  // written: K, V; of each group, written: P, products done: S (so K is free), O (so V
  // and P's S are); two buffers each
  enum { kKFull, kVFull, kPFull, kSDone = kPFull + NG, kODone = kSDone + NG, kBars = kODone + NG };
  __shared__ uint64_t s_bar[kBars][2];
  __shared__ uint32_t s_tmem;
  __shared__ volatile uint32_t s_fail;
  __shared__ int s_lost;  // the first page that the table does not name
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
  uint8_t* sq = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(kv4_prompt_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sk = sq + NG * NH * 128 * 128;  // Q [NG][NH][128 rows][128 B], K [2][NH][64 rows][128 B]
  uint8_t* sv = sk + NH * 128 * 128;  // V [2][D rows][128 B]
  constexpr int K_BUF = NH * 64 * 128, V_BUF = D * 128;
  pdl_wait();
  Kv4Tile tl;
  const unsigned unit = blockIdx.x / a.tiles, rank = unit / a.c.n_kv;
  const bool work = kv4_tile(a, kv4_seq_of_rank(a, rank), unit - rank * a.c.n_kv,
                             a.tiles - 1 - static_cast<int>(blockIdx.x - unit * a.tiles), blockIdx.y, tl);
  const int pages = work ? kv4_tile_pages(a, tl) : 0;
  const int lo = tl.split * a.split_pages, hi = min(pages, lo + a.split_pages);
  if (!work || (lo >= hi && tl.split > 0)) {  // (the first split always answers)
    pdl_launch();
    return;
  }
  constexpr int CODES = 4 * NG, ISSUE = CODES + 8;  // the parts' first warps
  if (warp == ISSUE) tmem_alloc(&s_tmem, NG * kKv4PromptTmem);
  if (tid == 0) {
    for (int i = 0; i < 2 * kBars; ++i) mbar_init(&s_bar[i >> 1][i & 1], i < 2 * kSDone ? 4 : 1);  // 4 warps, or a commit
    fence_mbar_init();
    s_fail = 0u;
    s_lost = INT_MAX;
  }
  const int c0 = tl.tile * NG * kKv4PromptCols, cols = tl.cols(a), tiles = (hi - lo + PAGES - 1) / PAGES;
  // Bounded wait for a barrier's phase of tile i; one that runs out marks the
  // CTA, whose parts then leave their loops, a warp's lanes together (the votes:
  // 151 us, not 148, on the 4 chunks).
  auto wait = [&](int which, int i) {
    if (__all_sync(0xffffffffu, kv4_wait(&s_bar[which][i & 1], static_cast<uint32_t>(i >> 1) & 1u))) return true;
    s_fail = 1u;
    return false;
  };

  // ---- softmax threads: the column and its query ----
  const int groups = min(NG, (cols - c0 + kKv4PromptCols - 1) / kKv4PromptCols);
  const int col = c0 + tid, gr = warp >> 2;
  const bool in = warp < CODES && col < cols;
  const int row = in && tl.rows > 1 ? kv4_row(a, col) : 0, head = in ? col - row * a.group : 0;
  const float up = a.scale_log2;
  if (warp < CODES) {
    // dims in the codes' order, to row tid of its group's Q
    const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(tl.r0 + row) * a.q_row +
                 static_cast<int64_t>(tl.g * a.group + head) * a.q_head;
    const bool vec = aligned16(a.q, a.q_row, a.q_head, sizeof(T));
#pragma unroll
    for (int b = 0; b < D / 16; ++b) {
      uint32_t w[8], f[8];
      load16(q + 16 * b, w, in, vec);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k) {  // pair s of block k: dims (8k + s, 8k + s + 4)
          const uint32_t x = w[4 * k + (s >> 1)], y = w[4 * k + 2 + (s >> 1)];
          f[4 * k + s] = __byte_perm(x, y, s & 1 ? 0x7632 : 0x5410);
        }
      uint8_t* dst = sq + (gr * NH + (b >> 2)) * 16384 + (tid & 127) * 128;
      const int c = (b & 3) * 2;
      *reinterpret_cast<uint4*>(dst + ((c ^ (tid & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<uint4*>(dst + (((c + 1) ^ (tid & 7)) << 4)) = make_uint4(f[4], f[5], f[6], f[7]);
    }
  }

  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch();  // (every CTA that runs now holds its tensor memory)
  // this group's tensor memory (groups of the issuing warps: below)
  auto t_s_of = [&](int g) { return s_tmem + 128 * g; };
  auto t_o_of = [&](int g) { return s_tmem + 128 * NG + D * g; };

  if (warp >= ISSUE) {  // ---- products: a warp a group ----
    // (the whole warp walks along, so that descriptors stay in uniform registers)
    const int g = warp - ISSUE;
    const uint32_t t_s = t_s_of(g), t_o = t_o_of(g);
    const bool leader = elect_one();
    const uint32_t q0 = smem_addr(sq) + g * NH * 16384, k0 = smem_addr(sk), v0 = smem_addr(sv);
    auto poll = [&](int which, int i) {
      if (__all_sync(0xffffffffu, kv4_poll(&s_bar[which][i & 1], static_cast<uint32_t>(i >> 1) & 1u))) return true;
      s_fail = 1u;
      return false;
    };
    auto issue_s = [&](int i) {
      if (!poll(kKFull, i) || (i >= 2 && !poll(kODone + g, i - 2))) return false;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint64_t qd = sdesc_kmajor_sw128(q0 + (k >> 2) * 16384 + (k & 3) * 32);
        const uint64_t kd = sdesc_kmajor_sw128(k0 + (i & 1) * K_BUF + (k >> 2) * 8192 + (k & 3) * 32);
        constexpr uint32_t idesc = std::is_same<T, __half>::value ? idesc_f16_f32(128, 64) : idesc_bf16_f32(128, 64);
        if (leader) tc_mma_bf16(t_s + 64 * (i & 1), qd, kd, idesc, k > 0);  // (the type is the descriptor's)
      }
      if (leader) tc_commit(&s_bar[kSDone + g][i & 1]);
      return true;
    };
    bool ok = g < groups && tiles > 0 && issue_s(0);
    for (int i = 0; ok && i < tiles; ++i) {
      if (i + 1 < tiles) ok = issue_s(i + 1);
      ok = ok && poll(kVFull, i) && poll(kPFull + g, i);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < kKv4PromptKeys / 16; ++k) {
        const uint64_t vd = sdesc_kmajor_sw128(v0 + (i & 1) * V_BUF + k * 32);
        if (leader) tc_mma_f16_ts(t_o, t_s + 64 * (i & 1) + 8 * k, vd, idesc_f16_f32(128, D), i > 0 || k > 0);
      }
      if (leader) tc_commit(&s_bar[kODone + g][i & 1]);
    }
  } else if (warp >= CODES) {  // ---- codes to values ----
    const int32_t* table = a.c.table + tl.seq * a.c.table_ld;
    const uint8_t* pool = a.c.pool + static_cast<int64_t>(tl.g) * PB;
    const int64_t block_bytes = static_cast<int64_t>(a.c.n_kv) * PB;
    const int mine = warp & 3;  // this warp's page of a tile
    // the block of this warp's page of tile i, as the table has it
    auto block_of = [&](int i) {
      const int pg = lo + i * PAGES + mine;
      return pg < hi ? __ldg(table + pg) : -1;
    };
    // null: zeros (past the split, or not named by the table)
    auto page_at = [&](int i, int blk) -> const uint8_t* {
      if (kv4_named(a.c, blk)) return pool + blk * block_bytes;
      if (lane == 0 && lo + i * PAGES + mine < hi) {
        atomicMin(&s_lost, lo + i * PAGES + mine);  // (before the tile's K: softmax threads look at their end)
        kv4_error(a.c.status, kKv4BadTable);
      }
      return nullptr;
    };
    // Tile i, whose page is in f; f takes tile i + 2's, so that a load has a tile's
    // time to arrive (block: its number in the pool, loaded a tile before).
    int block = block_of(2);
    Kv4Frag<NH> frag[2];
    auto walk = [&](auto&& load, auto&& convert) {
#pragma unroll
      for (int i = 0; i < 2; ++i) load(frag[i], page_at(i, block_of(i)));
      auto one = [&](int i, Kv4Frag<NH>& f) {
        if (!convert(i, f)) return false;
        const uint8_t* page = page_at(i + 2, block);
        block = block_of(i + 3);
        load(f, page);
        return true;
      };
      for (int i = 0; i < tiles; i += 2)
        if (!one(i, frag[0]) || (i + 1 < tiles && !one(i + 1, frag[1]))) break;
    };
    // the tile's buffer is written: for the products, and told by one lane
    auto written = [&](int which, int i) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_bar[which][i & 1]);
    };
    if (warp < CODES + 4) {
      // this lane's rows of the K tile: slots gid and gid + 8 of a page are its columns r, r + 2
      const int r = 16 * mine + 4 * (gid >> 1) + (gid & 1);
      uint8_t* const k_to = sk + r * 128;
      walk(
          [&](Kv4Frag<NH>& kf, const uint8_t* page) {
#pragma unroll
            for (int h = 0; h < NH; ++h) {
              kf.code[h] = make_uint4(0u, 0u, 0u, 0u);
              kf.scale[h] = 0u;
              if (page != nullptr) {
                kf.code[h] = __ldg(reinterpret_cast<const uint4*>(page) + h * 32 + lane);
                kf.scale[h] = __ldg(reinterpret_cast<const uint16_t*>(page + 8 * D) + h * 32 + lane);
              }
            }
          },
          [&](int i, const Kv4Frag<NH>& kf) {
            for (int g = 0; g < groups; ++g)
              if (i >= 2 && !wait(kSDone + g, i - 2)) return false;
#pragma unroll
            for (int h = 0; h < NH; ++h) {
              const auto s0 = kv4_scales_of<T>(kf.scale[h], 0x4040), s1 = kv4_scales_of<T>(kf.scale[h], 0x4141);
              uint32_t v[4];
              uint8_t* d0 = k_to + (i & 1) * K_BUF + h * 8192;
              uint8_t* d1 = d0 + 2 * 128;
              kv4_values(kf.code[h].x, s0, v);
              *reinterpret_cast<uint4*>(d0 + (((2 * tig) ^ (r & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
              kv4_values(kf.code[h].y, s0, v);
              *reinterpret_cast<uint4*>(d0 + (((2 * tig + 1) ^ (r & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
              kv4_values(kf.code[h].z, s1, v);
              *reinterpret_cast<uint4*>(d1 + (((2 * tig) ^ ((r + 2) & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
              kv4_values(kf.code[h].w, s1, v);
              *reinterpret_cast<uint4*>(d1 + (((2 * tig + 1) ^ ((r + 2) & 7)) << 4)) =
                  make_uint4(v[0], v[1], v[2], v[3]);
            }
            written(kKFull, i);
            return true;
          });
    } else {
      const int seen = kv4_limit(a, tl, min(cols, c0 + NG * kKv4PromptCols) - 1);  // positions that any column sees
      const int vrow = kv4_perm(gid);
      uint8_t* const v_to = sv + vrow * 128 + (((mine * 2 + (tig >> 1)) ^ vrow) << 4) + (tig & 1) * 8;
      walk(
          [&](Kv4Frag<NH>& vf, const uint8_t* page) {
#pragma unroll
            for (int h = 0; h < NH; ++h) {
              vf.code[h] = make_uint4(0u, 0u, 0u, 0u);
              vf.scale[h] = 0u;
              if (page != nullptr) {
                vf.code[h] = __ldg(reinterpret_cast<const uint4*>(page + 9 * D) + h * 32 + lane);
                vf.scale[h] = __ldg(reinterpret_cast<const uint32_t*>(page + 17 * D) + (h * 4 + (gid >> 1)) * 4 + tig);
              }
            }
          },
          [&](int i, const Kv4Frag<NH>& vf) {
            for (int g = 0; g < groups; ++g)
              if (i >= 2 && !wait(kODone + g, i - 2)) return false;
            // slots past the last position seen may never have been written: no scale
            const int left = seen - (lo + i * PAGES + mine) * kKv4Page;
            uint32_t keep = 0xFFFFFFFFu;
            if (left < kKv4Page) {
              keep = 0u;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (2 * tig + 8 * (j >> 1) + (j & 1) < left) keep |= 0xFFu << (8 * j);
            }
#pragma unroll
            for (int h = 0; h < NH; ++h) {
              uint8_t* dst = v_to + (i & 1) * V_BUF + h * 8192;
              const uint32_t sc = vf.scale[h] & keep;
              const uint32_t s0 = kv4_scales(sc, 0x4140), s1 = kv4_scales(sc, 0x4342);
              uint32_t x[4], y[4];
              kv4_values(vf.code[h].x, s0, x);
              kv4_values(vf.code[h].z, s1, y);
#pragma unroll
              for (int j = 0; j < 4; ++j) *reinterpret_cast<uint2*>(dst + 8 * j * 128) = make_uint2(x[j], y[j]);
              kv4_values(vf.code[h].y, s0, x);
              kv4_values(vf.code[h].w, s1, y);
#pragma unroll
              for (int j = 0; j < 4; ++j) *reinterpret_cast<uint2*>(dst + (32 + 8 * j) * 128) = make_uint2(x[j], y[j]);
            }
            written(kVFull, i);
            return true;
          });
    }
  } else if (gr < groups) {  // ---- softmax ----
    const uint32_t t_s = t_s_of(gr), t_o = t_o_of(gr), t_lane = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int lim = in ? kv4_limit(a, tl, col) : 0;  // positions this column sees
    const int all_see = kv4_limit(a, tl, c0 + gr * kKv4PromptCols);  // that all do
    float m = -INFINITY, l = 0.f;  // maximum of the scores before their scale, as used; sum of p
    for (int i = 0; i < tiles; ++i) {
      if (!wait(kSDone + gr, i)) break;
      tc_fence_after();
      const int tile_page = lo + i * PAGES, at = tile_page * kKv4Page;
      const uint32_t t_mine = t_s + t_lane + 64 * (i & 1);
      const bool edge = at + kKv4PromptKeys > all_see || tile_page + PAGES > hi;
      const int left = min(lim, hi * kKv4Page) - at;  // of the tile, those this column sees
      uint32_t s[32];  // half of the scores at a time: the second, the first, the second again
      auto scores = [&](int c0) {
        tmem_load32(t_mine + c0, s);
        tmem_wait_ld();
        if (edge) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c0 + 16 * (c >> 4) + kv4_slot(c & 15) >= left) s[c] = 0xFF800000u;  // -infinity
        }
      };
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c0 = 32; c0 >= 0; c0 -= 32) {
        scores(c0);
#pragma unroll
        for (int c = 0; c < 32; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], s[c], s[c + 1]);
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      // (from -infinity too; not for a column that sees nothing)
      if (__any_sync(0xffffffffu, (top - m) * up > kKv4PromptSlack)) {
        const float mn = fmaxf(m, top);
        const float f = mn == -INFINITY ? 0.f : exp2_fast((m - mn) * up);
        m = mn;
        l *= f;
        if (i > 0) {
          if (!wait(kODone + gr, i - 1)) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_load16(t_o + t_lane + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tmem_store16(t_o + t_lane + c, o);
          }
        }
      }
      auto twice = [](float x) { return pair_of(__float_as_uint(x), __float_as_uint(x)); };
      const uint64_t up2 = twice(up), offset2 = twice(kKv4PromptOffset), minus2 = twice(m == -INFINITY ? 0.f : -m);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        if (c > 0) scores(c);
        uint32_t p[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float2 e = floats_of(fma2(add2(pair_of(s[2 * k], s[2 * k + 1]), minus2), up2, offset2));
          const float x = exp2_fast(e.x), y = exp2_fast(e.y);
          sum[k & 1] = add2(sum[k & 1], pair_of(__float_as_uint(x), __float_as_uint(y)));
          p[k] = pack_half2(x, y);
        }
        tmem_store16(t_mine + (c >> 1), p);  // over scores that have been taken
      }
      const float2 s0 = floats_of(add2(sum[0], sum[1]));
      l += s0.x + s0.y;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_bar[kPFull + gr][i & 1]);
    }
    if (tiles > 0) wait(kODone + gr, tiles - 1);
    tc_fence_after();
    // (all of the tiles' pages have been looked up, and s_lost with them)
    const bool none = s_lost < INT_MAX && s_lost * kKv4Page < lim;
    if (none) {
      m = INFINITY;
      l = 0.f;
    }

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
          if (none) {
#pragma unroll
            for (int k = 0; k < 8; ++k) r[k] = 0.f;
          }
          *reinterpret_cast<float4*>(dst) = make_float4(r[0], r[1], r[2], r[3]);
          *reinterpret_cast<float4*>(dst + 4) = make_float4(r[4], r[5], r[6], r[7]);
        }
      }
    }
    if (in && a.splits > 1)
      *reinterpret_cast<float2*>(kv4_part(a, tl.seq, tl.g, tl.tile, tl.split, tid, D) + D) = make_float2(m, l);
  }
  tc_fence_before();
  __syncthreads();  // (all parts have left their loops: a wait that ran out has set s_fail)
  if (warp == ISSUE) {
    if (s_fail) {  // what was issued may still be running: a bounded wait for it (0.2 s) before its memory goes
      if (lane == 0) kv4_error(a.c.status, kKv4Timeout);
      for (uint32_t i = 0; i < kKv4Tries; ++i) __nanosleep(1000);
    }
    tmem_dealloc(s_tmem, NG * kKv4PromptTmem);
  }
}

}  // namespace b2d

// kv4.cu — launches of the 4-bit KV cache's kernels and their C entry points
// (b2d_kv4_* in include/b2d.h).
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstring>

#include "b2d_host.h"
#include "kv4.cuh"
#include "kv4_prompt.cuh"

namespace b2d {

namespace {

template <class T, class TQ>
cudaError_t append_typed(const Kv4AppendArgs& a, cudaStream_t st, bool pdl) {
  // Many rows: a warp takes a whole row, so its addresses and angles are worked
  // out once (10239 rows of 48 heads of 128: 98 us with the read-back, 108 with
  // four warps a row); few: a block per batch of heads, one head a thread.  Rows
  // of 48 heads of 128, of 24 of 64 (us, few and many): 512 10.2 and 15.6, 5.7 and
  // 5.7; 1024 16.8 and 17.0, 9.3 and 7.4; 2000 30.3 and 20.8, 15.8 and 8.4.
  const bool many = a.n_rows >= 8 * a.c.d;
  const int threads = many ? 32 : kKv4AppendThreads;
  const int slices = threads / (a.c.d / 8);
  const unsigned batches = many ? 1u : static_cast<unsigned>((a.n_heads + slices - 1) / slices + 2);
  const dim3 grid(static_cast<unsigned>(a.n_rows), batches), block(threads);
  if (!a.cos) return launch(kv4_append_kernel<T, TQ, kRopeNone>, grid, block, 0, st, pdl, a);
  if (a.interleaved) return launch(kv4_append_kernel<T, TQ, kRopePairs>, grid, block, 0, st, pdl, a);
  if (a.rotary % 16 == 0) return launch(kv4_append_kernel<T, TQ, kRopeBlocks>, grid, block, 0, st, pdl, a);
  return launch(kv4_append_kernel<T, TQ, kRopeAny>, grid, block, 0, st, pdl, a);
}

// Dynamic shared memory past 48 KB is granted per kernel and device, once.
template <auto Kernel, int Bytes>
cudaError_t raise_smem() {
  if (Bytes <= 48 * 1024) return cudaSuccess;
  static std::atomic<bool> raised[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && raised[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Bytes);
  if (e == cudaSuccess && dev < 64) raised[dev].store(true, std::memory_order_relaxed);
  return e;
}

template <class T, int NH>
cudaError_t join(const Kv4AttnArgs& a, cudaStream_t st) {
  if (a.splits == 1) return cudaSuccess;
  return launch(kv4_join_kernel<T, NH>,
                dim3(static_cast<unsigned>(a.n_seqs), static_cast<unsigned>(a.c.n_kv),
                     static_cast<unsigned>((a.max_rows * a.group + 3) / 4)),
                dim3(128), 0, st, true, a);
}

template <auto Kernel, int Threads, int Smem, class T, int NH>
cudaError_t launch_tiles(const Kv4AttnArgs& a, dim3 grid, cudaStream_t st, bool pdl) {
  cudaError_t e = raise_smem<Kernel, Smem>();
  if (e == cudaSuccess) e = launch(Kernel, grid, dim3(Threads), Smem, st, pdl, a);
  return e == cudaSuccess ? join<T, NH>(a, st) : e;
}
template <class T, int NH, int NB>
cudaError_t attn_launch(const Kv4AttnArgs& a, cudaStream_t st, bool pdl) {
  const dim3 grid(static_cast<unsigned>(a.n_seqs), static_cast<unsigned>(a.c.n_kv),
                  static_cast<unsigned>(a.tiles * a.splits));
  return launch_tiles<kv4_attn_kernel<T, NH, NB>, 32 * kKv4Warps, kv4_attn_smem<NH, NB>(), T, NH>(a, grid, st, pdl);
}
template <class T, int NH, int NG>
cudaError_t prompt_launch(const Kv4AttnArgs& a, cudaStream_t st, bool pdl) {
  const dim3 grid(static_cast<unsigned>(a.n_seqs) * a.c.n_kv * a.tiles, static_cast<unsigned>(a.splits));
  return launch_tiles<kv4_prompt_kernel<T, NH, NG>, kv4_prompt_threads<NG>(), kv4_prompt_smem<NH, NG>(), T, NH>(
      a, grid, st, pdl);
}

template <class T, int NH>
cudaError_t attn_shape(const Kv4AttnArgs& a, cudaStream_t st, bool pdl) {
  if (a.tile_cols == 2 * kKv4PromptCols) return prompt_launch<T, NH, 2>(a, st, pdl);
  if (a.tile_cols == kKv4PromptCols) return prompt_launch<T, NH, 1>(a, st, pdl);
  return a.tile_cols > 8 ? attn_launch<T, NH, 2>(a, st, pdl) : attn_launch<T, NH, 1>(a, st, pdl);
}

template <class T>
cudaError_t attn_typed(const Kv4AttnArgs& a, cudaStream_t st, bool pdl) {
  return a.c.d == 64 ? attn_shape<T, 1>(a, st, pdl) : attn_shape<T, 2>(a, st, pdl);
}

}  // namespace

cudaError_t kv4_append(const Kv4AppendArgs& a, cudaStream_t st, bool pdl) {
  if (a.n_rows == 0) return cudaSuccess;
  if (a.dtype == B2D_F32) {
    if (a.q_out_dtype == B2D_F32) return append_typed<float, float>(a, st, pdl);
    if (a.q_out_dtype == B2D_F16) return append_typed<float, __half>(a, st, pdl);
    return append_typed<float, __nv_bfloat16>(a, st, pdl);
  }
  if (a.dtype == B2D_F16) return append_typed<__half, __half>(a, st, pdl);
  return append_typed<__nv_bfloat16, __nv_bfloat16>(a, st, pdl);
}

cudaError_t kv4_read(const Kv4ReadArgs& a, cudaStream_t st) {
  if (a.n_rows == 0) return cudaSuccess;
  const int slices = 128 / (a.c.d / 8);
  const dim3 grid(static_cast<unsigned>(a.n_rows),
                  a.n_rows >= 1024 ? 1u : static_cast<unsigned>(std::min(65535, (2 * a.c.n_kv + slices - 1) / slices))),
      block(128);
  if (a.dtype == B2D_F32) return launch(kv4_read_kernel<float>, grid, block, 0, st, false, a);
  if (a.dtype == B2D_F16) return launch(kv4_read_kernel<__half>, grid, block, 0, st, false, a);
  return launch(kv4_read_kernel<__nv_bfloat16>, grid, block, 0, st, false, a);
}

namespace {
int64_t plan_pages(const Kv4AttnArgs& a) { return std::max(1, (a.max_len + kKv4Page - 1) / kKv4Page); }
int64_t plan_units(const Kv4AttnArgs& a) { return static_cast<int64_t>(a.n_seqs) * a.c.n_kv * a.tiles; }
// Splits: at least 32 pages each (8 a warp).  One sequence's splits are alike:
// one wave of CTAs, four to an SM (131071 positions, 8 kv heads of 128: 46 us,
// and 55 us with splits for four waves).  Several sequences differ in length:
// four waves even that out (32 of 1001 to 16384: 93 us, and 110 us with one).
// Prompts: one CTA to an SM, 64 pages each at least (256 rows of 4 heads on 8192
// positions, 64 tiles: 69 us, and 109 without splits).
int64_t plan_splits(const Kv4AttnArgs& a, int sms) {
  const bool prompt = a.tile_cols >= kKv4PromptCols;
  const int64_t ctas = int64_t(sms) * (prompt ? 1 : a.n_seqs == 1 ? 4 : 16), least = prompt ? 64 : 32;
  return std::max<int64_t>(
      1, std::min<int64_t>(ctas / std::max<int64_t>(1, plan_units(a)), (plan_pages(a) + least - 1) / least));
}
}  // namespace

bool kv4_attn_plan(Kv4AttnArgs& a, int sms) {
  a.group = a.n_heads / a.c.n_kv;
  a.group_inv = ((uint64_t(1) << 32) + a.group - 1) / a.group;
  const int64_t cols = static_cast<int64_t>(a.max_rows) * a.group;
  if (cols * a.group >= int64_t(1) << 32) return false;
  // The kernel for prompts takes 128 columns at the price of any; the other one
  // walks the pages once per 16.  From 65 columns on it is the prompts', and below
  // where the pages are many (the product of sequences, kv heads, positions, dims
  // over 128), else its start weighs more.  us, prompts' and other:
  //   48 columns, 128 dims, 64 Ki: 22 and 26;  16 Ki (64 dims): 18 and 12
  //   32 columns, 128 dims, 512 Ki: 64 and 85;  64 Ki: 22 and 17
  //   32 columns,  64 dims, 128 Ki: 34 and 27
  const int64_t work = int64_t(a.n_seqs) * a.c.n_kv * a.max_len * a.c.d / 128;
  const bool prompt = cols > 64 || (cols > 32 && work >= 1 << 16) || (cols > 16 && a.c.d == 128 && work >= 1 << 19);
  a.tile_cols = prompt ? kKv4PromptCols : cols <= 8 ? 8 : 16;
  a.tiles = static_cast<int>((cols + a.tile_cols - 1) / a.tile_cols);
  // Two groups of columns a CTA share the values of K and V: where one each would
  // leave no SM without a CTA (288 tiles of 128 columns on 8192 positions: 147 us,
  // and 212 with a group a CTA; 144 tiles: 126 and 111).  One tile of a sequence and
  // kv head has nobody to share with (256 of them on 4096 positions: 130 us a group a
  // CTA, 154 in pairs of which one is empty; on 512, 33 and 34).
  if (prompt && a.tiles > 1 && plan_units(a) > sms) {
    a.tile_cols *= 2;
    a.tiles = (a.tiles + 1) / 2;
  }
  const int64_t pages = plan_pages(a), splits = plan_splits(a, sms);
  a.split_pages = static_cast<int>((pages + splits - 1) / splits);
  a.splits = static_cast<int>((pages + a.split_pages - 1) / a.split_pages);
  // the grid's x, y and z
  return plan_units(a) <= INT_MAX && a.c.n_kv <= 65535 && int64_t(a.tiles) * a.splits <= 65535 && (a.splits == 1 || cols <= 65535);
}

uint64_t kv4_attn_scratch(const Kv4AttnArgs& a) {
  return a.splits <= 1 ? 0 : uint64_t(plan_units(a)) * a.splits * a.tile_cols * (a.c.d + 4) * sizeof(float);
}
uint64_t kv4_attn_scratch_most(int d, int sms) {
  // (split tiles are no more than the CTAs that plan_splits wants; prompts in pairs are not split)
  return uint64_t(sms) * std::max(16 * 16, kKv4PromptCols) * (d + 4) * sizeof(float);
}

cudaError_t kv4_attention(const Kv4AttnArgs& a, cudaStream_t st, bool pdl) {
  if (a.n_rows == 0 || a.n_seqs == 0) return cudaSuccess;
  return a.dtype == B2D_F16 ? attn_typed<__half>(a, st, pdl) : attn_typed<__nv_bfloat16>(a, st, pdl);
}

}  // namespace b2d

namespace {

#define KV4_CUDA(call, what)                              \
  do {                                                    \
    cudaError_t e_ = (call);                              \
    if (e_ != cudaSuccess) return b2d::cuda_failed(e_, what); \
  } while (0)

b2d_status check_cache(const b2d_kv4_cache* c, b2d::Kv4Cache& k) {
  if (!c || !c->pool || (reinterpret_cast<uintptr_t>(c->pool) & 15u) || !c->table || c->n_kv_heads < 1 ||
      c->num_blocks < 1 || c->blocks_per_seq < 1 || c->table_rows < 1 || c->device < 0)
    return B2D_ERR_INVALID_ARG;
  if (c->d_head != 64 && c->d_head != 128) return B2D_ERR_UNSUPPORTED;
  if (c->blocks_per_seq > 0x7fffffff / b2d::kKv4Page) return B2D_ERR_INVALID_ARG;
  k.pool = static_cast<uint8_t*>(c->pool);
  k.table = c->table;
  k.status = c->status;
  k.n_kv = c->n_kv_heads;
  k.d = c->d_head;
  k.num_blocks = c->num_blocks;
  k.bps = c->blocks_per_seq;
  k.table_rows = c->table_rows;
  k.table_ld = c->blocks_per_seq;
  return B2D_OK;
}

constexpr float kLog2e = 1.4426950408889634f;  // (exponents are of 2)
b2d_status check_query(const b2d_kv4_cache* c, const b2d_kv4_query* q, b2d::Kv4AttnArgs& a) {
  std::memset(&a, 0, sizeof(a));
  const b2d_status s = check_cache(c, a.c);
  if (s != B2D_OK) return s;
  if (!q || !q->q || !q->out || !q->lens || q->n_rows < 0 || q->n_seqs < 0 || q->n_heads < 1 ||
      q->n_heads % c->n_kv_heads || q->max_rows < 1 || q->n_seqs > c->table_rows || q->max_len < 0 ||
      int64_t(q->max_len) > int64_t(c->blocks_per_seq) * b2d::kKv4Page || !(q->scale > 0.f) || std::isinf(q->scale * kLog2e) ||
      (!q->q_start && (q->n_rows != q->n_seqs || q->max_rows != 1)))
    return B2D_ERR_INVALID_ARG;
  if (q->dtype != B2D_BF16 && q->dtype != B2D_F16) return B2D_ERR_UNSUPPORTED;
  a.q = q->q;
  a.out = q->out;
  a.q_row = q->q_row; a.q_head = q->q_head;
  a.o_row = q->out_row; a.o_head = q->out_head;
  a.lens = q->lens;
  a.q_start = q->q_start;
  a.scale_log2 = q->scale * kLog2e;
  a.n_rows = q->n_rows;
  a.n_heads = q->n_heads;
  a.n_seqs = q->n_seqs;
  a.max_rows = std::min(q->max_rows, std::max(1, q->n_rows));
  a.max_len = q->max_len;
  a.dtype = q->dtype;
  int sms = 0;
  const cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, c->device);
  if (e != cudaSuccess) return b2d::cuda_failed(e, "SM count");
  return b2d::kv4_attn_plan(a, sms) ? B2D_OK : B2D_ERR_UNSUPPORTED;
}

}  // namespace

extern "C" b2d_status b2d_kv4_append(const b2d_kv4_cache* cache, const b2d_kv4_rows* rows, void* stream) {
  b2d::Kv4AppendArgs a;
  std::memset(&a, 0, sizeof(a));
  const b2d_status s = check_cache(cache, a.c);
  if (s != B2D_OK) return s;
  if (!rows || !rows->k || !rows->v || !rows->pos ||
      (rows->q && rows->q == rows->q_out &&
       (rows->q_row != rows->q_out_row || rows->q_head != rows->q_out_head || rows->dtype != rows->q_out_dtype)) || rows->n_rows < 0 || (rows->q != nullptr) != (rows->q_out != nullptr) ||
      (rows->q && rows->n_heads < 1) || (rows->cos != nullptr) != (rows->sin != nullptr) ||
      (rows->cos && (rows->rotary_dim < 2 || rows->rotary_dim > cache->d_head || rows->rotary_dim % 2 ||
                     rows->max_pos < 1)) ||
      (!rows->seq && rows->n_rows > cache->table_rows))
    return B2D_ERR_INVALID_ARG;
  const bool same = rows->q_out_dtype == rows->dtype;
  if (rows->dtype < B2D_F32 || rows->dtype > B2D_F16 || rows->q_out_dtype < B2D_F32 || rows->q_out_dtype > B2D_F16 ||
      (rows->q && !same && rows->dtype != B2D_F32))
    return B2D_ERR_UNSUPPORTED;
  a.q = rows->q; a.k = rows->k; a.v = rows->v; a.q_out = rows->q_out;
  a.q_row = rows->q_row; a.q_head = rows->q_head; a.k_row = rows->k_row; a.k_head = rows->k_head;
  a.v_row = rows->v_row; a.v_head = rows->v_head; a.qo_row = rows->q_out_row; a.qo_head = rows->q_out_head;
  a.pos = rows->pos; a.seq = rows->seq; a.cos = rows->cos; a.sin = rows->sin;
  a.n_rows = rows->n_rows; a.n_heads = rows->q ? rows->n_heads : 0;
  a.rotary = rows->cos ? rows->rotary_dim : 0;
  a.interleaved = rows->interleaved != 0;
  a.max_pos = rows->max_pos;
  a.dtype = rows->dtype;
  a.q_out_dtype = rows->q ? rows->q_out_dtype : rows->dtype;
  b2d::DeviceScope dev(cache->device);
  KV4_CUDA(dev.error(), "device");
  KV4_CUDA(b2d::kv4_append(a, static_cast<cudaStream_t>(stream), false), "kv4 append");
  return B2D_OK;
}

extern "C" b2d_status b2d_kv4_read(const b2d_kv4_cache* cache, const int32_t* pos_dev, const int32_t* seq_dev,
                                   int n_rows, int dtype, void* k_dev, void* v_dev, void* stream) {
  b2d::Kv4ReadArgs a;
  std::memset(&a, 0, sizeof(a));
  const b2d_status s = check_cache(cache, a.c);
  if (s != B2D_OK) return s;
  if (!pos_dev || !k_dev || !v_dev || n_rows < 0 || (!seq_dev && n_rows > cache->table_rows)) return B2D_ERR_INVALID_ARG;
  if (dtype < B2D_F32 || dtype > B2D_F16) return B2D_ERR_UNSUPPORTED;
  a.k = k_dev; a.v = v_dev; a.pos = pos_dev; a.seq = seq_dev;
  a.n_rows = n_rows;
  a.dtype = dtype;
  b2d::DeviceScope dev(cache->device);
  KV4_CUDA(dev.error(), "device");
  KV4_CUDA(b2d::kv4_read(a, static_cast<cudaStream_t>(stream)), "kv4 read");
  return B2D_OK;
}

extern "C" b2d_status b2d_kv4_attention_scratch(const b2d_kv4_cache* cache, const b2d_kv4_query* query,
                                                uint64_t* bytes) {
  if (!bytes) return B2D_ERR_INVALID_ARG;
  *bytes = 0;
  b2d::Kv4AttnArgs a;
  const b2d_status s = check_query(cache, query, a);
  if (s == B2D_OK) *bytes = b2d::kv4_attn_scratch(a);
  return s;
}

extern "C" b2d_status b2d_kv4_attention(const b2d_kv4_cache* cache, const b2d_kv4_query* query, void* scratch_dev,
                                        uint64_t scratch_bytes, void* stream) {
  b2d::Kv4AttnArgs a;
  const b2d_status s = check_query(cache, query, a);
  if (s != B2D_OK) return s;
  const uint64_t need = b2d::kv4_attn_scratch(a);
  if (need > 0 && (!scratch_dev || (reinterpret_cast<uintptr_t>(scratch_dev) & 15u) || scratch_bytes < need))
    return B2D_ERR_INVALID_ARG;
  a.part = static_cast<float*>(scratch_dev);
  b2d::DeviceScope dev(cache->device);
  KV4_CUDA(dev.error(), "device");
  KV4_CUDA(b2d::kv4_attention(a, static_cast<cudaStream_t>(stream), false), "kv4 attention");
  return B2D_OK;
}

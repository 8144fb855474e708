// kv4.h — the 4-bit paged KV cache inside the library: the arguments of its
// kernels (kv4.cu) and their launches, for the C entry points and the batched
// step.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace b2d {

constexpr int kKv4Page = 16;    // positions per page
constexpr int kKv4Group = 16;   // dims per scale
constexpr int kKv4MaxByte = 0xE1;  // the largest scale, 9216: 7 * 9216 = 64512 is a finite half
// Bytes of one kv head's page: K codes 8 d, K scales d, V codes 8 d, V scales d.
constexpr __host__ __device__ int kv4_page_bytes(int d) { return 18 * d; }

// One layer's cache.
struct Kv4Cache {
  uint8_t* pool;         // [num_blocks][n_kv][18 d]
  const int32_t* table;  // sequence s: entries at table + s * table_ld
  uint32_t* status;      // first bad input seen by a kernel, or null
  int n_kv, d, num_blocks, bps, table_rows;
  int64_t table_ld;
};

struct Kv4AppendArgs {
  Kv4Cache c;
  const void *q, *k, *v;  // rows, `dtype`; q may be null
  void* q_out;            // `q_out_dtype`
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, qo_row, qo_head;  // strides in elements
  const int32_t* pos;
  const int32_t* seq;     // table row of each row, or null: row i uses table row i
  const float *cos, *sin; // [max_pos][rotary / 2], or null: no rotation
  int n_rows, n_heads, rotary, interleaved, max_pos;
  int dtype, q_out_dtype;
};

struct Kv4ReadArgs {
  Kv4Cache c;
  void *k, *v;            // [n_rows][n_kv][d], `dtype`
  const int32_t* pos;
  const int32_t* seq;
  int n_rows, dtype;
};

struct Kv4AttnArgs {
  Kv4Cache c;
  const void* q;
  void* out;
  int64_t q_row, q_head, o_row, o_head;
  const int32_t* lens;     // [n_seqs]; len_add is added to each
  const int32_t* q_start;  // [n_seqs + 1], or null: sequence i has the one row i ..
  int rows_of_one;         // .. or, when > 0, the one sequence has rows 0 .. rows_of_one - 1
  float* part;             // partials of split sequences (kv4_attn_scratch bytes)
  float scale_log2;        // softmax scale * log2(e)
  int n_rows, n_heads, n_seqs, max_rows, max_len, dtype;
  int len_add;
  int early;               // 1: what the kernel before writes to the pool is in each sequence's last page
                           // (lens and table come from earlier ones): the other pages are fetched before it
                           // ends (64 rows at position 500: 964 -> 934 us a step)
  // set by kv4_attn_plan: query columns (row, head) per tile, tiles per
  // (sequence, kv head), splits of the positions and pages per split
  int tile_cols, tiles, splits, split_pages;
  int group;               // query heads of a kv head
  uint64_t group_inv;      // ceil(2^32 / group): c / group = c * group_inv >> 32 while c * group < 2^32
};

cudaError_t kv4_append(const Kv4AppendArgs& a, cudaStream_t st, bool pdl);
cudaError_t kv4_read(const Kv4ReadArgs& a, cudaStream_t st);
// The split of a call's work (false: too large for a grid), then the bytes of
// a.part it needs.
bool kv4_attn_plan(Kv4AttnArgs& a, int sms);
uint64_t kv4_attn_scratch(const Kv4AttnArgs& a);
// The most that any call on heads of d dims needs.
uint64_t kv4_attn_scratch_most(int d, int sms);
cudaError_t kv4_attention(const Kv4AttnArgs& a, cudaStream_t st, bool pdl);

}  // namespace b2d

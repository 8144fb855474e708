// logits.cu — the logits adjustment (b2d_adjust_logits): penalties for tokens
// seen, biases and token masks, one row of rules per row of logits (sm_100a).
//
// One pass over the logits: a CTA owns `slice` tokens of a row, loads them
// first, and while they arrive looks through the row's lists for its tokens.
// The lists are short beside the vocabulary: a bit per token in `touched` says
// where counts and bias places need a look.  Counts are integers and a bias
// place is the largest index, so no result depends on an order.
// 256 rows of 32000 with masks, 511 tokens of history and 16 biases: 15.1 us, 4.4 TB/s
// (67 MB at the copy rate: 10.2); 65 rows of 100003 with 4096 of history: 18.9 us,
// since each of a row's 25 CTAs looks through all of the history.  Bound by the
// CTA's chain of list, count and store, five CTAs to an SM.  Measured against 16.0
// and 19.8: three ids of a list in flight 16.5 and 19.2, four 17.6 and 20.6, four
// CTAs 18.1 and 21.0, slices of 8192 by 512 threads 16.3 and 17.6.
#include <algorithm>

#include "b2d_host.h"
#include "b2d_ptx.cuh"

namespace b2d {
namespace {

constexpr int kLogitsThreads = 256;
constexpr int kLogitsSlice = 4096;                           // most tokens of a CTA
constexpr int kLogitsPer = kLogitsSlice / kLogitsThreads;    // loads a thread has in flight
constexpr uint32_t kInPrompt = 0x80000000u;                  // a count's flag: seen in the prompt

constexpr int kLogitsIds = 2;  // ids of a list a thread has in flight

__global__ void __launch_bounds__(kLogitsThreads, 5) adjust_logits_kernel(const __grid_constant__ b2d_logits_rules a,
                                                                       int slice) {
  // (the bits, which every token looks at, first: 15.1 and 18.9 us, and 16.0 and 19.8 behind the rest)
  __shared__ __align__(16) uint32_t lists_mem[kLogitsSlice / 32 + 2 * kLogitsSlice];
  uint32_t* touched = lists_mem;
  uint32_t* count = touched + kLogitsSlice / 32;
  uint32_t* place = count + kLogitsSlice;  // 1 + index of the bias that holds
  const int tid = threadIdx.x, lane = tid & 31;
  const int row = blockIdx.y, v0 = blockIdx.x * slice;
  const int n = min(slice, a.vocab - v0);
  const float* src = a.logits + row * a.logits_ld + v0;
  // Everything whose address is known goes out first: the logits, the mask (a
  // warp's 32 tokens share a word; lane i has the word of its i-th 32), the
  // row's numbers and the first ids of its lists, before their lengths are known.
  float x[kLogitsPer];
#pragma unroll
  for (int i = 0; i < kLogitsPer; ++i) {
    const int k = tid + i * kLogitsThreads;
    x[i] = k < n ? src[k] : 0.f;
  }
  uint32_t mask = 0xFFFFFFFFu;
  if (a.allowed != nullptr && lane < kLogitsPer) {
    const int w = (tid >> 5) + lane * (kLogitsThreads / 32);
    if (32 * w < n) mask = __ldg(a.allowed + row * a.allowed_ld + (v0 >> 5) + w);
  }
  const bool lists = a.history != nullptr || a.bias_ids != nullptr;  // (uniform over the grid)
  const int32_t* hist_ids = a.history + static_cast<int64_t>(row) * a.hist_cap;
  const int32_t* bias_ids = a.bias_ids + static_cast<int64_t>(row) * a.bias_cap;
  // kLogitsIds of a list's ids a thread, from place i0 on
  auto load_ids = [&](const int32_t* ids, int i0, int len, int (&id)[kLogitsIds]) {
#pragma unroll
    for (int j = 0; j < kLogitsIds; ++j) {
      const int i = i0 + j * kLogitsThreads;
      id[j] = i < len ? __ldg(ids + i) : -1;
    }
  };
  int hid[kLogitsIds], bid[kLogitsIds];
  load_ids(hist_ids, tid, a.history != nullptr ? a.hist_cap : 0, hid);
  load_ids(bias_ids, tid, a.bias_ids != nullptr ? a.bias_cap : 0, bid);
  const int hist = a.history != nullptr ? min(max(a.hist_len[row], 0), a.hist_cap) : 0;
  const int made = a.prompt_len != nullptr ? a.prompt_len[row] : 0;
  const int biases = a.bias_ids != nullptr ? min(max(a.bias_len[row], 0), a.bias_cap) : 0;
  const float rep = a.rep != nullptr ? a.rep[row] : 1.f;
  const float presence = a.presence != nullptr ? a.presence[row] : 0.f;
  const float frequency = a.frequency != nullptr ? a.frequency[row] : 0.f;
  if (lists) {
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    if (tid < kLogitsSlice / 128) reinterpret_cast<uint4*>(touched)[tid] = zero;
    for (int i = tid; i < (n + 3) / 4; i += kLogitsThreads)
      reinterpret_cast<uint4*>(count)[i] = reinterpret_cast<uint4*>(place)[i] = zero;
    // f(place in the list, place in the slice) for the list's ids in this slice
    auto each = [&](const int32_t* ids, int len, int (&id)[kLogitsIds], auto&& f) {
      for (int i0 = tid; i0 < len; i0 += kLogitsThreads * kLogitsIds) {
        if (i0 != tid) load_ids(ids, i0, len, id);
#pragma unroll
        for (int j = 0; j < kLogitsIds; ++j) {
          const int i = i0 + j * kLogitsThreads;
          const uint32_t k = static_cast<uint32_t>(id[j]) - static_cast<uint32_t>(v0);
          if (i < len && id[j] >= 0 && k < static_cast<uint32_t>(n)) {
            f(i, k);
            atomicOr(&touched[k >> 5], 1u << (k & 31));
          }
        }
      }
    };
    __syncthreads();
    each(hist_ids, hist, hid, [&](int i, uint32_t k) {
      if (i < made) atomicOr(&count[k], kInPrompt);
      else atomicAdd(&count[k], 1u);
    });
    each(bias_ids, biases, bid, [&](int i, uint32_t k) { atomicMax(&place[k], static_cast<uint32_t>(i) + 1u); });
    __syncthreads();
  }
  const float* bias = a.bias_values + static_cast<int64_t>(row) * a.bias_cap;
  float* dst = a.out + row * a.out_ld + v0;
#pragma unroll
  for (int i = 0; i < kLogitsPer; ++i) {
    const int k = tid + i * kLogitsThreads;
    const uint32_t word = __shfl_sync(0xffffffffu, mask, i);
    float y = x[i];
    if (lists && k < n && ((touched[k >> 5] >> lane) & 1u)) {
      const uint32_t c = count[k], made_n = c & ~kInPrompt;
      if (c != 0u) y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
      if (made_n != 0u) y -= fmaf(frequency, static_cast<float>(made_n), presence);
      if (place[k] != 0u) y += bias[place[k] - 1u];
    }
    if (!((word >> lane) & 1u)) y = -INFINITY;
    if (k < n) dst[k] = y;
  }
}

}  // namespace
}  // namespace b2d

extern "C" b2d_status b2d_adjust_logits(const b2d_logits_rules* r, void* stream) {
  if (!r || !r->logits || !r->out || r->batch < 0 || r->vocab < 1 || r->device < 0 ||
      (r->batch > 1 && (r->logits_ld < r->vocab || r->out_ld < r->vocab)) ||
      (r->logits == r->out && r->batch > 1 && r->logits_ld != r->out_ld) ||
      (r->history ? !r->hist_len || r->hist_cap < 0 : r->hist_len || r->prompt_len || r->rep || r->presence || r->frequency) ||
      (r->bias_ids ? !r->bias_values || !r->bias_len || r->bias_cap < 0 : r->bias_values || r->bias_len) ||
      (r->allowed && r->batch > 1 && r->allowed_ld < (int64_t(r->vocab) + 31) / 32))
    return B2D_ERR_INVALID_ARG;
  if (r->batch > 65535) return B2D_ERR_UNSUPPORTED;
  if (r->batch == 0) return B2D_OK;
  int sms = 0;
  const cudaError_t got = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, r->device);
  if (got != cudaSuccess) return b2d::cuda_failed(got, "SM count");
  // whole slices where the rows fill the GPU (two CTAs to each SM); a few rows are cut finer
  int slice = b2d::kLogitsSlice;
  while (slice > b2d::kLogitsThreads * 4 && int64_t(r->batch) * ((int64_t(r->vocab) + slice - 1) / slice) < 2 * sms) slice /= 2;
  b2d::DeviceScope dev(r->device);
  if (dev.error() != cudaSuccess) return b2d::cuda_failed(dev.error(), "device");
  const dim3 grid(static_cast<unsigned>((int64_t(r->vocab) + slice - 1) / slice), static_cast<unsigned>(r->batch));
  const cudaError_t e = b2d::launch(b2d::adjust_logits_kernel, grid, dim3(b2d::kLogitsThreads), 0,
                                    static_cast<cudaStream_t>(stream), false, *r, slice);
  return e == cudaSuccess ? B2D_OK : b2d::cuda_failed(e, "adjust logits");
}

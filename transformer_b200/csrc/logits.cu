// logits.cu — the logits adjustment (b2d_adjust_logits): penalties for tokens
// seen, biases and token masks, one row of rules per row of logits (sm_100a).
//
// One pass over the logits: a CTA owns `slice` tokens of a row, loads them
// first, and while they arrive looks through the row's lists for its tokens.
// The lists are short beside the vocabulary, so what they say is kept sparsely:
// a bit per token in `touched`, and counts and bias places that are only
// initialised and read where the bit is set.  Counts are integers and a bias
// place is the largest index, so no result depends on an order.
#include <algorithm>

#include "b2d_host.h"
#include "b2d_ptx.cuh"

namespace b2d {
namespace {

constexpr int kLogitsThreads = 256;
constexpr int kLogitsSlice = 4096;                           // most tokens of a CTA
constexpr int kLogitsPer = kLogitsSlice / kLogitsThreads;    // loads a thread has in flight
constexpr uint32_t kInPrompt = 0x80000000u;                  // a count's flag: seen in the prompt

__global__ void __launch_bounds__(kLogitsThreads) adjust_logits_kernel(const __grid_constant__ b2d_logits_rules a,
                                                                       int slice) {
  __shared__ uint32_t touched[kLogitsSlice / 32];
  __shared__ uint32_t count[kLogitsSlice];
  __shared__ uint32_t place[kLogitsSlice];  // 1 + index of the bias that holds
  const int tid = threadIdx.x, lane = tid & 31;
  const int row = blockIdx.y, v0 = blockIdx.x * slice;
  const int n = min(slice, a.vocab - v0);
  const float* src = a.logits + row * a.logits_ld + v0;
  float x[kLogitsPer];
#pragma unroll
  for (int i = 0; i < kLogitsPer; ++i) {
    const int k = tid + i * kLogitsThreads;
    x[i] = k < n ? src[k] : 0.f;
  }
  const int hist = a.history != nullptr ? min(max(a.hist_len[row], 0), a.hist_cap) : 0;
  const int made = a.prompt_len != nullptr ? a.prompt_len[row] : 0;
  const int biases = a.bias_ids != nullptr ? min(max(a.bias_len[row], 0), a.bias_cap) : 0;
  const int32_t* ids = a.history + static_cast<int64_t>(row) * a.hist_cap;
  const int32_t* bids = a.bias_ids + static_cast<int64_t>(row) * a.bias_cap;
  if (hist + biases > 0) {  // (uniform over the CTA)
    if (tid < kLogitsSlice / 32) touched[tid] = 0u;
    for (int i = tid; i < hist; i += kLogitsThreads) {
      const uint32_t k = static_cast<uint32_t>(ids[i] - v0);
      if (ids[i] >= 0 && k < static_cast<uint32_t>(n)) count[k] = place[k] = 0u;
    }
    for (int i = tid; i < biases; i += kLogitsThreads) {
      const uint32_t k = static_cast<uint32_t>(bids[i] - v0);
      if (bids[i] >= 0 && k < static_cast<uint32_t>(n)) count[k] = place[k] = 0u;
    }
    __syncthreads();
    for (int i = tid; i < hist; i += kLogitsThreads) {
      const uint32_t k = static_cast<uint32_t>(ids[i] - v0);
      if (ids[i] >= 0 && k < static_cast<uint32_t>(n)) {
        if (i < made) atomicOr(&count[k], kInPrompt);
        else atomicAdd(&count[k], 1u);
        atomicOr(&touched[k >> 5], 1u << (k & 31));
      }
    }
    for (int i = tid; i < biases; i += kLogitsThreads) {
      const uint32_t k = static_cast<uint32_t>(bids[i] - v0);
      if (bids[i] >= 0 && k < static_cast<uint32_t>(n)) {
        atomicMax(&place[k], static_cast<uint32_t>(i) + 1u);
        atomicOr(&touched[k >> 5], 1u << (k & 31));
      }
    }
    __syncthreads();
  }
  const float rep = a.rep != nullptr ? a.rep[row] : 1.f;
  const float presence = a.presence != nullptr ? a.presence[row] : 0.f;
  const float frequency = a.frequency != nullptr ? a.frequency[row] : 0.f;
  const float* bias = a.bias_values + static_cast<int64_t>(row) * a.bias_cap;
  const uint32_t* allowed = a.allowed != nullptr ? a.allowed + row * a.allowed_ld + (v0 >> 5) : nullptr;
  float* dst = a.out + row * a.out_ld + v0;
#pragma unroll
  for (int i = 0; i < kLogitsPer; ++i) {
    const int k = tid + i * kLogitsThreads;  // a warp's 32 tokens share a word of the mask
    if (k >= n) break;
    float y = x[i];
    if (hist + biases > 0 && ((touched[k >> 5] >> lane) & 1u)) {
      const uint32_t c = count[k], made_n = c & ~kInPrompt;
      if (c != 0u) y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
      if (made_n != 0u) y -= fmaf(frequency, static_cast<float>(made_n), presence);
      if (place[k] != 0u) y += bias[place[k] - 1u];
    }
    if (allowed != nullptr && !((__ldg(allowed + (k >> 5)) >> lane) & 1u)) y = -INFINITY;
    dst[k] = y;
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
  // whole slices where the rows fill the GPU; a few rows are cut finer
  int slice = b2d::kLogitsSlice;
  while (slice > b2d::kLogitsThreads * 4 && int64_t(r->batch) * ((int64_t(r->vocab) + slice - 1) / slice) < 2 * 148) slice /= 2;
  b2d::DeviceScope dev(r->device);
  if (dev.error() != cudaSuccess) return b2d::cuda_failed(dev.error(), "device");
  const dim3 grid(static_cast<unsigned>((int64_t(r->vocab) + slice - 1) / slice), static_cast<unsigned>(r->batch));
  const cudaError_t e = b2d::launch(b2d::adjust_logits_kernel, grid, dim3(b2d::kLogitsThreads), 0,
                                    static_cast<cudaStream_t>(stream), false, *r, slice);
  return e == cudaSuccess ? B2D_OK : b2d::cuda_failed(e, "adjust logits");
}

// Logits under penalties for repeated tokens, biases and grammar masks, and the
// greedy choice after them (fah_logits_adjust of the C ABI).
//
// Two launches. logits_kernel: a workgroup takes kChunk tokens of one row. It
// clears a table of one pair of words per token in LDS, scans the row's history
// and bias list once (each chunk scans them whole: a few KB, from the L2) and
// notes the entries that fall into its tokens with integer LDS atomics, whose
// result does not depend on their order: the word `seen` is the count behind
// the prompt and, in bit 31, whether the token stands in the history at all;
// `entry` is the last list entry of the token's bias plus one. Then it streams
// its logits through registers once, 16 bytes a lane, and keeps each lane's
// largest written value. choice_kernel takes the largest over a row's chunks.
#include "fah_device.h"
#include "fah_internal.h"

namespace fah {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 1024;

template <typename T>
__global__ __launch_bounds__(kThreads) void logits_kernel(fah_logits_adjust a, unsigned long long* keys) {
  __shared__ unsigned seen[kChunk], entry[kChunk];
  __shared__ unsigned long long part[kThreads / kWave];
  const int row = blockIdx.y, first = blockIdx.x * kChunk, tid = threadIdx.x;
  const int tokens = a.vocab - first < kChunk ? a.vocab - first : kChunk;
  for (int i = tid; i < kChunk; i += kThreads) seen[i] = entry[i] = 0;
  __syncthreads();
  if (a.history_capacity) {
    const int* list = a.history + row * a.history_stride;
    int n = a.history_counts ? a.history_counts[row] : a.history_capacity;
    n = n < a.history_capacity ? n : a.history_capacity;
    const int prompt = a.prompt_counts ? a.prompt_counts[row] : 0;
    for (int i = tid; i < n; i += kThreads) {
      const unsigned t = (unsigned)list[i] - (unsigned)first;
      if (list[i] >= 0 && t < (unsigned)tokens) {
        atomicOr(&seen[t], 0x80000000u);
        if (i >= prompt) atomicAdd(&seen[t], 1u);
      }
    }
  }
  if (a.bias_capacity) {
    const int* list = a.bias_tokens + row * a.bias_stride;
    int n = a.bias_counts ? a.bias_counts[row] : a.bias_capacity;
    n = n < a.bias_capacity ? n : a.bias_capacity;
    for (int i = tid; i < n; i += kThreads) {
      const unsigned t = (unsigned)list[i] - (unsigned)first;
      if (list[i] >= 0 && t < (unsigned)tokens) atomicMax(&entry[t], (unsigned)i + 1u);
    }
  }
  __syncthreads();
  const float repetition = a.repetition ? a.repetition[row] : 1.0f;
  const float presence = a.presence ? a.presence[row] : 0.0f;
  const float frequency = a.frequency ? a.frequency[row] : 0.0f;
  const uint32_t* mask = nullptr;
  if (a.mask_rows) {
    const int m = a.mask_index ? a.mask_index[row] : a.mask_rows == 1 ? 0 : row;
    if (m >= 0 && m < a.mask_rows) mask = a.masks + m * a.mask_stride;
  }
  const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride + first;
  T* out = static_cast<T*>(a.output) + row * a.output_stride + first;
  unsigned long long best = 0;
  for (int i = tid; i < tokens; i += kThreads) {
    float x = (float)in[i];
    const unsigned w = seen[i], e = entry[i];
    if (w) x = x > 0.0f ? x / repetition : x * repetition;
    const unsigned n = w & 0x7fffffffu;
    if (n) {
      x = x - frequency * (float)n;
      x = x - presence;
    }
    if (e) x = x + a.bias_values[row * a.bias_stride + (e - 1)];
    if (mask && !(mask[(first + i) >> 5] >> ((first + i) & 31) & 1u)) x = -__builtin_inff();
    const T y = (T)x;
    out[i] = y;
    if ((float)y > -__builtin_inff()) {
      const unsigned long long key = greedy_key((float)y, (uint32_t)(first + i));
      best = key > best ? key : best;
    }
  }
  if (!keys) return;
  best = wave_max_u64(best);
  if (tid % kWave == 0) part[tid / kWave] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kThreads / kWave; ++w) best = part[w] > best ? part[w] : best;
    keys[(size_t)row * gridDim.x + blockIdx.x] = best;
  }
}

__global__ __launch_bounds__(kWave) void choice_kernel(const unsigned long long* keys, int chunks, int* tokens) {
  unsigned long long best = 0;
  for (int i = threadIdx.x; i < chunks; i += kWave) {
    const unsigned long long key = keys[(size_t)blockIdx.x * chunks + i];
    best = key > best ? key : best;
  }
  best = wave_max_u64(best);
  if (threadIdx.x == 0) tokens[blockIdx.x] = best ? (int)greedy_index(best) : -1;
}

int chunks_of(const fah_logits_adjust& a) { return (a.vocab + kChunk - 1) / kChunk; }

}  // namespace

int64_t logits_adjust_workspace(const fah_logits_adjust& a) {
  return a.tokens && a.rows > 0 ? (int64_t)a.rows * chunks_of(a) * 8 : 0;
}

hipError_t launch_logits_adjust(const fah_logits_adjust& a, hipStream_t s) {
  const dim3 grid(chunks_of(a), a.rows);
  auto* keys = a.tokens ? static_cast<unsigned long long*>(a.workspace) : nullptr;
  if (a.type == FAH_TYPE_F32) logits_kernel<float><<<grid, kThreads, 0, s>>>(a, keys);
  else if (a.type == FAH_TYPE_F16) logits_kernel<_Float16><<<grid, kThreads, 0, s>>>(a, keys);
  else logits_kernel<__bf16><<<grid, kThreads, 0, s>>>(a, keys);
  if (keys) choice_kernel<<<a.rows, kWave, 0, s>>>(keys, grid.x, a.tokens);
  return hipGetLastError();
}

}  // namespace fah

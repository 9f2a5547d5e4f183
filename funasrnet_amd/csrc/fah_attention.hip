// Attention of the serving operators: packed causal prompts and single tokens
// behind a shared prefix, grouped heads (fah_packed_attention and
// fah_prefix_attention of the C ABI).
#include "fah_device.h"
#include "fah_internal.h"

#include <hip/hip_bf16.h>

namespace fah {
namespace {

template <typename T>
__device__ __forceinline__ float widen(T v) {
  return (float)v;
}

__device__ __forceinline__ int clamp_int(int v, int low, int high) { return v < low ? low : v > high ? high : v; }

// Running softmax of one query row over keys, a wave per row: lane l holds the
// channels l and l + 64.
template <typename Q, typename K>
struct Row {
  float q[2], o[2], top = -__builtin_inff(), total = 0.0f;
  int size, lane;
  __device__ Row(const Q* query, int n) : size(n), lane(threadIdx.x) {
    for (int i = 0; i < 2; ++i) {
      q[i] = lane + 64 * i < n ? widen(query[lane + 64 * i]) : 0.0f;
      o[i] = 0.0f;
    }
  }
  __device__ void add(const K* k, const K* v, int64_t k_row, int64_t v_row, int count, float scale) {
    for (int t = 0; t < count; ++t) {
      float s = 0.0f;
      for (int i = 0; i < 2; ++i)
        if (lane + 64 * i < size) s += q[i] * widen(k[t * k_row + lane + 64 * i]);
      for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
      s *= scale;
      const float next = s > top || s != s ? s : top;
      const float base = next == -__builtin_inff() ? 0.0f : next;
      const float keep = expf(top - base), p = expf(s - base);
      total = total * keep + p;
      for (int i = 0; i < 2; ++i)
        if (lane + 64 * i < size) o[i] = o[i] * keep + p * widen(v[t * v_row + lane + 64 * i]);
      top = next;
    }
  }
  __device__ void write(Q* out) const {
    for (int i = 0; i < 2; ++i)
      if (lane + 64 * i < size) out[lane + 64 * i] = (Q)(total == 0.0f ? 0.0f : o[i] / total);
  }
};

template <typename Q, typename K>
__global__ __launch_bounds__(64) void packed_rows_kernel(fah_packed_attention a) {
  const int row = blockIdx.x, head = blockIdx.y, kv = head / (a.heads / a.kv_heads);
  int lo = -1, begin = 0, end = 0;
  for (int s = 0; s < a.sequences; ++s) {
    begin = clamp_int(a.query_offsets[s], 0, a.query_rows);
    end = clamp_int(a.query_offsets[s + 1], 0, a.query_rows);
    if (row >= begin && row < end) {
      lo = s;
      break;
    }
  }
  if (lo < 0) return;
  const int* offsets = a.key_offsets ? a.key_offsets : a.query_offsets;
  const int kb = clamp_int(offsets[lo], 0, a.key_rows), ke = clamp_int(offsets[lo + 1], kb, a.key_rows);
  int count = (row - begin) + (ke - kb) - (end - begin) + 1;
  count = clamp_int(count, 0, ke - kb);
  Row<Q, K> r(static_cast<const Q*>(a.query) + row * a.query_row + head * a.query_head, a.head_size);
  r.add(static_cast<const K*>(a.key) + kb * a.key_row + kv * a.key_head,
        static_cast<const K*>(a.value) + kb * a.value_row + kv * a.value_head, a.key_row, a.value_row, count, a.scale);
  r.write(static_cast<Q*>(a.output) + row * a.output_row + head * a.output_head);
}

template <typename Q, typename K>
__global__ __launch_bounds__(64) void prefix_rows_kernel(fah_prefix_attention a) {
  const int s = blockIdx.x, head = blockIdx.y, kv = head / (a.heads / a.kv_heads);
  Row<Q, K> r(static_cast<const Q*>(a.query) + s * a.query_sequence + head * a.query_head, a.head_size);
  r.add(static_cast<const K*>(a.prefix_key) + kv * a.prefix_key_head,
        static_cast<const K*>(a.prefix_value) + kv * a.prefix_value_head, a.prefix_key_row, a.prefix_value_row, a.prefix,
        a.scale);
  r.add(static_cast<const K*>(a.key) + s * a.key_sequence + kv * a.key_head,
        static_cast<const K*>(a.value) + s * a.value_sequence + kv * a.value_head, a.key_row, a.value_row,
        clamp_int(a.lengths[s], 0, a.capacity), a.scale);
  r.write(static_cast<Q*>(a.output) + s * a.output_sequence + head * a.output_head);
}

}  // namespace

bool attention_supported(int heads, int kv_heads, int head_size, int query_type, int cache_type) {
  return heads / kv_heads <= 65535 && head_size % 8 == 0 && head_size <= 128 &&
         ((query_type == FAH_TYPE_F32 && cache_type == FAH_TYPE_F16) ||
          (query_type == FAH_TYPE_F16 && cache_type == FAH_TYPE_F16) ||
          (query_type == FAH_TYPE_BF16 && cache_type == FAH_TYPE_BF16));
}

int64_t packed_attention_workspace(const fah_packed_attention&) { return 0; }
int64_t prefix_attention_workspace(const fah_prefix_attention&) { return 0; }

hipError_t launch_packed_attention(const fah_packed_attention& a, hipStream_t s) {
  const dim3 grid(a.query_rows, a.heads);
  if (a.query_type == FAH_TYPE_F32) packed_rows_kernel<float, _Float16><<<grid, 64, 0, s>>>(a);
  else if (a.query_type == FAH_TYPE_F16) packed_rows_kernel<_Float16, _Float16><<<grid, 64, 0, s>>>(a);
  else packed_rows_kernel<__bf16, __bf16><<<grid, 64, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_prefix_attention(const fah_prefix_attention& a, hipStream_t s) {
  const dim3 grid(a.sequences, a.heads);
  if (a.query_type == FAH_TYPE_F32) prefix_rows_kernel<float, _Float16><<<grid, 64, 0, s>>>(a);
  else if (a.query_type == FAH_TYPE_F16) prefix_rows_kernel<_Float16, _Float16><<<grid, 64, 0, s>>>(a);
  else prefix_rows_kernel<__bf16, __bf16><<<grid, 64, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace fah

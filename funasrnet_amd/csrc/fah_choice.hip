// Logits under penalties for repeated tokens, biases and grammar masks, and the
// greedy choice after them (fah_logits_adjust of the C ABI).
//
// logits_kernel: a workgroup takes some chunks of one row's tokens. It holds the
// row's lists in registers and notes what they say of its chunks in a table in
// LDS while the first logits, 16 bytes a lane, are on their way: they name few
// tokens, so the stream itself only carries the mask, the running maximum and
// one bit a token that asks for the table. choice_kernel takes the largest over
// a row's workgroups.
#include "fah_device.h"
#include "fah_internal.h"

#include <algorithm>

namespace fah {
namespace {

constexpr int kThreads = 256;
constexpr float kInf = __builtin_inff();

// Values of T in 16 bytes, and back.
template <typename T>
struct alignas(16) Vec {
  static constexpr int kCount = 16 / sizeof(T);
  T v[kCount];
};

// 16 bytes past the caches: adjusted logits are not read again here, and would
// push the rows to come out of them. 256 rows of 151936 in bf16: 33.5 us where the
// inputs are in the 256 MB cache (34.7 with plain stores, 39 with loads past the
// caches as well), 41 where they are not (42.4). 64 rows in fp32 18.9 and 24.4
// (20, 26.3), 16 rows 11 (11.7), one row 7.5 either way. Whoever reads the adjusted
// logits next pays for it: a call and a copy of them 61.5 and 68.5 us for 256 rows
// (57.3, 70), 35.7 and 39.5 for 64 (32.2, 36.8), 16.6 for 16 (15.9 to 17.7).
template <typename T>
__device__ __forceinline__ void stream_out(T* p, const Vec<T>& v) {
  using Bits = __attribute__((ext_vector_type(4))) unsigned;
  __builtin_nontemporal_store(__builtin_bit_cast(Bits, v), reinterpret_cast<Bits*>(p));
}

// This thread's share of a list, every kThreads-th entry: the first kHeld in
// registers, requested together, the others when they are looked at.
template <int kHeld>
struct List {
  const int* at;
  int count, held[kHeld];
  __device__ __forceinline__ List(const int* list, int n) : at(list), count(n) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int i = threadIdx.x + k * kThreads;
      held[k] = i < count ? at[i] : -1;
    }
  }
  // f(token, entry)
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll
    for (int k = 0; k < kHeld; ++k) f(held[k], (int)threadIdx.x + k * kThreads);
    for (int i = threadIdx.x + kHeld * kThreads; i < count; i += kThreads) f(at[i], i);
  }
};

__device__ __forceinline__ int bounded(const int* counts, int row, int capacity) {
  const int n = counts ? counts[row] : capacity;
  return n < 0 ? 0 : n < capacity ? n : capacity;
}

// Chunks that a workgroup takes at most.
constexpr int kRun = 4;

// Tokens of a row are counted from the 16-byte boundary at or before its first
// logit: place u = token + lead, so that groups of Vec::kCount places are whole
// 16-byte loads whatever the row's alignment. A workgroup takes `run` chunks of
// kChunk places, a group a thread, the next chunk's on their way meanwhile.
template <typename T>
__global__ __launch_bounds__(kThreads, 8) void logits_kernel(fah_logits_adjust a, int run, unsigned long long* keys) {
  constexpr int V = Vec<T>::kCount, kChunk = kThreads * V, kEach = (kRun * V + 31) / 32, kWords = kThreads * kEach;
  // What the lists say of some places, the window. `named` has a bit for each
  // that they name; each has a slot: `seen` the count behind the prompt and in
  // bit 31 whether it is in the history at all; `entry` its last bias entry plus
  // one. A window of one chunk has a slot a place. For several chunks at once the
  // slots are those of the named places in turn, `start` where each word's
  // begin: the lists are looked through once (256 rows of 151936 in bf16, stores
  // through the caches: 47.6 us, 51 chunk by chunk). Integer atomics: no order
  // changes the result.
  struct Table {
    unsigned seen[kChunk], entry[kChunk], named[kWords], start[kWords];
  };
  __shared__ __align__(16) Table table;
  __shared__ unsigned sums[kThreads / kWave];
  __shared__ unsigned long long part[kThreads / kWave];
  const int row = blockIdx.y, tid = threadIdx.x;
  const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
  T* out = static_cast<T*>(a.output) + row * a.output_stride;
  const int lead = (int)(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T));
  const bool out_alike = reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T) == (unsigned)lead;
  const uint32_t* mask = nullptr;
  if (a.mask_rows) {
    const int m = a.mask_index ? a.mask_index[row] : a.mask_rows == 1 ? 0 : row;
    if (m >= 0 && m < a.mask_rows) mask = a.masks + m * a.mask_stride;
  }

  // A thread's logits and mask bits of a chunk; t: the token of its first place.
  struct Group {
    Vec<T> x;
    uint32_t low, high;
  };
  auto load = [&](int t) {
    Group g{};
    g.low = g.high = ~0u;
    if (t >= 0 && t + V <= a.vocab) {
      g.x = *reinterpret_cast<const Vec<T>*>(in + t);
      if (mask) {
        g.low = mask[t >> 5];
        g.high = mask[(t + V - 1) >> 5];
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) g.x.v[e] = t + e >= 0 && t + e < a.vocab ? in[t + e] : (T)0.0f;
      if (mask && t + V > 0 && t < a.vocab) {
        g.low = mask[t >= 0 ? t >> 5 : 0];
        g.high = mask[(t + V <= a.vocab ? t + V - 1 : a.vocab - 1) >> 5];
      }
    }
    return g;
  };
  // Bit e: token t + e is allowed (low: the mask's word with token t, or with
  // token 0; high: the one with the group's last token).
  auto allowed = [&](const Group& g, int t) {
    const int shift = t & 31;
    if (t < 0) return g.low << -t;
    return shift + V > 32 ? g.low >> shift | g.high << (32 - shift) : g.low >> shift;
  };
  int first = (int)blockIdx.x * run * kChunk - lead;  // token of the chunk's place 0
  Group next = load(first + tid * V);

  const int history_count = a.history_capacity ? bounded(a.history_counts, row, a.history_capacity) : 0;
  const int bias_count = a.bias_capacity ? bounded(a.bias_counts, row, a.bias_capacity) : 0;
  const bool listed = history_count > 0 || bias_count > 0;
  const int prompt = a.prompt_counts ? a.prompt_counts[row] : 0;
  const float repetition = a.repetition ? a.repetition[row] : 1.0f;
  const float presence = a.presence ? a.presence[row] : 0.0f;
  const float frequency = a.frequency ? a.frequency[row] : 0.0f;
  const float* bias = a.bias_values + row * a.bias_stride;
  const List<4> history(a.history + row * a.history_stride, history_count);
  const List<2> biases(a.bias_tokens + row * a.bias_stride, bias_count);
  auto adjust = [&](float v, int slot) {
    const unsigned w = table.seen[slot], e = table.entry[slot], n = w & 0x7fffffffu;
    if (w) v = v > 0.0f ? v / repetition : v * repetition;
    if (n) {
      v = v - frequency * (float)n;
      v = v - presence;
    }
    return e ? v + bias[e - 1] : v;
  };
  auto below = [](unsigned word, int bit) { return __popc(word & ((1u << bit) - 1)); };
  // Notes what the lists say of the places from token `first` on. False, and
  // nothing noted: they name more than there are slots (never in one chunk).
  auto note = [&](int first, int places, bool ranked) {
    // f(place, entry) for the list's entries in the window.
    auto within = [&](const auto& list, auto&& f) {
      list.each([&](int token, int i) {
        const unsigned u = (unsigned)(token - first);
        if (token >= 0 && token < a.vocab && u < (unsigned)places) f((int)u, i);
      });
    };
    auto name = [&](int u, int) { atomicOr(&table.named[u >> 5], 1u << (u & 31)); };
    const int entries = (history_count < kChunk ? history_count : kChunk) + (bias_count < kChunk ? bias_count : kChunk);
    const int slots = ranked && entries < kChunk ? entries : kChunk;
#pragma unroll
    for (int j = 0; j < kEach; ++j) table.named[tid * kEach + j] = 0;
    for (int i = tid; 4 * i < slots; i += kThreads) reinterpret_cast<uint4*>(table.seen)[i] = reinterpret_cast<uint4*>(table.entry)[i] = uint4{0, 0, 0, 0};
    lds_barrier();
    if (ranked) {
      within(history, name);
      within(biases, name);
      lds_barrier();
      const int lane = tid % kWave;
      int mine = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) mine += __popc(table.named[tid * kEach + j]);
      int through = mine;
#pragma unroll
      for (int x = 1; x < kWave; x *= 2) {
        const int other = __shfl_up(through, x, kWave);
        through += lane >= x ? other : 0;
      }
      if (lane == kWave - 1) sums[tid / kWave] = through;
      lds_barrier();
      int before = 0, total = 0;
#pragma unroll
      for (int w = 0; w < kThreads / kWave; ++w) {
        before += w < tid / kWave ? sums[w] : 0;
        total += sums[w];
      }
      if (total > kChunk) return false;
      int start = before + through - mine;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        table.start[tid * kEach + j] = start;
        start += __popc(table.named[tid * kEach + j]);
      }
      lds_barrier();
    }
    auto slot = [&](int u) { return ranked ? table.start[u >> 5] + below(table.named[u >> 5], u & 31) : u; };
    within(history, [&](int u, int i) {
      if (!ranked) name(u, i);
      const int at = slot(u);
      atomicOr(&table.seen[at], 0x80000000u);
      if (i >= prompt) atomicAdd(&table.seen[at], 1u);
    });
    within(biases, [&](int u, int i) {
      if (!ranked) name(u, i);
      atomicMax(&table.entry[slot(u)], (unsigned)i + 1);
    });
    lds_barrier();
    return true;
  };
  // (16 rows of 151936 in fp32, two chunks a workgroup: 12.4 us so, 11.6 else.)
  const bool ranked = listed && run > 2 && note(first, run * kChunk, true);

  float top = -kInf;  // NaN and -inf never replace it
  int at = -1;
  for (int c = 0; c < run && first < a.vocab; ++c, first += kChunk) {
    const int t = first + tid * V;
    Group g = next;
    if (c + 1 < run) next = load(t + kChunk);
    if (listed) {
      if (!ranked) {
        if (c > 0) lds_barrier();  // the table's readers are done
        note(first, kChunk, false);
      }
      const int u = (ranked ? c * kChunk : 0) + tid * V;  // of the window
      const unsigned word = table.named[u >> 5], bits = word >> (u & 31) & ((1u << V) - 1);
      if (bits) {
        const int slot = ranked ? table.start[u >> 5] + below(word, u & 31) : u;
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (bits >> e & 1) g.x.v[e] = (T)adjust((float)g.x.v[e], slot + (ranked ? below(bits, e) : e));
      }
    }
    const uint32_t open = allowed(g, t);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (!(open >> e & 1)) g.x.v[e] = (T)-kInf;
    if (t >= 0 && t + V <= a.vocab) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float y = (float)g.x.v[e];
        if (y > top) {
          top = y;
          at = t + e;
        }
      }
      if (out_alike) {
        stream_out(out + t, g.x);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) out[t + e] = g.x.v[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (t + e >= 0 && t + e < a.vocab) {
          const float y = (float)g.x.v[e];
          out[t + e] = g.x.v[e];
          if (y > top) {
            top = y;
            at = t + e;
          }
        }
    }
  }
  if (!keys) return;
  unsigned long long best = wave_max_u64(at < 0 ? 0ull : greedy_key(top, (uint32_t)at));
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

// Chunks a workgroup takes, and the workgroups of a row.
struct ChoiceCut {
  int run, groups;
};

// As many workgroups as the chip holds at once (8 a CU) have one chunk each;
// with more, a workgroup takes up to four, so that looking the lists up once
// serves them all (256 rows of 151936 in bf16: 33.4 us with four chunks, 35.3
// with three or five, 35 with eight).
constexpr int kGroups = 2048;

ChoiceCut choice_cut(const fah_logits_adjust& a) {
  const int V = a.type == FAH_TYPE_F32 ? 4 : 8;
  const int64_t chunks = ((int64_t)a.vocab + V - 1 + kThreads * V - 1) / (kThreads * V);
  const int run = (int)std::max<int64_t>(1, std::min<int64_t>((chunks * a.rows + kGroups - 1) / kGroups, kRun));
  return {run, (int)((chunks + run - 1) / run)};
}

}  // namespace

int64_t logits_adjust_workspace(const fah_logits_adjust& a) {
  return a.tokens && a.rows > 0 ? (int64_t)a.rows * choice_cut(a).groups * 8 : 0;
}

hipError_t launch_logits_adjust(const fah_logits_adjust& a, hipStream_t s) {
  const ChoiceCut c = choice_cut(a);
  const dim3 grid(c.groups, a.rows);
  auto* keys = a.tokens ? static_cast<unsigned long long*>(a.workspace) : nullptr;
  if (a.type == FAH_TYPE_F32) logits_kernel<float><<<grid, kThreads, 0, s>>>(a, c.run, keys);
  else if (a.type == FAH_TYPE_F16) logits_kernel<_Float16><<<grid, kThreads, 0, s>>>(a, c.run, keys);
  else logits_kernel<__bf16><<<grid, kThreads, 0, s>>>(a, c.run, keys);
  if (keys) choice_kernel<<<a.rows, kWave, 0, s>>>(keys, c.groups, a.tokens);
  return hipGetLastError();
}

}  // namespace fah

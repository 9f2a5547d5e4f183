// Attention of the serving operators: packed causal prompts and single tokens
// behind a shared prefix, grouped heads (fah_packed_attention and
// fah_prefix_attention of the C ABI).
//
// Per row, o = sum_j 2^(c s_j - r) v_j / sum_j 2^(c s_j - r) with s = q k and
// c = scale log2(e), in one pass over the keys: r is a reference that follows
// the largest score seen, and sums made with an earlier one are scaled when it
// moves. A row is a (token, query head of the K/V head's group) pair, so a tile
// of K and V serves all heads of a group.
//
// Layout. A wave has 32 rows. It forms S^T = K Q^T with 32 x 32 x 16 matrix
// instructions (keys x rows), whose result leaves each lane with 16 keys of one
// row: the softmax is per lane but for one exchange between the wave's halves,
// and the weights are, as they stand, the B operand of O^T = V^T P^T, whose sums
// again belong to the lane's row. Which key a B element is, is free as long as
// V^T's A operand names the same: it is read from the row-major tile by the
// transposing LDS read, four keys by 16 channels at a time. K and V tiles come
// by direct loads into LDS, 16 bytes a lane, in a swizzled order (0 bank
// conflicts counted).
//
// Rounding. Scores, references, totals and sums are fp32. Weights are rounded
// once to the values' type, as the matrix instructions take them (totals are of
// the unrounded ones); it is the only rounding that fp32 arithmetic on the same
// inputs has not, and adds to the error what rounding the output does: measured
// 2.3e-3 of the result in bf16 against 1.7e-3. fp32 queries, and the weights of
// their rows, are split into two fp16 parts and take two products each: 3e-7.
// (Second parts may be 0 or of the other sign, which makes infinite keys and
// values NaN: the rows are formed again in slow_row.)
//
// What bounds it: long prompts the matrix instructions and the card's power
// (8192 rows of 32/8 heads in bf16: 525 us, 1.05 PFLOP/s, matrix units 52% busy
// at 1.9 GHz; a library product of 8192^3 reaches 1.21); own cache rows of a
// large batch the memory (256 sequences: 121 us, 5.5 TB/s); everything small the
// chain offsets, queries and first tile, one pass, epilogue: 5 to 6 us.
#include "fah_device.h"
#include "fah_internal.h"

#include <algorithm>
#include <type_traits>

namespace fah {
namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using s16x8 = __attribute__((ext_vector_type(8))) short;
using LdsTr = s16x4 __attribute__((address_space(3))) *;
using LdsFrag = s16x8 __attribute__((address_space(3))) *;

constexpr int kThreads = 256;
constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;
// Weights are held as 2^(score - reference + kLift). The reference only moves
// when a row's largest score has risen by more than kSlack. For fp16 values they
// are at most 2^(kLift + kSlack) = 2^14, which fp16 holds, so that small weights
// keep fp16's full precision down to 2^-22 of the largest one. bf16 has the range
// of fp32, and so have its values: there weights are at most 2^-18, so that the
// sums of 2^17 of the largest values stay finite (values below 2^-102 lose bits
// instead). Partial sums keep the lift, which the join divides out.
constexpr float kSlack = 6.0f;
template <typename K>
constexpr float kLift = std::is_same_v<K, __bf16> ? -24.0f : 8.0f;
// A weight's exponent is formed as s c - (reference c) in one fma, which is off
// by the rounding of the reference's product, the same for all of a row. From
// this size on that rounding is a whole power of two and more, and weights would
// overflow or vanish: there it is (s - reference) c, one instruction a score more
// (not everywhere, for the vector units are half of what bounds long prompts).
constexpr float kFar = 8388608.0f;

__device__ __forceinline__ int clamp_int(int v, int low, int high) { return v < low ? low : v > high ? high : v; }

// a * b + c of 32 x 32 x 16 blocks, 16-bit operands of type T.
template <typename T>
__device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (std::is_same_v<T, __bf16>)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The value of lane l ^ 32.
__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return u2f(threadIdx.x & 32 ? r[0] : r[1]);
}

// What one workgroup attends: `rows` rows of one K/V head over the keys
// [begin, end). A row is a token and one of the group's query heads, heads
// first; the first row is head head0 of token 0.
template <typename Q, typename K>
struct Task {
  const Q* q;                // token 0, the K/V head's first query head
  int64_t q_token, q_head;   // strides
  const K *k, *v;            // key 0
  unsigned k_row, v_row;     // strides
  int rows, group, head0;
  float group_inverse;
  int begin, end;            // keys
  int first_limit;           // token 0 sees the keys below this; per token one more if causal
  bool causal;
  // Row r's token and head. r + head0 is below 65536 + 128: the product's error,
  // 2^-22 of it, is far below the half step that it is from a whole number.
  __device__ __forceinline__ int token(int r) const { return (int)((float)(r + head0) * group_inverse + 0.5f * group_inverse); }
  __device__ __forceinline__ int head(int r) const { return r + head0 - token(r) * group; }
  __device__ __forceinline__ int limit(int r) const {
    const int n = causal ? first_limit + token(r) : first_limit;
    return n < end ? n : end;
  }
  __device__ __forceinline__ const Q* query(int r) const { return q + token(r) * q_token + head(r) * q_head; }
};

// Where it goes: the finished rows, or partial ones for a join: sums and total
// of the weights 2^(c (s - mark) + kLift), and the mark, a score in units of
// mark_unit.
template <typename Q>
struct Sink {
  Q* out;                    // token 0, the K/V head's first query head; null: partial
  int64_t o_token, o_head;
  float* sums;               // [rows][D]
  float* marks;              // [rows][2]
};

// Marks are scores q k times the scale's power of two: exact, and neither too
// large nor too small where the scaled scores are not. What is left of the scale,
// as exponents of two, is mark_exponent.
__device__ __forceinline__ float mark_unit(float scale) { return fmaxf(u2f(f2u(scale) & 0x7f800000u), 0x1p-126f); }
__device__ __forceinline__ float mark_exponent(float scale) { return scale / mark_unit(scale) * kLog2e; }

template <int D>
struct Tile {
  static constexpr int kChunks = D / 8;               // 16-byte chunks a row
  static constexpr int kRowsLoad = 64 / kChunks;      // rows a wave loads at a time
  static constexpr int kRowBytes = 2 * D;
  // Chunk c of row r sits at place c ^ swizzle(r): fragment reads (16 rows, one
  // chunk) of keys and transposing reads (4 rows, 64 bytes) of values then
  // touch all 64 banks.
  __device__ static int key_swizzle(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }
  __device__ static int value_swizzle(int r) { return D == 128 ? (r & 3) << 2 : (r & 2) << 1; }
};

// A value that all lanes share, in scalar registers.
__device__ __forceinline__ unsigned uniform(unsigned v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const void* uniform(const void* p) {
  const uint64_t v = (uint64_t)p;
  return (const void*)((uint64_t)uniform((unsigned)(v >> 32)) << 32 | uniform((unsigned)v));
}

// 16 bytes a lane from base + offset to LDS at `to` + 16 lane. Inline, because
// the compiler would wait for a load into LDS before any read of LDS: the
// tiles' reads are ordered by wait_loads and a barrier instead. (It has no
// register that it writes; a load into M0's place needs one wait state.) ONCE:
// past the caches.
template <bool ONCE>
__device__ __forceinline__ void load_lds(const void* base, unsigned offset, unsigned to) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(uniform(to)), "v"(offset), "s"(uniform(base)) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(uniform(to)), "v"(offset), "s"(uniform(base)) : "memory");
}
template <bool ONCE>
__device__ __forceinline__ void load_lds(const void* from, unsigned to) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(uniform(to)), "v"(from) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(uniform(to)), "v"(from) : "memory");
}
// Every load of this wave is done (vmcnt 0, nothing else waited for). A barrier
// follows: reads of LDS may move up to it but not before it.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// All but the last N loads are done; reads of LDS stay behind it.
template <int N>
__device__ __forceinline__ void wait_loads_but() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// This wave's reads of LDS are done: their place may be loaded again.
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// Loads tiles of ROWS keys or values by the waves w of W, kRowsLoad rows a load.
// A lane's place in the source repeats, but for the base, after the rows whose
// swizzles differ: its offsets are kept, and the base moves in scalar registers.
template <typename K, int D, int ROWS, int W, bool VALUES, bool ONCE>
struct Loader {
  using T = Tile<D>;
  static constexpr int kLoads = ROWS / T::kRowsLoad / W, kStep = W * T::kRowsLoad;
  static constexpr int kPeriod = VALUES ? 4 : 16;      // rows after which the swizzle repeats
  static constexpr int kKinds = kStep >= kPeriod ? 1 : kPeriod / kStep;
  static_assert(kLoads >= 1 && kLoads % kKinds == 0);
  unsigned offset[kKinds];
  unsigned to;       // LDS place of the wave's first load
  int row0;          // its first row in the tile

  __device__ static int chunk(int r) {
    return (int)(threadIdx.x & 63) % T::kChunks ^ (VALUES ? T::value_swizzle(r) : T::key_swizzle(r));
  }
  __device__ Loader(const unsigned char* tile, unsigned stride, int w)
      : to(lds_address(tile) + w * 1024), row0(w * T::kRowsLoad) {
#pragma unroll
    for (int j = 0; j < kKinds; ++j) {
      const int r = row0 + j * kStep + (threadIdx.x & 63) / T::kChunks;
      offset[j] = (unsigned)r * stride * 2 + chunk(r) * 16;
    }
  }
  // Rows first ..: `shift` is the place of this buffer behind the constructor's.
  __device__ __forceinline__ void load(const K* base, unsigned stride, int first, int last, unsigned shift, int size) const {
    const bool whole = first + ROWS - 1 <= last && size == D;
    if (whole) {
      const K* at = base + (int64_t)first * stride;
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        load_lds<ONCE>(at + (int64_t)(i / kKinds * kKinds * kStep) * stride, offset[i % kKinds], to + shift + i * W * 1024);
    } else {
      // Rows past `last` repeat it (their scores are masked); places behind
      // head_size stay as they are (zero).
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int r = row0 + i * kStep + (threadIdx.x & 63) / T::kChunks;
        const int row = first + r < last ? first + r : last;
        if (chunk(r) * 8 < size) load_lds<ONCE>(base + (int64_t)row * stride + chunk(r) * 8, to + shift + i * W * 1024);
      }
    }
  }
};

// Whether a 16-bit value is infinite or NaN.
template <typename K>
__device__ __forceinline__ bool not_finite(K v) {
  constexpr unsigned kExponent = std::is_same_v<K, __bf16> ? 0x7f80 : 0x7c00;
  return (__builtin_bit_cast(unsigned short, v) & kExponent) == kExponent;
}

// A row that slow_row formed: the lane's channels 2 lane and 2 lane + 1, finished,
// which of them stand in for the row's own, and its mark and total (see Sink).
struct SlowRow {
  float value[2], mark, total;
  bool bad[2];
};

// A row by one wave, only keys that it sees read: all channels, or those that
// infinite or NaN values between `masked` and `last` can have reached, which the
// row's tiles masked or took in two parts. A key a lane for the scores, two
// channels a lane for the values; over once every channel asked for is NaN. (24
// prompts of 5014 rows, fp16, every value NaN: 1.1 ms, 12 key by key; one channel
// infinite everywhere 5.4; the first key alone 0.1.)
template <typename Q, typename K>
__device__ __noinline__ SlowRow slow_row(const Q* q, const K* k_rows, const K* v_rows, unsigned k_row, unsigned v_row, int begin,
                                         int lim, bool all, int masked, int last, int size, float scale) {
  const int lane = threadIdx.x & 63, d = 2 * lane;
  const bool holds = d < size;  // (sizes are multiples of 8)
  bool bad[2] = {all && holds, all && holds};
  for (int first = masked; !all && first <= last; first += 16) {
#pragma unroll 4
    for (int key = first; key < first + 16; ++key)
      if (holds && key <= last)
        for (int i = 0; i < 2; ++i) bad[i] |= not_finite(v_rows[(int64_t)key * v_row + d + i]);
    if (__builtin_amdgcn_ballot_w64(holds && !(bad[0] && bad[1])) == 0) break;
  }
  if (__builtin_amdgcn_ballot_w64(bad[0] || bad[1]) == 0) return {};
  const float unit = mark_unit(scale), c = mark_exponent(scale);
  float sum[2] = {}, top = -kInf, total = 0.0f;
  for (int first = begin; first < lim; first += 64) {
    const int n = lim - first < 64 ? lim - first : 64;
    float s = 0.0f;
    const K* k = k_rows + (int64_t)(first + (lane < n ? lane : n - 1)) * k_row;
    for (int e = 0; e < size; e += 8) {
      alignas(16) K part[8];
      *reinterpret_cast<uint4*>(part) = *reinterpret_cast<const uint4*>(k + e);
#pragma unroll
      for (int i = 0; i < 8; ++i) s += (float)q[e + i] * unit * (float)part[i];
    }
    if (lane >= n) s = -kInf;
    float next = fmaxf(top, s);  // (NaN scores make the total NaN below)
    for (int x = 32; x >= 1; x >>= 1) next = fmaxf(next, __shfl_xor(next, x, 64));
    const float base = next == -kInf ? 0.0f : next, keep = __builtin_amdgcn_exp2f((top - base) * c);
    const float p = lane < n ? __builtin_amdgcn_exp2f((s - base) * c + kLift<K>) : 0.0f;
    float add = p;
    for (int x = 32; x >= 1; x >>= 1) add += __shfl_xor(add, x, 64);
    total = total * keep + add;
    sum[0] *= keep;
    sum[1] *= keep;
    const K* v = v_rows + (int64_t)first * v_row + d;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const float w = __shfl(p, j, 64);
      if (holds) {
        sum[0] += w * (float)v[(int64_t)j * v_row];
        sum[1] += w * (float)v[(int64_t)j * v_row + 1];
      }
    }
    top = next;
    bool open = false;
    for (int i = 0; i < 2; ++i) open |= bad[i] && sum[i] == sum[i];
    if (total != total || (total != 0.0f && __builtin_amdgcn_ballot_w64(open) == 0)) break;
  }
  if (total == 0.0f) sum[0] = sum[1] = 0.0f;
  else sum[0] /= total, sum[1] /= total;
  return {{sum[0], sum[1]}, top, total, {bad[0], bad[1]}};
}

// A 16-bit type's packed pair.
template <typename K>
__device__ __forceinline__ unsigned pack2(float a, float b) {
  if constexpr (std::is_same_v<K, __bf16>) {
    using V = __attribute__((ext_vector_type(2))) __bf16;
    return __builtin_bit_cast(unsigned, V{(__bf16)a, (__bf16)b});
  } else {
    using V = __attribute__((ext_vector_type(2))) _Float16;
    return __builtin_bit_cast(unsigned, V{(_Float16)a, (_Float16)b});
  }
}

// The workgroup's waves as WR groups of 32 rows times WK shares of each key
// tile; a wave takes NK keys of a tile. Used as 4 x 1 (64 keys a wave), 2 x 2 and
// 1 x 4 (32 keys): the first loads the fewest bytes a product, the last gives few
// rows the most waves. Eight waves (2 x 4, 4 x 2, 1 x 8) were slower everywhere,
// and so were scores formed a tile ahead of the weights (256 registers do not
// hold both: 8192 rows 675 us).
template <typename Q, typename K, int D, int WR, int WK, int NK, bool ONCE = false>
struct Core {
  static constexpr int kWaves = WR * WK, kThreads = 64 * kWaves, BM = 32 * WR, TR = WK * NK;
  static constexpr int kTileBytes = TR * 2 * D;        // keys, or values
  // One group of rows: each wave's keys and values are its own, in one buffer.
  // Several groups share them, in two.
  static constexpr int kTiles = (WR == 1 ? 2 : 4) * kTileBytes, kSums = WK == 1 ? 0 : kWaves * 32 * D * 4;
  static constexpr int kArea = kTiles > kSums ? kTiles : kSums;
  // Behind the area: one group of rows shares its queries' fragments there, and
  // at the end the waves' references and totals stand there.
  static constexpr bool kSplit = std::is_same_v<Q, float>;
  static constexpr int kSteps = D / 16, kShared = WR == 1 ? kSteps * 1024 * (kSplit ? 2 : 1) : 0, kMarks = 8 * 32 * (kWaves + WR) + 4 * kWaves;
  static constexpr int kLds = kArea + (kShared > kMarks ? kShared : kMarks);

  // slow_row for row r of the workgroup with this total. Masked places: from the
  // row's first unseen key on, and the last key, which is repeated behind it.
  __device__ static SlowRow repaired(const Task<Q, K>& t, int r, float total, int masked_last, int size, float scale) {
    const int lim = t.limit(r), from = kSplit ? t.begin : lim < t.end - 1 ? lim : t.end - 1;
    return slow_row(t.query(r), t.k, t.v, t.k_row, t.v_row, t.begin, lim, kSplit && total != total,
                    from > t.begin ? from : t.begin, masked_last, size, scale);
  }

  // lds: one or two buffers of a key tile and a value tile; at the end the
  // waves' sums. Behind them marks: [kWaves][32][2] of the waves, then [BM][2]
  // of the rows, then whether each wave masked scores.
  __device__ static void run(const Task<Q, K>& t, const Sink<Q>& sink, int size, float scale, unsigned char* lds) {
    float* marks = reinterpret_cast<float*>(lds + kArea);
    using T = Tile<D>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, col = lane & 31;
    const int wr = wave / WK, wk = wave % WK;
    const int my_row = wr * 32 + col;
    const bool valid = my_row < t.rows;
    const int lim = valid ? t.limit(my_row) : 0;
    const int wave_rows = clamp_int(t.rows - wr * 32, 0, 32);
    const int lim_low = wave_rows ? (int)uniform(t.limit(wr * 32)) : 0;
    const int lim_high = wave_rows ? (int)uniform(t.limit(wr * 32 + wave_rows - 1)) : 0;
    const int end = (int)uniform(t.limit(t.rows - 1));  // of the workgroup
    const int last = t.end - 1;

    if (D != size) {
      for (int i = tid; i < kTiles / 16; i += kThreads) reinterpret_cast<uint4*>(lds)[i] = uint4{0, 0, 0, 0};
      __syncthreads();
    }
    constexpr int kOwn = WR == 1 ? NK : TR, kLoaders = WR == 1 ? 1 : kWaves;
    const int own = WR == 1 ? wave * NK : 0, loader = WR == 1 ? 0 : wave;
    using KeyLoader = Loader<K, D, kOwn, kLoaders, false, ONCE>;
    using ValueLoader = Loader<K, D, kOwn, kLoaders, true, ONCE>;
    const KeyLoader key_loader(lds + own * T::kRowBytes, t.k_row, loader);
    const ValueLoader value_loader(lds + kTileBytes + own * T::kRowBytes, t.v_row, loader);
    // The wave's first key, and the end of those that its rows see.
    const int wave_begin = t.begin + wk * NK, wave_end = lim_high;

    // Queries: the B operand, lane (row col, channels 16 s + 8 half ..), requested
    // ahead of the first tile and looked at when both are here. fp32 queries are
    // scaled by a power of two to below 2^14 and split into two fp16 parts (22
    // bits; the scale keeps the second part normal). Waves that have the same
    // rows read a part of the channels each and share the fragments: four times
    // 16 loads that touch 32 rows each held the first tile up (a prompt of 750
    // rows spent 6000 cycles there).
    constexpr int kMine = WR == 1 ? kSteps / kWaves : kSteps;
    const int first_step = WR == 1 ? wave * kMine : 0;
    s16x8 part[kSplit ? 2 : 1][kMine];
    f32x4 raw[kSplit ? kMine : 1][2];
    float c = scale * kLog2e, unlift = 1.0f;  // (of a score of lifted queries)
    {
      const Q* q = t.query(valid ? my_row : 0);
#pragma unroll
      for (int s = 0; s < kMine; ++s) {
        // (Channels behind head_size are asked for at 0, and cleared below.)
        int d = 16 * (first_step + s) + 8 * half;
        d = d < size ? d : 0;
        if constexpr (kSplit) {
          raw[s][0] = *reinterpret_cast<const f32x4*>(q + d);
          raw[s][1] = *reinterpret_cast<const f32x4*>(q + d + 4);
        } else {
          part[0][s] = *reinterpret_cast<const s16x8*>(q + d);
        }
      }
    }
    if (WR == 1 ? wave_begin < wave_end : t.begin < end) {
      key_loader.load(t.k, t.k_row, t.begin + own, last, 0, size);
      value_loader.load(t.v, t.v_row, t.begin + own, last, 0, size);
    }
    wait_loads();  // of the queries, as the compiler must know
    if (D != size) {
#pragma unroll
      for (int s = 0; s < kMine; ++s)
        if (16 * (first_step + s) + 8 * half >= size) {
          if constexpr (kSplit) raw[s][0] = raw[s][1] = f32x4{};
          else part[0][s] = s16x8{};
        }
    }
    if constexpr (kSplit) {
      float most = 0.0f;
#pragma unroll
      for (int s = 0; s < kMine; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(raw[s][j >> 2][j & 3]));
      most = fmaxf(most, other_half(most));
      if constexpr (WR == 1) {
        if (half == 0) marks[wave * 32 + col] = most;
        lds_barrier();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) most = fmaxf(most, marks[w * 32 + col]);
        lds_barrier();
      }
      // With an infinity in it the row's scores are infinite or NaN whatever the
      // second parts hold: they are 0, for infinity - infinity is not.
      const int e = (int)(f2u(most) >> 23) - 127;
      const int up = clamp_int(13 - e, -114, 126);
      const float lift = u2f((unsigned)(up + 127) << 23);
#pragma unroll
      for (int s = 0; s < kMine; ++s) {
        f16x8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = raw[s][j >> 2][j & 3] * lift;
          hi[j] = (_Float16)v;
          lo[j] = (_Float16)(e == 128 ? 0.0f : v - (float)hi[j]);
        }
        part[0][s] = __builtin_bit_cast(s16x8, hi);
        part[kSplit ? 1 : 0][s] = __builtin_bit_cast(s16x8, lo);
      }
      unlift = u2f((unsigned)(127 - up) << 23);
      c = fminf(fmaxf(c * unlift, 1.2e-38f), 3.4e38f);
    }
    s16x8 qf[kSplit ? 2 : 1][kSteps];
    if constexpr (WR == 1) {
      s16x8* shared = reinterpret_cast<s16x8*>(lds + kArea) + lane;
#pragma unroll
      for (int p = 0; p < (kSplit ? 2 : 1); ++p)
#pragma unroll
        for (int s = 0; s < kMine; ++s) shared[(p * kSteps + first_step + s) * 64] = part[p][s];
      lds_barrier();
#pragma unroll
      for (int p = 0; p < (kSplit ? 2 : 1); ++p)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) qf[p][s] = shared[(p * kSteps + s) * 64];
      lds_barrier();  // the marks take their place
    } else {
#pragma unroll
      for (int p = 0; p < (kSplit ? 2 : 1); ++p)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) qf[p][s] = part[p][WR == 1 ? 0 : s];
    }

    f32x16 acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = f32x16{};
    float ref = -kInf, ref_c = -kInf, total = 0.0f;  // the reference, a score, and its product with c
    bool masked = false, any_far = false;  // any_far: a row's reference is beyond kFar
    // What a weight's exponent has over (s - reference) c + kLift.
    auto over = [&](float x, float x_c) { return fabsf(x_c) < kFar ? __builtin_fmaf(x, c, -x_c) : 0.0f; };

    // Fragment places within a tile. Keys: lane's row, chunk 2 s + half.
    // Values: lane 16 g + i of a half reads row i / 4 of four, 8 bytes of the
    // 32 that are channels 16 g .. 16 g + 15, and gets channel i of the four rows.
    const int key_at = (wk * NK + col) * T::kRowBytes, key_sw = T::key_swizzle(col);
    const int vi = lane & 15, vg = (lane >> 4) & 1;
    const int value_at = (wk * NK + 4 * half + vi / 4) * T::kRowBytes + (vi & 1) * 8;
    const int value_sw = T::value_swizzle(vi / 4), value_chunk = 2 * vg + ((vi & 3) >> 1);

    f32x16 s[NK / 32];
    auto score = [&](int shift) {
      const unsigned char* kt = lds + shift;
#pragma unroll
      for (int b = 0; b < NK / 32; ++b) s[b] = f32x16{};
#pragma unroll
      for (int step = 0; step < kSteps; ++step)
#pragma unroll
        for (int b = 0; b < NK / 32; ++b) {
          const s16x8 kf = *(LdsFrag)(kt + key_at + b * 32 * T::kRowBytes + (((2 * step + half) ^ key_sw) << 4));
          s[b] = mfma<K>(kf, qf[0][step], s[b]);
          if constexpr (kSplit) s[b] = mfma<K>(kf, qf[kSplit ? 1 : 0][step], s[b]);
        }
    };
    // Scores to weights, in place.
    auto weigh = [&](int key0) {
      if (key0 + NK > lim_low) {
        masked = true;
        const int room = lim - key0 - 4 * half;
#pragma unroll
        for (int b = 0; b < NK / 32; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[b][i] = 32 * b + 8 * (i >> 2) + (i & 3) < room ? s[b][i] : -kInf;
      }
      float top = -kInf;
#pragma unroll
      for (int b = 0; b < NK / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
      top = fmaxf(top, other_half(top));
      const bool rise = (top - ref) * c > kSlack;
      if (__builtin_amdgcn_ballot_w64(rise) != 0) {
        const float next = rise ? top : ref, next_c = next * c;
        const bool were_far = any_far;
        // (Rows of infinite scores are zeros or NaN either way.)
        any_far = __builtin_amdgcn_ballot_w64(fabsf(next_c) >= kFar && fabsf(next) < kInf) != 0;
        float down = ref_c - next_c;
        if (__builtin_expect(any_far || were_far, false)) down = (ref - next) * c + (over(next, next_c) - over(ref, ref_c));
        const float keep = rise ? __builtin_amdgcn_exp2f(down) : 1.0f;
        ref = next;
        ref_c = next_c;
        total *= keep;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] *= keep;
      }
      float base = ref == -kInf ? 0.0f : kLift<K> - ref_c;
      if (__builtin_expect(any_far, false)) {
        base = kLift<K> + over(ref, ref_c);
#pragma unroll
        for (int b = 0; b < NK / 32; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[b][i] -= ref == -kInf ? 0.0f : ref;
      }
#pragma unroll
      for (int b = 0; b < NK / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], c, base));
          total += s[b][i];
        }
    };
    auto collect = [&](int shift) {
      const unsigned char* vt = lds + shift + kTileBytes;
#pragma unroll
      for (int step = 0; step < NK / 16; ++step) {
        // The B operand of 16 keys: a lane's eight weights as they are, rounded
        // to the values' type (see the top); the values are read in the same key
        // order.
        uint4 hi, lo;
        unsigned* ph = reinterpret_cast<unsigned*>(&hi);
        unsigned* pl = reinterpret_cast<unsigned*>(&lo);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = s[step >> 1][8 * (step & 1) + 2 * i], b = s[step >> 1][8 * (step & 1) + 2 * i + 1];
          ph[i] = pack2<K>(a, b);
          if constexpr (kSplit) {
            using V = __attribute__((ext_vector_type(2))) _Float16;
            const V h = __builtin_bit_cast(V, ph[i]);
            pl[i] = pack2<K>(a - (float)h[0], b - (float)h[1]);
          }
        }
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const unsigned char* at = vt + value_at + step * 16 * T::kRowBytes + (((4 * i + value_chunk) ^ value_sw) << 4);
          const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr)(at));
          const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr)(at + 8 * T::kRowBytes));
          const s16x8 vf = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
          acc[i] = mfma<K>(vf, __builtin_bit_cast(s16x8, hi), acc[i]);
          if constexpr (kSplit) acc[i] = mfma<K>(vf, __builtin_bit_cast(s16x8, lo), acc[i]);
        }
      }
    };

    if constexpr (WR == 1) {
      // The next keys are on their way from the moment these are read, the next
      // values likewise: one buffer, and no wave waits for another.
      for (int key = wave_begin; key < wave_end; key += TR) {
        const bool more = key + TR < wave_end;
        wait_loads_but<ValueLoader::kLoads>();
        score(0);
        wait_reads();
        if (more) key_loader.load(t.k, t.k_row, key + TR, last, 0, size);
        weigh(key);
        if (more) wait_loads_but<KeyLoader::kLoads>();
        else wait_loads_but<0>();
        collect(0);
        wait_reads();
        if (more) value_loader.load(t.v, t.v_row, key + TR, last, 0, size);
      }
    } else {
      // Two buffers. The barrier: this one's tile is here, and the other one's
      // readers are done.
      int shift = 0;
      for (int key = t.begin; key < end; key += TR) {
        wait_loads();
        __syncthreads();
        const int from = shift;
        shift ^= 2 * kTileBytes;
        if (key + TR < end) {
          key_loader.load(t.k, t.k_row, key + TR, last, shift, size);
          value_loader.load(t.v, t.v_row, key + TR, last, shift, size);
        }
        if (key + wk * NK < wave_end) {
          score(from);
          weigh(key + wk * NK);
          collect(from);
        }
      }
    }
    total += other_half(total);
    const float unit = __builtin_amdgcn_exp2f(-over(ref, ref_c));  // sums to those of the mark
    const float to_mark = fminf(fmaxf(unlift * mark_unit(scale), 0x1p-126f), 0x1p127f);

    // The last key that a tile with masked places can have held.
    const int tiles_end = t.begin + (end - t.begin + TR - 1) / TR * TR, masked_last = tiles_end <= last ? tiles_end - 1 : last;

    if constexpr (WK == 1) {
      // The rows are the wave's own: from registers to memory, a lane four
      // channels of eight, both halves together 16 or 32 bytes.
      const float factor = !sink.out ? unit : total == 0.0f ? 0.0f : 1.0f / total;
      // A row that saw nothing is zeros, also where its values are not finite.
      if (total == 0.0f)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] = f32x16{};
      bool bad = false;
      if (masked || kSplit) {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (D == size || 32 * i + 8 * (j >> 2) + 4 * half < size) most += fabsf(acc[i][j]);
        bad = valid && !(most + other_half(most) < kInf) && (kSplit || total == total);
      }
      if (valid) {
        if (sink.out) {
          Q* dst = sink.out + t.token(my_row) * sink.o_token + t.head(my_row) * sink.o_head + 4 * half;
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int d = 32 * i + 8 * j;
              if (D != size && d + 4 * half >= size) continue;
              const f32x4 o = f32x4{acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]} * factor;
              if constexpr (kSplit) *reinterpret_cast<f32x4*>(dst + d) = o;
              else *reinterpret_cast<uint2*>(dst + d) = uint2{pack2<K>(o[0], o[1]), pack2<K>(o[2], o[3])};
            }
        } else {
          float* dst = sink.sums + (size_t)my_row * D + 4 * half;
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<f32x4*>(dst + 32 * i + 8 * j) =
                  f32x4{acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]} * factor;
          if (half == 0) {
            sink.marks[2 * my_row] = ref * to_mark;
            sink.marks[2 * my_row + 1] = total * factor;
          }
        }
      }
      unsigned rows_bad = (unsigned)__builtin_amdgcn_ballot_w64(bad);
      if (rows_bad != 0) __threadfence_block();  // the stores above come first
      for (; rows_bad != 0; rows_bad &= rows_bad - 1) {
        const int r = __builtin_ctz(rows_bad), row = wr * 32 + r;
        const float whole = __shfl(total * factor, r, 64);
        const SlowRow v = repaired(t, row, whole, masked_last, size, scale);
        const bool all = whole != whole;
        for (int i = 0; i < 2; ++i) {
          const int d = 2 * lane + i;
          if (!v.bad[i]) continue;
          if (sink.out) sink.out[t.token(row) * sink.o_token + t.head(row) * sink.o_head + d] = (Q)v.value[i];
          else sink.sums[(size_t)row * D + d] = v.value[i] * (all ? v.total : whole);
        }
        if (!sink.out && all && lane == 0) {
          sink.marks[2 * row] = v.mark;
          sink.marks[2 * row + 1] = v.total;
        }
      }
      return;
    }
    // The shares of a row agree on one reference; a wave scales its sums to it
    // (to the finished row's scale where the row ends here) and leaves them in
    // LDS, [wave][32 rows][D] with the 16-byte chunks of a row swizzled.
    if (half == 0) {
      marks[(wave * 32 + col) * 2] = ref;
      marks[(wave * 32 + col) * 2 + 1] = total * unit;
    }
    if (lane == 0) marks[64 * (kWaves + WR) + wave] = masked ? 1.0f : 0.0f;
    __syncthreads();
    bool any_masked = false;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) any_masked |= marks[64 * (kWaves + WR) + w] != 0.0f;
    float top = -kInf, sum = 0.0f, factor;
    {
      float m[WK];
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        m[w] = marks[((wr * WK + w) * 32 + col) * 2];
        top = fmaxf(top, m[w]);
      }
      auto weight = [&](float x) { return x == -kInf ? 0.0f : x == top ? 1.0f : __builtin_amdgcn_exp2f((x - top) * c); };
#pragma unroll
      for (int w = 0; w < WK; ++w) sum += weight(m[w]) * marks[((wr * WK + w) * 32 + col) * 2 + 1];
      factor = weight(ref) * unit * (sink.out ? sum == 0.0f ? 0.0f : 1.0f / sum : 1.0f);
    }
    if (half == 0 && wk == 0) {
      marks[64 * kWaves + my_row * 2] = top * to_mark;
      marks[64 * kWaves + my_row * 2 + 1] = sum;
    }
    // A share that saw nothing is zeros, also where its values are not finite.
    if (factor == 0.0f)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] = f32x16{};
    if (valid) {
      float* sums = reinterpret_cast<float*>(lds) + (wave * 32 + col) * D;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int chunk = 8 * i + 2 * j + half;
          *reinterpret_cast<f32x4*>(sums + ((chunk ^ (col & (D / 4 - 1))) << 2)) =
              f32x4{acc[i][4 * j] * factor, acc[i][4 * j + 1] * factor, acc[i][4 * j + 2] * factor, acc[i][4 * j + 3] * factor};
        }
    }
    __syncthreads();
    constexpr int kLanes = D / 4, kAt = 64 / kLanes;  // lanes a row, four channels each; rows a wave has at a time
    const int chunk = lane % kLanes;
    for (int r = wave * kAt + lane / kLanes; r - lane / kLanes < t.rows; r += kWaves * kAt) {
      const float* at = reinterpret_cast<const float*>(lds) + ((r / 32) * WK * 32 + r % 32) * D + ((chunk ^ (r % 32 & (D / 4 - 1))) << 2);
      f32x4 o = *reinterpret_cast<const f32x4*>(at);
#pragma unroll
      for (int w = 1; w < WK; ++w) o += *reinterpret_cast<const f32x4*>(at + w * 32 * D);
      const bool stored = r < t.rows && 4 * chunk < size;
      f32x4 mark = {};
      if (!sink.out) mark = f32x4{marks[64 * kWaves + 2 * r], marks[64 * kWaves + 2 * r + 1]};
      if (any_masked || kSplit) {
        const unsigned long long bad =
            __builtin_amdgcn_ballot_w64(stored && (!(fabsf(o[0]) + fabsf(o[1]) + fabsf(o[2]) + fabsf(o[3]) < kInf) ||
                                                   (kSplit && mark[1] != mark[1])));
        if (bad != 0) {
          for (int g = 0; g < kAt; ++g) {
            if (!(bad >> (g * kLanes) & (kLanes == 64 ? ~0ull : (1ull << kLanes) - 1))) continue;
            const int row = r - lane / kLanes + g;
            const float total = marks[64 * kWaves + 2 * row + 1];
            if (!kSplit && total != total) continue;  // NaN as it should be
            const SlowRow v = repaired(t, row, total, masked_last, size, scale);
            const bool all = total != total;
            // Lane l holds channels 2 l, 2 l + 1.
            for (int i = 0; i < 4; ++i) {
              const float w = __shfl(v.value[i & 1], 2 * chunk + (i >> 1), 64);
              const int stands = __shfl((int)v.bad[i & 1], 2 * chunk + (i >> 1), 64);
              if (lane / kLanes == g && stands) o[i] = sink.out ? w : w * (all ? v.total : total);
            }
            if (lane / kLanes == g && all) mark = f32x4{v.mark, v.total};
          }
        }
      }
      if (!stored) continue;
      if (sink.out) {
        Q* dst = sink.out + t.token(r) * sink.o_token + t.head(r) * sink.o_head + 4 * chunk;
        if constexpr (kSplit) *reinterpret_cast<f32x4*>(dst) = o;
        else *reinterpret_cast<uint2*>(dst) = uint2{pack2<K>(o[0], o[1]), pack2<K>(o[2], o[3])};
      } else {
        *reinterpret_cast<f32x4*>(sink.sums + (size_t)r * D + 4 * chunk) = o;
        if (chunk == 0) {
          sink.marks[2 * r] = mark[0];
          sink.marks[2 * r + 1] = mark[1];
        }
      }
    }
  }
};

// ---- Packed prompts ---------------------------------------------------------------

struct PackedTile {
  int begin, row0, rows, key_begin, keys, first_limit;  // rows 0: none
};

// Sums of the lanes up to this one, over a wave.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // from 1, 2, 4 and 8 lanes before, in rows of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row 0's last lane to row 1, row 2's to row 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row 1's last lane to rows 2 and 3
  return v;
}

__device__ __forceinline__ int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }
// The largest of the lanes' values, none below 0.
__device__ __forceinline__ int wave_max(int v) {
  for (int x = 32; x >= 1; x >>= 1) {
    const int other = __shfl_xor(v, x, 64);
    v = other > v ? other : v;
  }
  return (int)uniform((unsigned)v);
}

// Tile `at`, counted from the last tile of BM rows of the last sequence. A wave
// cuts the sequences into 64 parts, counts their tiles, and goes on in the part
// that has the tile: one round for up to 64 sequences. What is behind the first
// tile is none, so that workgroups without one come last.
// levels: 2 to 64 sequences' tiles are counted level by level from the highest,
// all sequences' third tiles before their second ones: a tile's passes grow with
// its place, and the longest must not start last (24 prompts 27 us, 33 in the
// other order; but six behind caches 56 against 50, whose tiles then share no
// keys with those beside them).
__device__ __forceinline__ PackedTile packed_tile(const fah_packed_attention& a, int at, int group, int BM, bool levels) {
  const int lane = threadIdx.x & 63;
  const int* ko = a.key_offsets ? a.key_offsets : a.query_offsets;
  auto rows_at = [&](int s) { return clamp_int(a.query_offsets[s], 0, a.query_rows); };
  PackedTile p{};
  int lo = 0, hi = a.sequences, target = -1;
  for (bool first = true;; first = false) {
    const int part = (hi - lo + 63) / 64;
    int q0 = 0, q1 = 0, k0 = 0, k1 = 0, tiles = 0;
    auto tiles_of = [&] { return q1 > q0 ? ((q1 - q0) * group + BM - 1) / BM : 0; };
    // Tile n of lane l's sequence.
    auto tile = [&](int l, int n) {
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      p.begin = of(q0);
      const int queries = of(q1) - p.begin;
      p.key_begin = of(k0);
      p.keys = of(k1) > p.key_begin ? of(k1) - p.key_begin : 0;
      p.first_limit = p.keys - queries + 1;
      p.row0 = n * BM;
      p.rows = clamp_int(queries * group - p.row0, 0, BM);
      return p;
    };
    if (part == 1) {
      const int s = lo + lane < hi ? lo + lane : hi - 1;
      q0 = rows_at(s);
      q1 = rows_at(s + 1);
      k0 = clamp_int(ko[s], 0, a.key_rows);
      k1 = clamp_int(ko[s + 1], 0, a.key_rows);
      tiles = lo + lane < hi ? tiles_of() : 0;
    } else {
      const int from = lo + lane * part < hi ? lo + lane * part : hi, to = from + part < hi ? from + part : hi;
      for (int s = from; s < to; ++s) {
        q0 = rows_at(s);
        q1 = rows_at(s + 1);
        tiles += tiles_of();
      }
    }
    if (levels && part == 1) {
      int low = 0, high = wave_max(tiles), count = wave_sum(tiles), above = 0;
      if (at >= count) return p;
      while (high - low > 1) {  // `low`: more than `at` tiles are there or higher; `high`: not
        const int mid = (low + high) / 2, n = wave_sum(tiles > mid ? tiles - mid : 0);
        if (n > at) low = mid;
        else high = mid, above = n;
      }
      const unsigned long long there = __builtin_amdgcn_ballot_w64(tiles > low);
      const int before = __builtin_amdgcn_mbcnt_hi((unsigned)(there >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)there, 0));
      return tile(__builtin_ctzll(__builtin_amdgcn_ballot_w64(tiles > low && before == at - above)), low);
    }
    const int through = wave_scan(tiles);
    if (first) target = __builtin_amdgcn_readlane(through, 63) - 1 - at;
    const unsigned long long past = __builtin_amdgcn_ballot_w64(through > target);
    if (target < 0 || past == 0) return p;
    const int l = __builtin_ctzll(past);
    target -= __builtin_amdgcn_readlane(through - tiles, l);
    if (part == 1) return tile(l, target);
    lo += l * part;
    hi = lo + part < hi ? lo + part : hi;
  }
}

// How packed_kernel's work is cut: tiles of 32 `rows` rows, at most `slots`, whose
// keys are cut into shares of about `share`, at most `splits`.
struct PackedCut {
  int rows, splits, share;
  int64_t slots;
};

// Keys that some row of the tile sees, and the shares they are cut into.
__device__ __forceinline__ int visible_keys(const PackedTile& p, int group) {
  return clamp_int(p.first_limit + (p.row0 + p.rows - 1) / group, 0, p.keys);
}
__device__ __forceinline__ int shares_of(int visible, const PackedCut& cut) {
  return clamp_int((visible + cut.share / 2) / cut.share, 1, cut.splits);
}

// Workgroup: (share of the keys, tile from the last one on, K/V head), the K/V
// head fastest, so that with 8 of them each XCD's L2 serves one head, and the
// shares slowest: most tiles have one, and those that only find that out come
// last (in between they hold up the others' start: 750 rows 22.9 -> 35 us).
template <typename Q, typename K, int D, int WR, int WK, int NK>
__global__ __launch_bounds__(64 * WR * WK, 2) void packed_kernel(fah_packed_attention a, PackedCut cut) {
  using C = Core<Q, K, D, WR, WK, NK>;
  __shared__ __align__(16) unsigned char lds[C::kLds];
  const int group = a.heads / a.kv_heads, head = blockIdx.x % a.kv_heads;
  const int rest = blockIdx.x / a.kv_heads, split = rest / (int)cut.slots, slot = rest % (int)cut.slots;
  const PackedTile p = packed_tile(a, slot, group, C::BM, cut.splits == 1 && a.sequences > 1 && a.sequences <= 64);
  if (p.rows == 0) return;
  const int token0 = p.row0 / group;
  Task<Q, K> t;
  t.q = static_cast<const Q*>(a.query) + (int64_t)(p.begin + token0) * a.query_row + (int64_t)head * group * a.query_head;
  t.q_token = a.query_row;
  t.q_head = a.query_head;
  t.k = static_cast<const K*>(a.key) + p.key_begin * a.key_row + head * a.key_head;
  t.v = static_cast<const K*>(a.value) + p.key_begin * a.value_row + head * a.value_head;
  t.k_row = (unsigned)a.key_row;
  t.v_row = (unsigned)a.value_row;
  t.rows = p.rows;
  t.group = group;
  t.group_inverse = 1.0f / (float)group;
  t.head0 = p.row0 - token0 * group;
  t.first_limit = p.first_limit + token0;
  t.causal = true;
  t.begin = 0;
  t.end = p.keys;
  Sink<Q> sink{};
  const int visible = visible_keys(p, group), shares = shares_of(visible, cut);
  if (split >= shares) return;
  if (shares == 1) {
    sink.out = static_cast<Q*>(a.output) + (int64_t)(p.begin + token0) * a.output_row + (int64_t)head * group * a.output_head;
    sink.o_token = a.output_row;
    sink.o_head = a.output_head;
  } else {
    const int share = ((visible + C::TR - 1) / C::TR + shares - 1) / shares * C::TR;
    t.begin = split * share;
    t.end = t.begin + share < visible ? t.begin + share : visible;
    const size_t item = ((size_t)slot * a.kv_heads + head) * cut.splits + split;
    sink.sums = static_cast<float*>(a.workspace) + item * C::BM * (D + 2);
    sink.marks = sink.sums + C::BM * D;
  }
  C::run(t, sink, a.head_size, a.scale, lds);
}

// Joins partial rows by groups of D / 4 lanes, four channels a lane: at(i) is
// where partial i's row has its sums, marks(i) its marks. The marks are read by
// a lane each and shared, so that every load stands alone.
template <int D>
struct Joined {
  static constexpr int kLanes = D / 4;
  float c;                           // mark_exponent
  float top = -kInf, total = 0.0f;   // the mark of what is joined so far
  f32x4 o = {};
  template <typename At, typename Marks>
  __device__ __forceinline__ void add(int count, At at, Marks marks) {
    const int lane = threadIdx.x % kLanes;
    for (int first = 0; first < count; first += kLanes) {
      const int n = count - first < kLanes ? count - first : kLanes;
      // Eight rows at a time, the first ones requested with the marks.
      f32x4 v[8];
      auto request = [&](int i0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const f32x4*>(at(first + (i0 + i < n ? i0 + i : n - 1)));
      };
      request(0);
      float m = -kInf, w = 0.0f;
      if (lane < n) {
        const float2 mark = *reinterpret_cast<const float2*>(marks(first + lane));
        m = mark.x;
        w = mark.y;
      }
      float next = fmaxf(top, m);
      for (int x = kLanes / 2; x >= 1; x >>= 1) next = fmaxf(next, __shfl_xor(next, x, kLanes));
      // A partial row that saw nothing counts as nothing, unless its total is NaN.
      const float weight = m == -kInf ? 0.0f : m == next ? 1.0f : __builtin_amdgcn_exp2f((m - next) * c);
      const float keep = top == -kInf || top == next ? 1.0f : __builtin_amdgcn_exp2f((top - next) * c);
      float sum = w == w ? weight * w : w;
      for (int x = kLanes / 2; x >= 1; x >>= 1) sum += __shfl_xor(sum, x, kLanes);
      total = total * keep + sum;
      o *= keep;
      for (int i0 = 0; i0 < n; i0 += 8) {
        if (i0 > 0) request(i0);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float wi = __shfl(weight, (i0 + i) % kLanes, kLanes);  // 0 from n on
          o += i0 + i >= n || wi == 0.0f ? f32x4{} : v[i] * wi;
        }
      }
      top = next;
    }
  }
  template <typename Q>
  __device__ void write(Q* dst) const {
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    if constexpr (std::is_same_v<Q, float>) {
      *reinterpret_cast<f32x4*>(dst) = o * inverse;
    } else {
      *reinterpret_cast<uint2*>(dst) = uint2{pack2<Q>(o[0] * inverse, o[1] * inverse), pack2<Q>(o[2] * inverse, o[3] * inverse)};
    }
  }
};

// Workgroup: (tile, K/V head), as many rows of it as it has groups of lanes.
template <typename Q, int D, int BM>
__global__ __launch_bounds__(kThreads) void packed_join_kernel(fah_packed_attention a, PackedCut cut) {
  const int group = a.heads / a.kv_heads, head = blockIdx.x % a.kv_heads, slot = blockIdx.x / a.kv_heads;
  const PackedTile p = packed_tile(a, slot, group, BM, false);
  constexpr int kLanes = D / 4;
  const int chunk = threadIdx.x % kLanes, r = blockIdx.y * (kThreads / kLanes) + threadIdx.x / kLanes;
  if (r >= p.rows) return;
  const int shares = shares_of(visible_keys(p, group), cut);
  if (shares == 1) return;
  const float* sums = static_cast<const float*>(a.workspace) + ((size_t)slot * a.kv_heads + head) * cut.splits * BM * (D + 2);
  Joined<D> j{mark_exponent(a.scale)};
  j.add(shares, [&](int i) { return sums + (size_t)i * BM * (D + 2) + r * D + 4 * chunk; },
        [&](int i) { return sums + (size_t)i * BM * (D + 2) + BM * D + 2 * r; });
  const int row = p.row0 + r;
  if (4 * chunk < a.head_size)
    j.write(static_cast<Q*>(a.output) + (int64_t)(p.begin + row / group) * a.output_row +
            (int64_t)(head * group + row % group) * a.output_head + 4 * chunk);
}

// ---- A shared prefix ----------------------------------------------------------------

// How prefix_kernel's work is cut: prefix tiles of BM rows (a row is a sequence
// and a head of the group) times shares of the prefix, then for every sequence
// tiles of 32 heads times shares of its own rows.
struct PrefixCut {
  int tiles, shares, own_tiles, own_shares;
  int64_t prefix_items, own_items;
  int64_t prefix_rows, rows;  // partial rows of the prefix, and of all
};

// Partial rows: [K/V head][share][sequences * group] of the prefix, then
// [sequence][K/V head][own share][group]. All rows' sums, [D] each and so on 16
// bytes, then all rows' marks and totals. ONCE: own rows pass the caches by.
template <typename Q, typename K, int D, int WR, int WK, int NK, bool ONCE>
__global__ __launch_bounds__(kThreads, 2) void prefix_kernel(fah_prefix_attention a, PrefixCut cut) {
  using Shared = Core<Q, K, D, WR, WK, NK>;
  using Own = Core<Q, K, D, 1, 4, 32, ONCE>;
  static_assert(Shared::kThreads == kThreads && Own::kThreads == kThreads);
  __shared__ __align__(16) unsigned char lds[std::max(Shared::kLds, Own::kLds)];
  const int group = a.heads / a.kv_heads;
  float* partial = static_cast<float*>(a.workspace);
  Task<Q, K> t;
  Sink<Q> sink{};
  t.q_token = a.query_sequence;
  t.q_head = a.query_head;
  t.group = group;
  t.group_inverse = 1.0f / (float)group;
  t.causal = false;
  if (blockIdx.x < cut.prefix_items) {
    using C = Shared;
    const int head = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads;
    const int share_at = rest % cut.shares, tile = rest / cut.shares;
    const int all = a.sequences * group;
    const int row0 = tile * C::BM, token0 = row0 / group;
    t.head0 = row0 - token0 * group;
    t.q = static_cast<const Q*>(a.query) + token0 * a.query_sequence + (int64_t)head * group * a.query_head;
    t.k = static_cast<const K*>(a.prefix_key) + head * a.prefix_key_head;
    t.v = static_cast<const K*>(a.prefix_value) + head * a.prefix_value_head;
    t.k_row = (unsigned)a.prefix_key_row;
    t.v_row = (unsigned)a.prefix_value_row;
    t.rows = clamp_int(all - row0, 0, C::BM);
    const int share = ((a.prefix + C::TR - 1) / C::TR + cut.shares - 1) / cut.shares * C::TR;
    t.begin = share_at * share;
    t.end = t.begin + share < a.prefix ? t.begin + share : a.prefix;
    t.first_limit = t.end;
    const size_t row = ((size_t)head * cut.shares + share_at) * all + row0;
    sink.sums = partial + row * D;
    sink.marks = partial + cut.rows * D + 2 * row;
    C::run(t, sink, a.head_size, a.scale, lds);
  } else {
    using C = Own;
    const int64_t at = blockIdx.x - cut.prefix_items;
    const int head = at % a.kv_heads;
    int64_t rest = at / a.kv_heads;
    const int share_at = rest % cut.own_shares;
    rest /= cut.own_shares;
    const int tile = rest % cut.own_tiles, s = rest / cut.own_tiles;
    const int length = __builtin_amdgcn_readfirstlane(clamp_int(a.lengths[s], 0, a.capacity));
    t.q = static_cast<const Q*>(a.query) + s * a.query_sequence + (int64_t)head * group * a.query_head;
    t.k = static_cast<const K*>(a.key) + s * a.key_sequence + head * a.key_head;
    t.v = static_cast<const K*>(a.value) + s * a.value_sequence + head * a.value_head;
    t.k_row = (unsigned)a.key_row;
    t.v_row = (unsigned)a.value_row;
    t.head0 = tile * C::BM;
    t.rows = clamp_int(group - t.head0, 0, C::BM);
    const int share = ((length + C::TR - 1) / C::TR + cut.own_shares - 1) / cut.own_shares * C::TR;
    t.begin = share_at * share;
    t.end = t.begin + share < length ? t.begin + share : length;
    t.first_limit = t.end;
    if (cut.prefix_items == 0 && cut.own_shares == 1) {
      sink.out = static_cast<Q*>(a.output) + s * a.output_sequence + (int64_t)head * group * a.output_head;
      sink.o_token = a.output_sequence;
      sink.o_head = a.output_head;
    } else {
      const size_t row = cut.prefix_rows + (((size_t)s * a.kv_heads + head) * cut.own_shares + share_at) * group + t.head0;
      sink.sums = partial + row * D;
      sink.marks = partial + cut.rows * D + 2 * row;
    }
    C::run(t, sink, a.head_size, a.scale, lds);
  }
}

template <typename Q, int D>
__global__ __launch_bounds__(kThreads) void prefix_join_kernel(fah_prefix_attention a, PrefixCut cut) {
  constexpr int kLanes = D / 4;
  const int group = a.heads / a.kv_heads, all = a.sequences * group;
  const int64_t at = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  const int chunk = threadIdx.x % kLanes;
  if (at >= (int64_t)a.sequences * a.heads) return;
  const int s = at / a.heads, q_head = at % a.heads, head = q_head / group, g = q_head % group;
  // The prefix's shares, then the own rows'.
  const int shares = cut.prefix_items ? cut.shares : 0;
  const float* sums = static_cast<const float*>(a.workspace) + 4 * chunk;
  const float* marks = static_cast<const float*>(a.workspace) + cut.rows * D;
  const size_t first = (size_t)head * shares * all + s * group + g;
  const size_t own = cut.prefix_rows + ((size_t)s * a.kv_heads + head) * cut.own_shares * group + g;
  auto row = [&](int i) { return i < shares ? first + (size_t)i * all : own + (size_t)(i - shares) * group; };
  Joined<D> j{mark_exponent(a.scale)};
  j.add(shares + cut.own_shares, [&](int i) { return sums + row(i) * D; }, [&](int i) { return marks + 2 * row(i); });
  if (4 * chunk < a.head_size) j.write(static_cast<Q*>(a.output) + s * a.output_sequence + q_head * a.output_head + 4 * chunk);
}

// ---- Launch rules -------------------------------------------------------------------

constexpr int kFill = 512;  // workgroups that fill the chip: two a CU

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows of a tile. 128 where that fills the chip; and with fewer items where the
// sequences are short, because what a workgroup spends around its passes (5 us)
// then counts more than the passes (30 x 100 rows, 16/8 heads: 14.2 us, 20.7 with
// 64 rows; 4 x 819: 26.1 against 31.4; but one of 3200: 69 against 62). 32 where 64-row
// tiles leave CUs without work (750 rows: 15.5 us, 21.5 with 64 rows) or a
// sequence has no more rows. Behind long caches the same by the work that the
// keys' shares make of the items.
//
// Shares of the keys only behind long caches: the joined rows pass through
// memory and a second launch (six resumed prompts 50 us, 60 at best without;
// one token behind 5000 keys 15.5 against 49; a prompt alone of 3200 rows 74
// against 62).
PackedCut packed_cut(const fah_packed_attention& a) {
  const int group = a.heads / a.kv_heads;
  const int64_t rows = (int64_t)a.query_rows * group, keys = a.key_rows / a.sequences, rows_each = rows / a.sequences;
  auto items = [&](int waves) { return std::max<int64_t>(ceil_div(rows, 32 * waves), a.sequences) * a.kv_heads; };
  PackedCut c;
  const bool cached = (a.key_rows - a.query_rows) / a.sequences >= 1024;
  if ((int64_t)a.longest_query * group <= 32) c.rows = 1;
  else if (cached) c.rows = rows_each >= 192 && items(4) * keys / 1280 >= 256 ? 4 : rows_each > 32 ? 2 : 1;
  else c.rows = items(4) >= kFill || (items(4) >= 64 && a.longest_key <= 2 * items(4)) ? 4 : items(2) < 448 ? 1 : 2;
  c.slots = rows / (32 * c.rows) + a.sequences;
  const int64_t n = items(c.rows);
  c.share = (int)std::min<int64_t>(std::max<int64_t>(512, n * keys / kFill), 1280);
  c.splits = cached ? (int)std::max<int64_t>(1, std::min<int64_t>(2048 / n, (a.longest_key + c.share / 2) / c.share)) : 1;
  return c;
}

// Few and long shares of the prefix: each costs its rows' partial sums twice
// through memory. 256 items, or 128 where the sequences' own rows fill the chip
// beside them, of 256 to 4096 keys (61 sequences behind 8191 keys: 26 us with 256
// items, 34 with 128, 29 to 45 with 512; 256 behind 4096, own rows through the
// caches, 128 to 133 us with 64 or 128 items, 142 with 256; 256 behind 8000, fp32: 84 us with shares of
// 4000 keys, 133 with one). 64 rows a tile until 1024 of them (256 sequences of
// 8 heads a group: 65 us, 86 with 128 rows; 1024 sequences 185 against 173); 32
// for no more rows.
PrefixCut prefix_cut(const fah_prefix_attention& a, int* waves_rows) {
  const int group = a.heads / a.kv_heads, longest = std::min(a.longest, a.capacity);
  const int64_t rows = (int64_t)a.sequences * group;
  PrefixCut c{};
  c.own_tiles = (int)ceil_div(group, 32);
  const int64_t own = (int64_t)a.sequences * a.kv_heads * c.own_tiles;
  *waves_rows = rows <= 32 ? 1 : ceil_div(rows, 64) * a.kv_heads < 1024 ? 2 : 4;
  c.own_shares = (int)std::max<int64_t>(1, std::min<int64_t>(256 / own, ceil_div(longest, 256)));
  c.tiles = (int)ceil_div(rows, 32 * *waves_rows);
  const int64_t fill = own * c.own_shares >= 1024 ? 128 : 256;
  c.shares = (int)std::max<int64_t>({1, ceil_div(a.prefix, 4096), std::min<int64_t>(fill / (c.tiles * a.kv_heads), ceil_div(a.prefix, 256))});
  c.prefix_items = a.prefix ? (int64_t)c.tiles * a.kv_heads * c.shares : 0;
  c.own_items = own * c.own_shares;
  c.prefix_rows = a.prefix ? (int64_t)c.shares * a.sequences * a.heads : 0;
  c.rows = c.prefix_rows + (int64_t)c.own_shares * a.sequences * a.heads;
  return c;
}

int width_of(int head_size) { return head_size <= 64 ? 64 : 128; }

template <typename Q, typename K, int D, int WR, int WK, int NK>
hipError_t packed_launch(const fah_packed_attention& a, const PackedCut& c, hipStream_t s) {
  using C = Core<Q, K, D, WR, WK, NK>;
  auto kernel = packed_kernel<Q, K, D, WR, WK, NK>;
  kernel<<<(unsigned)(c.slots * c.splits * a.kv_heads), C::kThreads, 0, s>>>(a, c);
  if (c.splits > 1) {
    const dim3 grid((unsigned)(c.slots * a.kv_heads), (unsigned)ceil_div(C::BM, kThreads / (D / 4)));
    packed_join_kernel<Q, D, C::BM><<<grid, kThreads, 0, s>>>(a, c);
  }
  return hipGetLastError();
}

template <typename Q, typename K, int D>
hipError_t packed_typed(const fah_packed_attention& a, hipStream_t s) {
  const PackedCut c = packed_cut(a);
  if (c.rows == 1) return packed_launch<Q, K, D, 1, 4, 32>(a, c, s);
  if (c.rows == 2) return packed_launch<Q, K, D, 2, 2, 32>(a, c, s);
  return packed_launch<Q, K, D, 4, 1, 64>(a, c, s);
}

template <typename Q, typename K, int D, int WR, int WK, int NK, bool ONCE>
hipError_t prefix_launch(const fah_prefix_attention& a, const PrefixCut& c, hipStream_t s) {
  prefix_kernel<Q, K, D, WR, WK, NK, ONCE><<<(unsigned)(c.prefix_items + c.own_items), kThreads, 0, s>>>(a, c);
  if (c.prefix_items || c.own_shares > 1)
    prefix_join_kernel<Q, D><<<(unsigned)ceil_div((int64_t)a.sequences * a.heads, kThreads / (D / 4)), kThreads, 0, s>>>(a, c);
  return hipGetLastError();
}

template <typename Q, typename K, int D>
hipError_t prefix_typed(const fah_prefix_attention& a, hipStream_t s) {
  int waves_rows;
  const PrefixCut c = prefix_cut(a, &waves_rows);
  // Own rows are read once a call, and past the caches where these (256 MB)
  // could not hold them to the next call (256 sequences of 800 rows on average:
  // 121 us, 133 through the caches; 61 of 350: 27.8 against 26.2).
  const bool once = (int64_t)a.sequences * std::min(a.longest, a.capacity) * a.kv_heads * a.head_size * 4 > 256 << 20;
  if (waves_rows == 1) return prefix_launch<Q, K, D, 1, 4, 32, false>(a, c, s);
  if (waves_rows == 2) return once ? prefix_launch<Q, K, D, 2, 2, 32, true>(a, c, s) : prefix_launch<Q, K, D, 2, 2, 32, false>(a, c, s);
  return once ? prefix_launch<Q, K, D, 4, 1, 64, true>(a, c, s) : prefix_launch<Q, K, D, 4, 1, 64, false>(a, c, s);
}

}  // namespace

bool attention_supported(int heads, int kv_heads, int head_size, int query_type, int cache_type) {
  return heads <= 65536 && head_size % 8 == 0 && head_size <= 128 &&
         ((query_type == FAH_TYPE_F32 && cache_type == FAH_TYPE_F16) ||
          (query_type == FAH_TYPE_F16 && cache_type == FAH_TYPE_F16) ||
          (query_type == FAH_TYPE_BF16 && cache_type == FAH_TYPE_BF16));
}

int64_t packed_attention_workspace(const fah_packed_attention& a) {
  if (a.sequences == 0 || a.query_rows == 0) return 0;
  const PackedCut c = packed_cut(a);
  return c.splits == 1 ? 0 : c.slots * a.kv_heads * c.splits * 32 * c.rows * (width_of(a.head_size) + 2) * 4;
}

int64_t prefix_attention_workspace(const fah_prefix_attention& a) {
  if (a.sequences == 0) return 0;
  int waves_rows;
  const PrefixCut c = prefix_cut(a, &waves_rows);
  if (!c.prefix_items && c.own_shares == 1) return 0;
  return c.rows * (width_of(a.head_size) + 2) * 4;
}

hipError_t launch_packed_attention(const fah_packed_attention& a, hipStream_t s) {
  const bool wide = width_of(a.head_size) == 128;
  if (a.query_type == FAH_TYPE_F32)
    return wide ? packed_typed<float, _Float16, 128>(a, s) : packed_typed<float, _Float16, 64>(a, s);
  if (a.query_type == FAH_TYPE_F16)
    return wide ? packed_typed<_Float16, _Float16, 128>(a, s) : packed_typed<_Float16, _Float16, 64>(a, s);
  return wide ? packed_typed<__bf16, __bf16, 128>(a, s) : packed_typed<__bf16, __bf16, 64>(a, s);
}

hipError_t launch_prefix_attention(const fah_prefix_attention& a, hipStream_t s) {
  const bool wide = width_of(a.head_size) == 128;
  if (a.query_type == FAH_TYPE_F32)
    return wide ? prefix_typed<float, _Float16, 128>(a, s) : prefix_typed<float, _Float16, 64>(a, s);
  if (a.query_type == FAH_TYPE_F16)
    return wide ? prefix_typed<_Float16, _Float16, 128>(a, s) : prefix_typed<_Float16, _Float16, 64>(a, s);
  return wide ? prefix_typed<__bf16, __bf16, 128>(a, s) : prefix_typed<__bf16, __bf16, 64>(a, s);
}

}  // namespace fah

// The 8-bit key/value cache: what its append, read-back and attention kernels share.
//
// A block holds 64 tokens of one head: keys [64][head_dim] and values TRANSPOSED, [head_dim][64], one byte each (code + 128,
// code in [-127, 127]), and one binary32 scale for its keys and one for its values; value = code * scale.  Values lie
// transposed because the product with the probabilities contracts over tokens: a matrix instruction's operand then is 16
// contiguous bytes of a lane, straight from memory, as it is for keys in the product with the queries.
#pragma once
#include "gq_common.h"

namespace gq {

constexpr int kBlock = GQ_KV_BLOCK;

struct KvCache {
  uint8_t *k_codes, *v_codes;  // [n_blocks][heads][64][dim], [n_blocks][heads][dim][64]
  float *k_scale, *v_scale;    // [n_blocks][heads]
  int n_blocks, heads, dim;
};

struct KvBatch {
  const int *offsets, *seq_lens, *table;
  int sequences, width, tokens;
};

// One sequence's new tokens: rows [begin, begin + count) hold positions [first, first + count); `first` is negative where
// the sequence is given more rows than it has tokens (its leading rows then are padding).  The offsets are device data:
// whatever they hold, the rows lie in [0, tokens) and the positions end at the table's capacity.
struct KvSequence {
  int begin, count, first, length;
};

__device__ __forceinline__ KvSequence kv_sequence(const KvBatch &batch, int b) {
  KvSequence s;
  s.begin = min(max(batch.offsets[b], 0), batch.tokens);
  s.count = min(max(batch.offsets[b + 1], s.begin), batch.tokens) - s.begin;
  const int64_t capacity = (int64_t)batch.width * kBlock;
  s.length = (int)min((int64_t)max(batch.seq_lens[b], 0), min(capacity, (int64_t)1 << 30));
  s.first = s.length - s.count;
  return s;
}

// The sequence b and the index in it of unit `unit`, where sequence b has units(b) >= 0 of them: a wave's prefix sum over 64
// sequences at a time.  Every lane gets the answer; false: there are fewer units.  `base` gets the units before b.
template <typename F>
__device__ __forceinline__ bool kv_locate(int64_t unit, int sequences, F units, int &b, int64_t &base) {
  const int lane = threadIdx.x & 63;
  base = 0;
  for (int b0 = 0; b0 < sequences; b0 += 64) {
    const int64_t own = b0 + lane < sequences ? (int64_t)units(b0 + lane) : 0;
    int64_t sum = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t up = __shfl_up((long long)sum, d);
      if (lane >= d) sum += up;
    }
    const int64_t total = __shfl((long long)sum, 63);
    if (unit < base + total) {
      const int at = __builtin_ctzll(__ballot(base + sum > unit));
      b = __builtin_amdgcn_readfirstlane(b0 + at);
      base += __shfl((long long)(sum - own), at);
      return true;
    }
    base += total;
  }
  return false;
}

}  // namespace gq

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

// The sequence b that has unit `unit`, where sequence b has units(sequence) of them, and the units before b: a wave's prefix sum
// over 64 sequences at a time.  Every lane gets the answer (uniform); false: there are fewer units.  (32 bits: the host sees
// to it that there are fewer than 2^31.)
template <typename F>
__device__ __forceinline__ bool kv_locate(const KvBatch &batch, uint32_t unit, F units, int &b, KvSequence &s, uint32_t &base) {
  const int lane = threadIdx.x & 63;
  base = 0;
  for (int b0 = 0; b0 < batch.sequences; b0 += 64) {
    KvSequence own_s = {};
    uint32_t own = 0;
    if (b0 + lane < batch.sequences) {
      own_s = kv_sequence(batch, b0 + lane);
      own = units(own_s);
    }
    uint32_t sum = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    const uint32_t total = __builtin_amdgcn_readlane(sum, 63);
    if (unit < base + total) {
      const int at = __builtin_ctzll(__ballot(base + sum > unit));
      b = b0 + at;
      s.begin = __builtin_amdgcn_readlane(own_s.begin, at), s.count = __builtin_amdgcn_readlane(own_s.count, at);
      s.first = __builtin_amdgcn_readlane(own_s.first, at), s.length = __builtin_amdgcn_readlane(own_s.length, at);
      base += __builtin_amdgcn_readlane(sum - own, at);
      return true;
    }
    base += total;
  }
  return false;
}

// Units of all sequences.
template <typename F>
__device__ __forceinline__ uint32_t kv_units(const KvBatch &batch, F units) {
  uint32_t sum = 0;
  for (int b = threadIdx.x & 63; b < batch.sequences; b += 64) sum += units(kv_sequence(batch, b));
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  return __builtin_amdgcn_readfirstlane(sum);
}

}  // namespace gq

// Attention over the 8-bit key/value cache (layout: gq_kv.h), causal, grouped heads, ragged batches.
//
//   o[row] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t - max),  t <= position of the row
//
// kv_split_kernel: any number of new tokens; the kernel for decoding.  Bound by the cache's bytes: 2 dim bytes a token and
// head.  The rows of one kv head (its group of query heads x new tokens) are taken 16 at a time, the N side of
// 16x16x32 products; keys and values are the M side, so that both come from memory as they lie, a lane's 16 bytes at a time,
// without LDS:  S^T = K Q^T, O^T = V^T P^T.  The contraction order is free as long as both operands agree on it:
//   - product over dims: lane group g = lane / 16 holds dims 64 c + 16 g + 8 u ... + 7 at step (c, u);
//   - row 4 g' + i of key tile t is token 16 g' + 4 t + i, so that the scores a lane gets (row 4 g + i of each tile, in the
//     accumulator's layout) are those of its tokens 16 g ... 16 g + 15: exactly the order in which its 16 bytes of V^T hold
//     tokens.  P^T goes from the accumulators of one product into the operand of the next without leaving the lane.
// Codes become binary16 exactly: byte b under exponent 0x64 is 1024 + b, and 1152 is subtracted (2 instructions a pair).
// A block's scales are constant over a tile: one factor on the scores, one on the tile's product.
//
// Work is cut into equal ranges of blocks over all sequences, heads and row tiles, whatever their lengths: workgroup w of W
// takes units [U w / W, U (w + 1) / W), the four waves of it every fourth block.  A range may end inside a (sequence, head):
// what it has then goes to the workspace and kv_join_kernel adds the parts, in the order of the blocks.  Nothing depends on
// lengths that only the device knows, and results do not depend on timing.
#include "gq_kv.h"

namespace gq {
namespace {

constexpr int kThreads = 256, kWaves = 4, kRows = 16;
constexpr int kMostGroups = 512;

struct AttentionArgs {
  KvCache cache;
  KvBatch batch;
  const half_t *q;
  half_t *out;
  int64_t q_token, q_head, o_token, o_head;
  int group;         // query heads of one kv head
  float scale_log2;  // softmax scale x log2(e)
  float *parts;      // [2 groups of the grid][kRows][dim], then maxima and sums [2 groups][2][kRows]
  int groups;
};

struct Shape {  // one sequence's share of the work
  int tiles;   // of 16 rows
  int blocks;  // that its last token sees, one at least (a row that sees nothing still gets its zeros)
};

__device__ __forceinline__ Shape shape_of(const AttentionArgs &a, const KvSequence &s) {
  Shape r;
  r.tiles = (int)(((int64_t)s.count * a.group + kRows - 1) / kRows);
  r.blocks = max(1, (s.length + kBlock - 1) / kBlock);
  return r;
}

__device__ __forceinline__ int64_t units_of(const AttentionArgs &a, int b) {
  const Shape s = shape_of(a, kv_sequence(a.batch, b));
  return (int64_t)s.tiles * s.blocks * a.cache.heads;
}

__device__ __forceinline__ int64_t all_units(const AttentionArgs &a) {
  int64_t sum = 0;
  for (int b = threadIdx.x & 63; b < a.batch.sequences; b += 64) sum += units_of(a, b);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor((long long)sum, d);
  return sum;
}

// Workgroups that take part: enough that each has four blocks, one for each wave.
__device__ __forceinline__ int64_t active_groups(int64_t units, int groups) {
  const int64_t want = (units + kWaves - 1) / kWaves;
  return want < groups ? max(want, (int64_t)1) : groups;
}

__device__ __forceinline__ half2_t two_codes(uint32_t bytes, uint32_t selector) {
  const uint32_t w = __builtin_amdgcn_perm(0x64646464u, bytes, selector);
  const half2_t bias = {(half_t)1152.f, (half_t)1152.f};
  return __builtin_bit_cast(half2_t, w) - bias;
}

// 8 codes in binary16, exact
__device__ __forceinline__ half8_t eight_codes(uint32_t lo, uint32_t hi) {
  const half2_t a = two_codes(lo, 0x04010400u), b = two_codes(lo, 0x04030402u);
  const half2_t c = two_codes(hi, 0x04010400u), d = two_codes(hi, 0x04030402u);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// DP: head_dim rounded up to 64, 128 or 256; dims behind head_dim are read as zeros of q and never stored.
template <int DP>
__global__ __launch_bounds__(kThreads, DP > 128 ? 1 : 2) void kv_split_kernel(AttentionArgs a) {
  constexpr int kChunks = DP / 64, kTiles = DP / 16;
  extern __shared__ float shared[];  // [waves][kRows][DP + 4] and [waves][2][kRows]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
  const int dim = a.cache.dim, heads = a.cache.heads;
  const int64_t units = all_units(a), groups = active_groups(units, a.groups);
  if (units == 0 || (int64_t)blockIdx.x >= groups) return;
  int64_t unit = units * blockIdx.x / groups;
  const int64_t end = units * (blockIdx.x + 1) / groups;
  const int64_t start = unit;

  while (unit < end) {
    int b;
    int64_t base;
    if (!kv_locate(unit, a.batch.sequences, [&](int i) { return units_of(a, i); }, b, base)) return;
    const KvSequence s = kv_sequence(a.batch, b);
    const Shape shape = shape_of(a, s);
    const int64_t within = unit - base;
    const int block0 = (int)(within % shape.blocks);
    const int tile = (int)(within / shape.blocks % shape.tiles), h = (int)(within / shape.blocks / shape.tiles);
    const int block1 = (int)min((int64_t)shape.blocks, block0 + end - unit);
    const int *table = a.batch.table + (int64_t)b * a.batch.width;

    // this lane's row of the tile: new token `token`, query head h * group + member
    const int row = tile * kRows + m, rows = s.count * a.group;
    const bool has_row = row < rows;
    const int token = has_row ? row / a.group : 0, member = has_row ? row % a.group : 0;
    const int position = has_row ? s.first + token : -1;
    const int least = s.first + tile * kRows / a.group;  // the tile's first position
    half8_t qf[kChunks][2];
    const half_t *q = a.q + (s.begin + token) * a.q_token + (int64_t)(h * a.group + member) * a.q_head;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int d = c * 64 + g * 16 + u * 8;
        qf[c][u] = half8_t{};
        if (has_row && d < dim) qf[c][u] = *(const half8_t *)(q + d);
      }

    float4_t o[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[i] = float4_t{};
    float most = -__builtin_inff(), sum = 0.f;

    for (int block = block0 + wave; block < block1; block += kWaves) {
      const int at = block * kBlock;
      if (at >= s.length) continue;  // (the one block of an empty sequence: the table need not have a column for it)
      const int id = __builtin_amdgcn_readfirstlane(table[block]);
      if (id < 0 || id >= a.cache.n_blocks) continue;
      const int64_t place = (int64_t)id * heads + h;
      const uint8_t *kc = a.cache.k_codes + place * kBlock * dim, *vc = a.cache.v_codes + place * kBlock * dim;
      const float ks = a.cache.k_scale[place] * a.scale_log2, vs = a.cache.v_scale[place];

      uint4_t kf[4][kChunks];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int key = 16 * (m >> 2) + 4 * t + (m & 3), d = min(c * 64 + g * 16, dim - 16);
          kf[t][c] = *(const uint4_t *)(kc + key * dim + d);
        }
      float4_t score[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        score[t] = float4_t{};
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          score[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight_codes(kf[t][c][0], kf[t][c][1]), qf[c][0], score[t], 0, 0, 0);
          score[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight_codes(kf[t][c][2], kf[t][c][3]), qf[c][1], score[t], 0, 0, 0);
        }
      }
      const bool masked = at + kBlock - 1 > least;
      float top = -__builtin_inff();
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          score[t][i] *= ks;
          if (masked && at + 16 * g + 4 * t + i > position) score[t][i] = -__builtin_inff();
          top = fmaxf(top, score[t][i]);
        }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float next = fmaxf(most, top);
      const float zero_point = next == -__builtin_inff() ? 0.f : next;  // (a row that has seen nothing: every p is 0)
      const float keep = __builtin_amdgcn_exp2f(most - zero_point);
      most = next;
      half8_t pf[2];
      float part = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = __builtin_amdgcn_exp2f(score[t][i] - zero_point);
          part += p;
          // (binary16 for the matrix product: at most 2^-11 of each p, the sum keeps all of it)
          pf[t >> 1][4 * (t & 1) + i] = (half_t)p;
        }
      sum = sum * keep + part;
      // a row that sees none of this block takes nothing from it, also where its scale is not finite
      const float factor = at > position ? 0.f : vs;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        const int d = min(i * 16 + m, dim - 1);
        const uint4_t w = *(const uint4_t *)(vc + d * kBlock + 16 * g);
        float4_t r = {};
        r = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight_codes(w[0], w[1]), pf[0], r, 0, 0, 0);
        r = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight_codes(w[2], w[3]), pf[1], r, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = __builtin_fmaf(r[j], factor, o[i][j] * keep);
      }
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);

    // the four waves' parts, joined in LDS
    float *mine = shared + wave * kRows * (DP + 4), *stats = shared + kWaves * kRows * (DP + 4);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) *(float4_t *)(mine + m * (DP + 4) + i * 16 + 4 * g) = o[i];
    if (g == 0) stats[wave * 2 * kRows + m] = most, stats[wave * 2 * kRows + kRows + m] = sum;
    __syncthreads();
    const bool whole = block0 == 0 && block1 == shape.blocks;
    const int slot = 2 * blockIdx.x + (unit == start ? 0 : 1);
    const int here = min(kRows, rows - tile * kRows);
    for (int n = threadIdx.x; n < here * dim; n += kThreads) {
      const int r = n / dim, d = n % dim;
      float all = -__builtin_inff();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) all = fmaxf(all, stats[w * 2 * kRows + r]);
      const float zero_point = all == -__builtin_inff() ? 0.f : all;
      float value = 0.f, weight = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(stats[w * 2 * kRows + r] - zero_point);
        value += f * shared[(w * kRows + r) * (DP + 4) + d];
        weight += f * stats[w * 2 * kRows + kRows + r];
      }
      if (whole) {
        const int at = tile * kRows + r;
        half_t *to = a.out + (s.begin + at / a.group) * a.o_token + (int64_t)(h * a.group + at % a.group) * a.o_head;
        to[d] = (half_t)(weight == 0.f ? 0.f : value / weight);
      } else {
        a.parts[((int64_t)slot * kRows + r) * dim + d] = value;
        if (d == 0) {
          float *st = a.parts + (int64_t)2 * a.groups * kRows * dim + (int64_t)slot * 2 * kRows;
          st[r] = all, st[kRows + r] = weight;
        }
      }
    }
    __syncthreads();
    unit += block1 - block0;
  }
}

// Adds the parts of every (sequence, head, row tile) that more than one workgroup worked on.  Workgroup w of this grid has
// boundary w + 1 of the cut; the first boundary inside a tile's units takes the tile.
__global__ __launch_bounds__(kThreads) void kv_join_kernel(AttentionArgs a) {
  const int dim = a.cache.dim;
  const int64_t units = all_units(a), groups = active_groups(units, a.groups);
  const int64_t w = blockIdx.x + 1;
  if (units == 0 || w >= groups) return;
  const int64_t unit = units * w / groups;
  int b;
  int64_t base;
  if (!kv_locate(unit, a.batch.sequences, [&](int i) { return units_of(a, i); }, b, base)) return;
  const KvSequence s = kv_sequence(a.batch, b);
  const Shape shape = shape_of(a, s);
  const int64_t which = (unit - base) / shape.blocks;
  const int64_t from = base + which * shape.blocks, to = from + shape.blocks;
  if (unit == from || units * (w - 1) / groups > from) return;
  const int tile = (int)(which % shape.tiles), h = (int)(which / shape.tiles);
  const int64_t last = (to * groups - 1) / units;  // the workgroup that has unit to - 1
  const int here = min(kRows, s.count * a.group - tile * kRows);
  const float *stats = a.parts + (int64_t)2 * a.groups * kRows * dim;
  for (int n = threadIdx.x; n < here * dim; n += kThreads) {
    const int r = n / dim, d = n % dim;
    float most = -__builtin_inff(), value = 0.f, weight = 0.f;
    for (int64_t i = w - 1; i <= last; ++i) {
      const int64_t slot = 2 * i + (units * i / groups < from ? 1 : 0);
      const float m = stats[slot * 2 * kRows + r], l = stats[slot * 2 * kRows + kRows + r];
      const float v = a.parts[(slot * kRows + r) * dim + d];
      const float next = fmaxf(most, m), zero_point = next == -__builtin_inff() ? 0.f : next;
      const float keep = __builtin_amdgcn_exp2f(most - zero_point), f = __builtin_amdgcn_exp2f(m - zero_point);
      value = value * keep + v * f, weight = weight * keep + l * f, most = next;
    }
    const int at = tile * kRows + r;
    half_t *o = a.out + (s.begin + at / a.group) * a.o_token + (int64_t)(h * a.group + at % a.group) * a.o_head;
    o[d] = (half_t)(weight == 0.f ? 0.f : value / weight);
  }
}

template <int DP>
int launch_split(const AttentionArgs &a, hipStream_t stream) {
  const size_t lds = (size_t)kWaves * kRows * (DP + 4 + 2) * sizeof(float);
  if (lds > 64 << 10) {
    const hipError_t e = hipFuncSetAttribute((const void *)kv_split_kernel<DP>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return fail((int)e, "kv_split_kernel: %s", hipGetErrorString(e));
  }
  kv_split_kernel<DP><<<a.groups, kThreads, lds, stream>>>(a);
  return check_launch("kv_split_kernel");
}

}  // namespace

int64_t kv_attention_workspace_bytes(int64_t dim) {
  return (int64_t)2 * kMostGroups * kRows * (dim + 2) * sizeof(float);
}

int launch_kv_attention(const KvCache &cache, const KvBatch &batch, const uint16_t *q, int64_t q_token, int64_t q_head,
                        uint16_t *out, int64_t o_token, int64_t o_head, int64_t q_heads, float scale, void *workspace,
                        hipStream_t stream) {
  AttentionArgs a;
  a.cache = cache, a.batch = batch;
  a.q = (const half_t *)q, a.q_token = q_token, a.q_head = q_head;
  a.out = (half_t *)out, a.o_token = o_token, a.o_head = o_head;
  a.group = (int)(q_heads / cache.heads);
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.parts = (float *)workspace;
  a.groups = kMostGroups;
  int rc = cache.dim <= 64 ? launch_split<64>(a, stream) : cache.dim <= 128 ? launch_split<128>(a, stream) : launch_split<256>(a, stream);
  if (rc != GQ_OK) return rc;
  kv_join_kernel<<<a.groups - 1, kThreads, 0, stream>>>(a);
  return check_launch("kv_join_kernel");
}

}  // namespace gq

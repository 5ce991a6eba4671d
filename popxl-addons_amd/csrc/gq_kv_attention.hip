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
//
// Measured: 64 sequences of up to 32768, 8 kv heads of 128, 4 query heads each: 376 us, 5.8 TB/s of codes; one sequence of 777, 16
// heads of 256: 9 us, four dependent loads and the sums, and 4.6 us for kv_join_kernel.
#include "gq_kv.h"

namespace gq {
namespace {

constexpr int kThreads = 256, kWaves = 4, kRows = 16;
constexpr int kMostGroups = 512, kTileRows = 128, kTileLeast = 64;

struct AttentionArgs {
  KvCache cache;
  KvBatch batch;
  const half_t *q;
  half_t *out;
  int64_t q_token, q_head, o_token, o_head;
  int group;         // query heads of one kv head
  float scale_log2;  // softmax scale x log2(e)
  // kv_split_kernel: [2 groups][kRows][dim], then maxima and sums [2 groups][2][kRows] (groups: the grid's);
  // kv_tile_kernel, where `splits` of them share a tile: [groups][splits][kTileRows][dim], then [groups][splits][2][kTileRows]
  float *parts;
  int groups, splits;
};

struct Shape {  // one sequence's share of the work
  int tiles;   // of 16 rows
  int blocks;  // that its last token sees, one at least (a row that sees nothing still gets its zeros)
};

__device__ __forceinline__ Shape shape_of(const AttentionArgs &a, const KvSequence &s) {
  Shape r;
  r.tiles = (s.count * a.group + kRows - 1) / kRows;
  r.blocks = max(1, (s.length + kBlock - 1) / kBlock);
  return r;
}

__device__ __forceinline__ uint32_t units_of(const AttentionArgs &a, const KvSequence &s) {
  const Shape shape = shape_of(a, s);
  return (uint32_t)shape.tiles * shape.blocks * a.cache.heads;
}

// The cut of the units: `groups` workgroups take part, the first `more` of them with one unit more than the others.  Up to 256
// units every one has a workgroup, and so a compute unit, of its own: what a compute unit gets from memory is what a short
// history waits for (13 blocks x 16 heads of 256: 9 us, with a block for each wave of 52 workgroups 15 us).  More units make
// workgroups of four, one for each wave.
struct Cut {
  uint32_t units, groups, each, more;
  __device__ Cut(uint32_t units_, uint32_t most) : units(units_) {
    const uint32_t want = max(min(units, 256u), (units + kWaves - 1) / kWaves);
    groups = min(max(want, 1u), most);
    each = units / groups, more = units - each * groups;
  }
  __device__ uint32_t start(uint32_t group) const { return group * each + min(group, more); }
  __device__ uint32_t owner(uint32_t unit) const {
    const uint32_t large = more * (each + 1);
    return unit < large ? unit / (each + 1) : more + (unit - large) / each;
  }
};

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

// 4 dims of a row of the result; a row that has seen nothing is zeros
__device__ __forceinline__ void store_row(const AttentionArgs &a, const KvSequence &s, int h, int row, int d, float4_t value, float weight) {
  const int token = row / a.group, member = row - token * a.group;
  half_t *to = a.out + (s.begin + token) * a.o_token + (int64_t)(h * a.group + member) * a.o_head + d;
  const float factor = weight == 0.f ? 0.f : 1.f / weight;
#pragma unroll
  for (int j = 0; j < 4; ++j) to[j] = (half_t)(value[j] * factor);
}

// DP: head_dim rounded up to 64, 128 or 256; dims behind head_dim are read as zeros of q and never stored.  A block's values are
// asked for before its scores are formed, the next block's keys before the probabilities: loads arrive in order, so that
// each wait leaves the later ones on their way.
template <int DP>
__global__ __launch_bounds__(kThreads, DP > 128 ? 1 : 2) void kv_split_kernel(AttentionArgs a) {
  constexpr int kChunks = DP / 64, kTiles = DP / 16;
  extern __shared__ float shared[];  // [waves][kRows][DP + 4] and [waves][2][kRows]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
  const int dim = a.cache.dim, heads = a.cache.heads;
  const auto units_of_sequence = [&](const KvSequence &s) { return units_of(a, s); };
  const Cut cut(kv_units(a.batch, units_of_sequence), a.groups);
  if (blockIdx.x >= cut.groups) return;
  const uint32_t start = cut.start(blockIdx.x), end = cut.start(blockIdx.x + 1);
  uint32_t unit = start;

  while (unit < end) {
    int b;
    uint32_t base;
    KvSequence s;
    if (!kv_locate(a.batch, unit, units_of_sequence, b, s, base)) return;
    const Shape shape = shape_of(a, s);
    const uint32_t which = (unit - base) / shape.blocks;
    const int block0 = unit - base - which * shape.blocks, block1 = min((uint32_t)shape.blocks, block0 + end - unit);
    const int h = which / shape.tiles, tile = which - h * shape.tiles;
    const int *table = a.batch.table + (int64_t)b * a.batch.width;
    const int stop = min(block1, (s.length + kBlock - 1) / kBlock);  // (an empty sequence has no block to read)

    // ids of blocks that are not there are -1
    const auto id_of = [&](int block) {
      const int id = block < stop ? __builtin_amdgcn_readfirstlane(table[block]) : -1;
      return id < a.cache.n_blocks ? id : -1;
    };
    uint4_t kf[4][kChunks];
    float key_scale = 0.f, value_scale = 0.f;
    const auto load_keys = [&](int id) {
      if (id < 0) return;
      const int64_t place = (int64_t)id * heads + h;
      const uint8_t *kc = a.cache.k_codes + place * kBlock * dim;
      key_scale = a.cache.k_scale[place] * a.scale_log2, value_scale = a.cache.v_scale[place];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int key = 16 * (m >> 2) + 4 * t + (m & 3), d = min(c * 64 + g * 16, dim - 16);
          kf[t][c] = *(const uint4_t *)(kc + key * dim + d);
        }
    };
    int id = id_of(block0 + wave), next_id = id_of(block0 + wave + kWaves);
    load_keys(id);

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

    for (int block = block0 + wave; block < stop; block += kWaves) {
      const int at = block * kBlock, after = id_of(block + 2 * kWaves);
      const float ks = key_scale, vs = value_scale;
      if (id >= 0) {
        const uint8_t *vc = a.cache.v_codes + ((int64_t)id * heads + h) * kBlock * dim;
        uint4_t vf[kTiles];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) vf[i] = *(const uint4_t *)(vc + min(i * 16 + m, dim - 1) * kBlock + 16 * g);
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
        load_keys(next_id);
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
          float4_t r = {};
          r = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight_codes(vf[i][0], vf[i][1]), pf[0], r, 0, 0, 0);
          r = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight_codes(vf[i][2], vf[i][3]), pf[1], r, 0, 0, 0);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][j] = __builtin_fmaf(r[j], factor, o[i][j] * keep);
        }
      } else {
        load_keys(next_id);
      }
      id = next_id, next_id = after;
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
    for (int r = wave; r < here; r += kWaves) {  // a wave has a row, a lane 4 dims
      float all = -__builtin_inff(), weight = 0.f, f[kWaves];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) all = fmaxf(all, stats[w * 2 * kRows + r]);
      const float zero_point = all == -__builtin_inff() ? 0.f : all;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        f[w] = __builtin_amdgcn_exp2f(stats[w * 2 * kRows + r] - zero_point);
        weight += f[w] * stats[w * 2 * kRows + kRows + r];
      }
      const int d = lane * 4;
      if (d >= dim) continue;
      float4_t value = {};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) value += *(const float4_t *)(shared + (w * kRows + r) * (DP + 4) + d) * f[w];
      if (whole) {
        store_row(a, s, h, tile * kRows + r, d, value, weight);
      } else {
        *(float4_t *)(a.parts + ((int64_t)slot * kRows + r) * dim + d) = value;
        if (lane == 0) {
          float *st = a.parts + (int64_t)2 * a.groups * kRows * dim + (int64_t)slot * 2 * kRows;
          st[r] = all, st[kRows + r] = weight;
        }
      }
    }
    __syncthreads();
    unit += block1 - block0;
  }
}

// ------------------------------------------------------------------------------------------------- many rows at a time
//
// kv_tile_kernel: prompts.  Bound by the matrix units: 4 dim operations for each row and key.  The products are turned as in
// kv_split_kernel (S^T = K Q^T, O^T = V^T P^T, now 32x32x16), so that probabilities stay in their lanes: row 8 a + 4 g + b of a
// key tile is token 16 g + 4 a + b, g = lane / 32, which makes a lane's 16 scores those of 16 consecutive tokens, in
// the order of its 16 bytes of V^T.  Four waves with 32 rows each share a block's keys and values through LDS, where
// they lie in binary16 in the order of the operands (1 KiB for a wave's load): every code is converted once a workgroup, not
// once a wave.  The next block's bytes are loaded into registers before this block's products and converted behind them.
//
// Rescaling the accumulators for every block would cost as many vector instructions as the softmax.  The maximum in
// use is only raised when scores pass it by more than 8 (probabilities up to 2^8 then), and the value scale enters the exponent
// as its ratio to a reference, which only moves when the ratio leaves [1/16, 16]; the sum takes the ratio back out.
//
// Measured: 2 sequences of up to 2048 new tokens over 8000, 16 heads of 256: 450 to 500 us, 600 to 690 TFLOP/s (a large matrix
// product: 1150).  Of a compute unit's time the matrix units are busy for 30 %, vector instructions for 33 %, and a third is waited:
// with 454 registers a wave there is one to a SIMD, whose softmax nothing covers (products of the next scores moved among
// it, by order or by scheduling barriers, took 520 to 590 us: the compiler then keeps fewer loads from LDS under way).
// At 128 dims two waves share a SIMD: 4096 tokens, 32 heads: 195 us, 700 TFLOP/s.
//
// A grid too small for the device is divided over the keys as well: `splits` workgroups share a tile and kv_tile_join_kernel adds
// their parts, in their order.

constexpr int kTileThreads = 256;

__device__ __forceinline__ void store_codes(half_t *to, uint32_t lo, uint32_t hi) { *(half8_t *)to = eight_codes(lo, hi); }

template <int DP>
__global__ __launch_bounds__(kTileThreads, DP > 128 ? 1 : 2) void kv_tile_kernel(AttentionArgs a) {
  constexpr int kSteps = DP / 16;                    // of the product over dims
  constexpr int kDimTiles = DP / 32;                 // of 32 dims of the result
  constexpr int kRowsOfWave = 32, kRowsOfGroup = kTileRows;
  constexpr int kHalves = kBlock * DP;               // binary16 of a block's keys (or values)
  constexpr int kPieces = kBlock * DP / 16 / kTileThreads;  // 16-byte pieces of the keys (values) a thread stages
  extern __shared__ half_t tile_shared[];  // [2][keys, values]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 31, g = lane >> 5;
  const int dim = a.cache.dim, heads = a.cache.heads;

  int b;
  uint32_t base;
  KvSequence s;
  const auto units = [&](const KvSequence &s) { return (uint32_t)(s.count * a.group + kRowsOfGroup - 1) / kRowsOfGroup * heads; };
  if (!kv_locate(a.batch, blockIdx.x, units, b, s, base)) return;
  const int rows = s.count * a.group, tiles = (rows + kRowsOfGroup - 1) / kRowsOfGroup;
  const int within = (int)(blockIdx.x - base), h = within % heads;
  const int row0 = (tiles - 1 - within / heads) * kRowsOfGroup;  // the longest tiles first
  const int *table = a.batch.table + (int64_t)b * a.batch.width;

  // rows of this lane and of this wave
  half8_t qf[kSteps];
  int position;
  const float sign = a.scale_log2 < 0.f ? -1.f : 1.f;
  {
    const int row = row0 + wave * kRowsOfWave + m;
    const bool has_row = row < rows;
    const int token = has_row ? row / a.group : 0, member = has_row ? row % a.group : 0;
    position = has_row ? s.first + token : -1;
    const half_t *q = a.q + (s.begin + token) * a.q_token + (int64_t)(h * a.group + member) * a.q_head;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      qf[k] = half8_t{};
      if (has_row && k * 16 < dim) qf[k] = *(const half8_t *)(q + k * 16 + g * 8) * (half_t)sign;
    }
  }
  const int wave_row = row0 + wave * kRowsOfWave;
  const int wave_first = s.first + wave_row / a.group;                                          // its first row's position
  const int wave_last = wave_row < rows ? s.first + (min(wave_row + kRowsOfWave, rows) - 1) / a.group : -1;
  const int group_last = s.first + (min(row0 + kRowsOfGroup, rows) - 1) / a.group;
  const int all_blocks = group_last < 0 ? 0 : group_last / kBlock + 1, share_of = (all_blocks + a.splits - 1) / a.splits;
  const int first_block = min(all_blocks, (int)blockIdx.y * share_of), blocks = a.cache.n_blocks > 0 ? min(all_blocks, first_block + share_of) : 0;

  // staging: thread n has keys' piece (key, 16 dims c) and values' piece (dim d, 16 tokens)
  static_assert(2 * kPieces == kDimTiles, "a piece for every dim tile of the result");
  uint4_t raw_k[kPieces], raw_v[kPieces];
  float ks = 0.f, vs = 0.f;  // of the block that is staged
  bool there = false;
  int ahead = 0;  // the next block's id: it is asked for a block before its bytes are
  const auto id_of = [&](int block) { return table[min(block, blocks - 1)]; };
  // Loads are made without conditions, as in the adapters' products: of block 0 where an id is none, of other dims where a dim
  // is behind the last (its queries are zeros, its results are not stored).
  const auto load = [&](int block) {
    const int id = __builtin_amdgcn_readfirstlane(ahead);
    there = id >= 0 && id < a.cache.n_blocks;
    ahead = id_of(block + 1);
    const int64_t place = (int64_t)(there ? id : 0) * heads + h;
    const uint8_t *kc = a.cache.k_codes + place * kBlock * dim, *vc = a.cache.v_codes + place * kBlock * dim;
    ks = a.cache.k_scale[place], vs = a.cache.v_scale[place];
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      const int i = tid + n * kTileThreads, key = i / (DP / 16), c = i % (DP / 16), d = i / 4;
      raw_k[n] = *(const uint4_t *)(kc + key * dim + (c * 16 < dim ? c * 16 : 0));
      raw_v[n] = *(const uint4_t *)(vc + (d < dim ? d : 0) * kBlock + i % 4 * 16);
    }
  };
  // Keys: operand (tile T, step c) is 1 KiB, lane (g, row) has dims 16 c + 8 g ...; a row's two halves are stored by the thread
  // that has its 16 dims.  The place within 512 bytes is turned by c, so that threads of one key and different c use
  // different banks.  Values: operand (dim tile, T, u), lane (g, dim) has tokens 32 T + 16 g + 8 u ..., turned by the piece for the
  // same reason (four threads of a dim would write to one bank).
  const auto stage_piece = [&](int buffer, int n, bool values) {
    half_t *keys = tile_shared + buffer * 2 * kHalves, *vals = keys + kHalves;
    const int i = tid + n * kTileThreads;
    if (!values) {
      const int key = i / (DP / 16), c = i % (DP / 16), in_tile = key & 31, row = (in_tile >> 2 & 3) * 8 + (in_tile >> 4) * 4 + (in_tile & 3);
      half_t *to = keys + (((key >> 5) * kSteps + c) * 64 + (row ^ (c & 15))) * 8;
      store_codes(to, raw_k[n][0], raw_k[n][1]);
      store_codes(to + 32 * 8, raw_k[n][2], raw_k[n][3]);
    } else {
      const int d = i / 4, piece = i % 4;
      half_t *to = vals + (((d >> 5) * 4 + (piece >> 1) * 2) * 64 + (piece & 1) * 32 + ((d & 31) ^ (2 * piece))) * 8;
      store_codes(to, raw_v[n][0], raw_v[n][1]);
      store_codes(to + 64 * 8, raw_v[n][2], raw_v[n][3]);
    }
  };
  const auto stage = [&](int buffer) {
#pragma unroll
    for (int n = 0; n < 2 * kPieces; ++n) stage_piece(buffer, n / 2, n & 1);
  };

  float16_t o[kDimTiles];
  float most = -__builtin_inff(), sum = 0.f;
  float reference = 1.f;
#pragma unroll
  for (int i = 0; i < kDimTiles; ++i) o[i] = float16_t{};
  if (first_block < blocks) {
    ahead = id_of(first_block);
    load(first_block);
    stage(first_block & 1);
  }
  // Rescaling takes the accumulators out of the matrix units' registers and back, so it stands outside the loop over blocks,
  // which leaves for it (before a block's probabilities) and comes back to the block: inside the loop, however seldom it ran, the
  // compiler moved all of them for every block (2 x 2048 rows over 8000 keys, 16 heads of 256: 566 us).
  bool fresh = true, again = false, now = false;
  float keep = 1.f, key_scale = 1.f, value_scale = 0.f;
  int block = first_block;
  while (block < blocks) {
#pragma unroll
    for (int i = 0; i < kDimTiles; ++i) o[i] *= keep;
    for (; block < blocks; ++block, again = false) {
      if (!again) {
        __syncthreads();
        now = there;
        // (not 0, which a masked score of -infinity would not survive: below 1e-30 every score is 0 to all that exp2 can tell)
        key_scale = ks * fabsf(a.scale_log2);
        if (key_scale < 1e-30f) key_scale = 1e-30f;
        value_scale = vs;
        load(min(block + 1, blocks - 1));
      }
      const int at = block * kBlock;
      if (!now || at > wave_last) {
        stage((block + 1) & 1);
        continue;
      }
      const half_t *keys = tile_shared + (block & 1) * 2 * kHalves, *vals = keys + kHalves;
      const bool masked = at + kBlock - 1 > wave_first;
      float16_t score[2];
#pragma unroll
      for (int T = 0; T < 2; ++T) {
        score[T] = float16_t{};
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          const half8_t kf = *(const half8_t *)(keys + ((T * kSteps + k) * 64 + g * 32 + (m ^ (k & 15))) * 8);
          score[T] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[k], score[T], 0, 0, 0);
        }
      }
      // a row that sees none of this block takes nothing from it, also where its scales are not finite
      const bool none = at > position;
      const float factor = none ? 1.f : key_scale;
      float top = -__builtin_inff();
      if (masked) {
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (at + T * 32 + 16 * g + i > position) score[T][i] = -__builtin_inff();
      }
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, score[T][i]);
      top = fmaxf(top, __shfl_xor(top, 32)) * factor;
      const bool raise = top > most + 8.f || (most == -__builtin_inff() && top > most);
      // the value scale against its reference.  Values under a scale below 1e-12 are nothing to a binary16 result (2e-10 at most, half
      // its smallest number is 3e-8), and the accumulators need not hold what its ratio to another scale makes of them; the
      // append makes no scale below 2^-24 / 127.
      const bool nothing = value_scale < 1e-12f, scaled = !nothing && value_scale < __builtin_inff();
      const bool turn = scaled && (fresh || value_scale > 16.f * reference || value_scale * 16.f < reference);
      if (__builtin_expect(!again && (turn || __any(raise)), 0)) {
        const float next = raise ? top : most;
        keep = raise ? __builtin_amdgcn_exp2f(most - next) : 1.f;
        most = next;
        sum *= keep;
        if (turn) {
          if (!fresh) keep *= fminf(reference / value_scale, 3e38f);
          reference = value_scale, fresh = false;
        }
        if (block > first_block) {
          again = true;
          break;
        }
      }
      const float ratio = nothing ? 1.f : value_scale / reference, share = none ? 1.f : ratio;
      const float shift = __builtin_amdgcn_logf(share) - (most == -__builtin_inff() ? 0.f : most);
      half8_t pf[2][2];
      float part = 0.f;
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(score[T][i], factor, shift));
          part += p;
          pf[T][i >> 3][i & 7] = (half_t)p;
        }
      sum += part / share;
      if (nothing) {
#pragma unroll
        for (int T = 0; T < 2; ++T) pf[T][0] = pf[T][1] = half8_t{};
      }
#pragma unroll
      for (int i = 0; i < kDimTiles; ++i) {
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const half8_t vf = *(const half8_t *)(vals + (((i * 2 + T) * 2 + u) * 64 + g * 32 + (m ^ (2 * (2 * T + g)))) * 8);
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[T][u], o[i], 0, 0, 0);
          }
        // (of bytes that are not there, or behind the last block, where nobody reads them)
        stage_piece((block + 1) & 1, i / 2, i & 1);
      }
    }
  }
  const float weight = sum + __shfl_xor(sum, 32);
  const int in_tile = wave * kRowsOfWave + m, row = row0 + in_tile;
  if (row >= rows) return;
  if (a.splits > 1) {
    const int64_t slot = (int64_t)blockIdx.x * a.splits + blockIdx.y;
    float *to = a.parts + (slot * kTileRows + in_tile) * dim, *stats = a.parts + (int64_t)a.groups * a.splits * kTileRows * dim + slot * 2 * kTileRows;
    if (g == 0) stats[in_tile] = most, stats[kTileRows + in_tile] = weight;
#pragma unroll
    for (int i = 0; i < kDimTiles; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = i * 32 + c * 8 + g * 4;
        if (d < dim) *(float4_t *)(to + d) = float4_t{o[i][4 * c], o[i][4 * c + 1], o[i][4 * c + 2], o[i][4 * c + 3]} * reference;
      }
    return;
  }
  const float factor = weight == 0.f ? 0.f : reference / weight;
  half_t *to = a.out + (s.begin + row / a.group) * a.o_token + (int64_t)(h * a.group + row % a.group) * a.o_head;
#pragma unroll
  for (int i = 0; i < kDimTiles; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int d = i * 32 + c * 8 + g * 4;
      if (d >= dim) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) to[d + j] = (half_t)(o[i][4 * c + j] * factor);
    }
}

// A wave adds the parts of a row, a lane 4 dims of it; a workgroup takes 16 rows of a tile.
__global__ __launch_bounds__(kThreads) void kv_tile_join_kernel(AttentionArgs a) {
  constexpr int kAhead = 4, kRowsOfJoin = 16;
  const int dim = a.cache.dim, heads = a.cache.heads, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int b;
  uint32_t base;
  KvSequence s;
  const auto units = [&](const KvSequence &s) { return (uint32_t)(s.count * a.group + kTileRows - 1) / kTileRows * heads; };
  if (!kv_locate(a.batch, blockIdx.x, units, b, s, base)) return;
  const int rows = s.count * a.group, tiles = (rows + kTileRows - 1) / kTileRows;
  const int within = (int)(blockIdx.x - base), h = within % heads, row0 = (tiles - 1 - within / heads) * kTileRows;
  const int64_t slot0 = (int64_t)blockIdx.x * a.splits;
  const float *stats = a.parts + (int64_t)a.groups * a.splits * kTileRows * dim;
  const int d = lane * 4;
  for (int r = blockIdx.y * kRowsOfJoin + wave; r < min((int)(blockIdx.y + 1) * kRowsOfJoin, rows - row0); r += kThreads / 64) {
    float most = -__builtin_inff(), weight = 0.f;
    float4_t value = {};
    for (int i = 0; i < a.splits; i += kAhead) {
      float m[kAhead], l[kAhead];
      float4_t v[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        const int64_t slot = slot0 + min(i + n, a.splits - 1);
        m[n] = stats[slot * 2 * kTileRows + r], l[n] = stats[slot * 2 * kTileRows + kTileRows + r];
        v[n] = *(const float4_t *)(a.parts + (slot * kTileRows + r) * dim + min(d, dim - 4));
      }
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        if (i + n >= a.splits) break;
        const float next = fmaxf(most, m[n]), zero_point = next == -__builtin_inff() ? 0.f : next;
        const float keep = __builtin_amdgcn_exp2f(most - zero_point), f = __builtin_amdgcn_exp2f(m[n] - zero_point);
        value = value * keep + v[n] * f, weight = weight * keep + l[n] * f, most = next;
      }
    }
    if (d < dim) store_row(a, s, h, row0 + r, d, value, weight);
  }
}

// Adds the parts of every (sequence, head, row tile) that more than one workgroup worked on.  Workgroup w of this grid has
// boundary w + 1 of the cut; the first boundary inside a tile's units takes the tile.
__global__ __launch_bounds__(kThreads) void kv_join_kernel(AttentionArgs a) {
  constexpr int kAhead = 4;
  const int dim = a.cache.dim, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto units_of_sequence = [&](const KvSequence &s) { return units_of(a, s); };
  const Cut cut(kv_units(a.batch, units_of_sequence), a.groups);
  const uint32_t w = blockIdx.x + 1;
  if (w >= cut.groups) return;
  const uint32_t unit = cut.start(w);
  int b;
  uint32_t base;
  KvSequence s;
  if (!kv_locate(a.batch, unit, units_of_sequence, b, s, base)) return;
  const Shape shape = shape_of(a, s);
  const uint32_t which = (unit - base) / shape.blocks;
  const uint32_t from = base + which * shape.blocks, to = from + shape.blocks;
  if (unit == from || cut.start(w - 1) > from) return;
  const int h = which / shape.tiles, tile = which - h * shape.tiles;
  // (the last group at most: where offsets that do not ascend make 2^32 units or more, their number wraps, and a tile's units may
  // end behind it)
  const int first = w - 1, last = min(cut.owner(to - 1), cut.groups - 1);
  const int here = min(kRows, s.count * a.group - tile * kRows), d = lane * 4;
  const float *stats = a.parts + (int64_t)2 * a.groups * kRows * dim;
  // a wave has a row, or, of few rows, every fourth part of each
  __shared__ float4_t values[kWaves][64];
  __shared__ float maxima[kWaves], weights[kWaves];
  const bool alone = here >= kWaves;
  for (int r = alone ? wave : 0; r < here; r += alone ? kWaves : 1) {
    float most = -__builtin_inff(), weight = 0.f;
    float4_t value = {};
    const auto add = [&](float m, float l, float4_t v) {
      const float next = fmaxf(most, m), zero_point = next == -__builtin_inff() ? 0.f : next;
      const float keep = __builtin_amdgcn_exp2f(most - zero_point), f = __builtin_amdgcn_exp2f(m - zero_point);
      value = value * keep + v * f, weight = weight * keep + l * f, most = next;
    };
    const int step = alone ? 1 : kWaves;
    for (int i = first + (alone ? 0 : wave); i <= last; i += kAhead * step) {
      float m[kAhead], l[kAhead];
      float4_t v[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        // (the part of a workgroup that starts before this tile is its second one; behind the last: nothing)
        const int part = min(i + n * step, last);
        const int64_t slot = 2 * part + (part == first && cut.start(first) < from ? 1 : 0);
        m[n] = stats[slot * 2 * kRows + r], l[n] = stats[slot * 2 * kRows + kRows + r];
        v[n] = d < dim ? *(const float4_t *)(a.parts + (slot * kRows + r) * dim + d) : float4_t{};
      }
#pragma unroll
      for (int n = 0; n < kAhead; ++n)
        if (i + n * step <= last) add(m[n], l[n], v[n]);
    }
    if (!alone) {
      __syncthreads();
      values[wave][lane] = value;
      if (lane == 0) maxima[wave] = most, weights[wave] = weight;
      __syncthreads();
      if (wave > 0) continue;
#pragma unroll
      for (int w = 1; w < kWaves; ++w) add(maxima[w], weights[w], values[w][lane]);
    }
    if (d < dim) store_row(a, s, h, tile * kRows + r, d, value, weight);
  }
}

template <int DP>
int launch_split(const AttentionArgs &a, hipStream_t stream) {
  constexpr size_t lds = (size_t)kWaves * kRows * (DP + 4 + 2) * sizeof(float);
  if (const int rc = allow_lds<kv_split_kernel<DP>, lds>(lds, "kv_split_kernel")) return rc;
  kv_split_kernel<DP><<<a.groups, kThreads, lds, stream>>>(a);
  return check_launch("kv_split_kernel");
}

// Workgroups of kv_tile_kernel at most (what the sequences make of the rows only the device knows)
int64_t tile_groups(const KvBatch &batch, int heads, int group) {
  return heads * ((int64_t)batch.tokens * group / kTileRows + batch.sequences);
}

// Workgroups that share a tile: as many as fill the device (one a compute unit above 128 dims, two below), with four blocks at
// least each, if the longest sequence that the table has room for is there.
int tile_splits(int64_t groups, int64_t dim, int64_t width) {
  const int64_t fill = (dim > 128 ? kMostGroups / 2 : kMostGroups) / groups, most = width / 4;
  const int64_t splits = fill < most ? fill : most;
  return splits > 1 ? (int)splits : 1;
}

template <int DP>
int launch_tile(AttentionArgs &a, hipStream_t stream) {
  constexpr size_t lds = (size_t)2 * 2 * kBlock * DP * sizeof(half_t);
  if (const int rc = allow_lds<kv_tile_kernel<DP>, lds>(lds, "kv_tile_kernel")) return rc;
  const int64_t groups = tile_groups(a.batch, a.cache.heads, a.group);
  if (groups > 0x7fffff) return fail(GQ_ERR_UNSUPPORTED, "gq_kv_attention_f16: too many rows for one launch");
  a.groups = (int)groups, a.splits = tile_splits(groups, a.cache.dim, a.batch.width);
  kv_tile_kernel<DP><<<dim3((unsigned)groups, (unsigned)a.splits), kTileThreads, lds, stream>>>(a);
  const int rc = check_launch("kv_tile_kernel");
  if (rc != GQ_OK || a.splits == 1) return rc;
  kv_tile_join_kernel<<<dim3((unsigned)groups, kTileRows / 16), kThreads, 0, stream>>>(a);
  return check_launch("kv_tile_join_kernel");
}

}  // namespace

// The larger of what the two kernels keep: 2 x 512 parts of 16 rows, or one of 128 rows for each workgroup of a divided grid
// (512 at most, 256 above 128 dims).
int64_t kv_attention_workspace_bytes(int64_t dim) {
  return (int64_t)(dim > 128 ? kMostGroups / 2 : kMostGroups) * kTileRows * (dim + 2) * sizeof(float);
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
  a.groups = kMostGroups, a.splits = 1;
  // Both kernels are right for every batch; which is faster goes by the rows of a sequence and kv head, on average: a tile of 128
  // costs what kv_split_kernel takes for 16 to 32.  Measured at 32 rows 66 us by kv_split_kernel and 160 us by
  // kv_tile_kernel (8 sequences of up to 3000, 16 heads of 256), 67 and 94 (32 of up to 3000, 8 heads of 128), at 64
  // rows 49 and 49 (one of 4000, 16 heads of 256) and 105 and 95 (32 of up to 3000, 8 heads of 128), at 256 rows 90 and 52.
  // A batch of both kinds goes to one of them: 64 single tokens over up to 32768 beside a prompt of 1024, 32 / 8 heads of 128, take
  // 902 us, as two calls 383 + 40; 64 over up to 2048 beside a prompt of 2048, 16 heads of 256, 561 us, as two calls 201 + 112.
  // (The units of kv_split_kernel have to be countable in 31 bits.)
  const double most_units = (double)cache.heads * ((double)batch.tokens * a.group / kRows + batch.sequences) * (batch.width + 1);
  if (most_units >= 2147483648. || (int64_t)batch.tokens * a.group >= (int64_t)kTileLeast * batch.sequences)
    return cache.dim <= 64    ? launch_tile<64>(a, stream)
           : cache.dim <= 128 ? launch_tile<128>(a, stream)
                              : launch_tile<256>(a, stream);
  int rc = cache.dim <= 64 ? launch_split<64>(a, stream) : cache.dim <= 128 ? launch_split<128>(a, stream) : launch_split<256>(a, stream);
  if (rc != GQ_OK) return rc;
  kv_join_kernel<<<a.groups - 1, kThreads, 0, stream>>>(a);
  return check_launch("kv_join_kernel");
}

}  // namespace gq

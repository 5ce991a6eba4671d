// Low-rank adapters of many requests beside a shared projection:  y' = act(y + s_a (x A_a^T) B_a^T), each row its adapter a.
//   A [rank, in], B [out, rank] (the layouts that adapters are published in), s one binary32 number an adapter.
//
// adapter_plan_kernel  sorts a batch's rows by adapter once, for every projection that they pass: tiles of rows of ONE
//                      adapter, so that each product below is a plain matrix product over gathered rows.
// adapter_down_kernel  v = x A^T (contraction over the features): a split of the features per workgroup, binary32 parts.
// adapter_up_kernel    y' = act(y + s v B^T) (contraction over the rank).
//   The gradients are the same two products with the weights turned (turn_weights): dv = dy B, dx' = dx + s dv A, and
// adapter_outer_kernel dA = s dv^T x, dB = s dy^T v (contraction over rows; parts of 2048 rows, added in order by
//                      adapter_sum_kernel; no atomics anywhere, so results do not depend on timing).
//
// v is held in 32 bits.  Where it enters a second product it is split into two binary16 numbers, v = hi + lo, after a power of
// two has brought the largest of its row (or segment) near 1: 22 bits of the largest, for twice the matrix instructions of a
// contraction over no more than 128.
//
// Bound by memory: x, y, y' and the adapters in use, each once; ranks of 8 ... 64 give 2 rank flops a byte of x.
//
// Measured (TB/s of rows): 6001 rows, 4096 to 12288, rank 32: adapter_down_kernel 23 us (2.1), adapter_up_kernel 73 us (4.0).
// Gradients of 8192 rows, 4096 to 16384, rank 64: x A^T 28 us (2.4, the turned weights with it), dy B 77 us (3.5), dx 42 us
// (3.2, the operands with it), the outer products 101 us (3.3), their sum 9 us.  A decode batch of 8 rows: 4 and 4.4 us, two launches.
#include "gq_adapters.h"

namespace gq {
namespace {

// ------------------------------------------------------------------------------------------------------------- plan

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

struct PlanArgs {
  const int *ids;
  int *plan;
  int64_t counts, order, parts, small, large, segments;
  int rows, adapters;
};

// lanes of the wave with the same kind as this one
__device__ __forceinline__ uint64_t same_kind(int kind, bool valid) {
  uint64_t mask = __ballot(valid);
#pragma unroll
  for (int bit = 0; bit < 12; ++bit) {  // kMostAdapters + 1 kinds
    const uint64_t set = __ballot(kind >> bit & 1);
    mask &= (kind >> bit & 1) ? set : ~set;
  }
  return mask;
}

// An adapter's rows in the lists of tiles and segments.
struct Listed {
  int adapter, rows, begin, small, large, segment, part;
};

__device__ __forceinline__ void list(const PlanArgs &a, const Listed &l, int first, int step) {
  for (int i = first; i * kAdapterSmallTile < l.rows; i += step)
    ((AdapterTile *)(a.plan + a.small))[l.small + i] =
        AdapterTile{l.adapter, l.begin + i * kAdapterSmallTile, min(l.rows - i * kAdapterSmallTile, kAdapterSmallTile)};
  for (int i = first; i * kAdapterLargeTile < l.rows; i += step)
    ((AdapterTile *)(a.plan + a.large))[l.large + i] =
        AdapterTile{l.adapter, l.begin + i * kAdapterLargeTile, min(l.rows - i * kAdapterLargeTile, kAdapterLargeTile)};
  if (l.adapter < 0) return;
  for (int i = first; i * kAdapterSegment < l.rows; i += step)
    ((AdapterTile *)(a.plan + a.segments))[l.segment + i] =
        AdapterTile{l.adapter, l.begin + i * kAdapterSegment, min(l.rows - i * kAdapterSegment, kAdapterSegment),
                    l.small + i * (kAdapterSegment / kAdapterSmallTile), l.large + i * (kAdapterSegment / kAdapterLargeTile),
                    l.part < 0 ? -1 : l.part + i};
}

// One workgroup, for a plan serves every projection of a batch and is small beside them (150 rows 7.6 us, 8192 rows 22 us, 65536
// rows 145 us; bound by the chain of two passes over the ids, 64 rows of a wave at a time).  Wave w takes the w-th stretch of
// rows: it counts them by kind (adapter, or none = the last kind), a scan over kinds and waves gives every (kind, wave) its
// place, and the wave puts its rows there in their order.
__global__ __launch_bounds__(kPlanThreads) void adapter_plan_kernel(PlanArgs a) {
  extern __shared__ int count[];  // [waves][kinds]
  __shared__ int wave_sum[4][kPlanWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kinds = a.adapters + 1;
  const int stretch = (a.rows + kPlanThreads - 1) / kPlanThreads * 64;
  const int row0 = min(a.rows, wave * stretch), row1 = min(a.rows, row0 + stretch);
  for (int n = tid; n < kPlanWaves * kinds; n += kPlanThreads) count[n] = 0;
  __syncthreads();
  volatile int *mine = count + wave * kinds;
  for (int r = row0; r < row1; r += 64) {
    const bool valid = r + lane < row1;
    int kind = valid ? a.ids[r + lane] : 0;
    if (kind < 0 || kind >= a.adapters) kind = a.adapters;
    const uint64_t same = same_kind(kind, valid);
    if (valid && __builtin_ctzll(same) == lane) mine[kind] = mine[kind] + __builtin_popcountll(same);
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  // each thread scans three kinds at most (kMostAdapters + 1 <= 3 x 1024)
  constexpr int kEach = (kMostAdapters + kPlanThreads) / kPlanThreads;
  const int each = (kinds + kPlanThreads - 1) / kPlanThreads;
  int total[kEach], own[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int kind = tid * each + e;
    total[e] = 0;
    if (e >= each || kind >= kinds) continue;
    for (int w = 0; w < kPlanWaves; ++w) total[e] += count[w * kinds + kind];
    own[0] += total[e];
    own[1] += (total[e] + kAdapterSmallTile - 1) / kAdapterSmallTile;
    own[2] += (total[e] + kAdapterLargeTile - 1) / kAdapterLargeTile;
    own[3] += kind < a.adapters ? (total[e] + kAdapterSegment - 1) / kAdapterSegment : 0;
  }
  int before[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int sum = own[i];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    before[i] = sum - own[i];
    if (lane == 63) wave_sum[i][wave] = sum;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int all = 0;
    for (int w = 0; w < kPlanWaves; ++w) {
      if (w < wave) before[i] += wave_sum[i][w];
      all += wave_sum[i][w];
    }
    if (tid == 0 && i > 0) a.plan[a.counts + i - 1] = all;
  }
  // Parts: the segments of adapters that have several, in the same order, counted apart (an adapter of one segment writes
  // its gradient itself).
  __syncthreads();
  int several = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int kind = tid * each + e, n = (total[e] + kAdapterSegment - 1) / kAdapterSegment;
    if (e < each && kind < a.adapters && n > 1) several += n;
  }
  int part = several;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(part, d);
    if (lane >= d) part += up;
  }
  if (lane == 63) wave_sum[0][wave] = part;
  part -= several;
  __syncthreads();
  for (int w = 0; w < wave; ++w) part += wave_sum[0][w];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int kind = tid * each + e;
    const bool valid = e < each && kind < kinds;
    Listed l = {valid && kind < a.adapters ? kind : -1, valid ? total[e] : 0, before[0], before[1], before[2], before[3], 0};
    const int segments = l.adapter >= 0 ? (l.rows + kAdapterSegment - 1) / kAdapterSegment : 0;
    l.part = segments > 1 ? part : -1;
    // an adapter of few rows is listed by its thread, one of many by the wave
    if (l.rows <= kAdapterLargeTile) list(a, l, 0, 1);
    for (uint64_t many = __ballot(l.rows > kAdapterLargeTile); many; many &= many - 1) {
      const int from = __builtin_ctzll(many);
      const Listed other = {__builtin_amdgcn_readlane(l.adapter, from), __builtin_amdgcn_readlane(l.rows, from),
                            __builtin_amdgcn_readlane(l.begin, from), __builtin_amdgcn_readlane(l.small, from),
                            __builtin_amdgcn_readlane(l.large, from), __builtin_amdgcn_readlane(l.segment, from),
                            __builtin_amdgcn_readlane(l.part, from)};
      list(a, other, lane, 64);
    }
    if (!valid) continue;
    if (l.adapter >= 0) {
      a.plan[a.parts + 2 * kind] = part, a.plan[a.parts + 2 * kind + 1] = segments;
      if (segments > 1) part += segments;
    }
    before[1] += (l.rows + kAdapterSmallTile - 1) / kAdapterSmallTile;
    before[2] += (l.rows + kAdapterLargeTile - 1) / kAdapterLargeTile;
    before[3] += segments;
    int at = l.begin;
    for (int w = 0; w < kPlanWaves; ++w) {
      const int c = count[w * kinds + kind];
      count[w * kinds + kind] = at;
      at += c;
    }
    before[0] = at;
  }
  __syncthreads();
  for (int r = row0; r < row1; r += 64) {
    const bool valid = r + lane < row1;
    int kind = valid ? a.ids[r + lane] : 0;
    if (kind < 0 || kind >= a.adapters) kind = a.adapters;
    const uint64_t same = same_kind(kind, valid);
    const int at = mine[kind];
    __builtin_amdgcn_wave_barrier();
    if (valid) {
      a.plan[a.order + at + __builtin_popcountll(same & (((uint64_t)1 << lane) - 1))] = r + lane;
      if (__builtin_ctzll(same) == lane) mine[kind] = at + __builtin_popcountll(same);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// --------------------------------------------------------------------------------------------------------- products

constexpr int kThreads = 256, kWaves = 4;

// 8 values from p, of which `valid` exist (the rest are zeros); kWide: all or none of them, 16-byte aligned.  Rows that are not
// (4097 features to 4095, 4096 rows, rank 16) take 201 us where aligned ones of 4096 take 34, rank 15 with aligned rows 104.
template <bool kWide>
__device__ __forceinline__ half8_t load8(const half_t *p, int64_t valid) {
  half8_t v = {};
  if (kWide) {
    if (valid > 0) v = *(const half8_t *)p;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) v[i] = p[i];
  }
  return v;
}

// The same where the other operand is zero at values that do not exist: row[at ... at + 7] of a row of `size`, or others of it.
template <bool kWide>
__device__ __forceinline__ half8_t load8_any(const half_t *row, int64_t at, int64_t size) {
  if (kWide) return *(const half8_t *)(row + min(at, size - 8));
  return load8<false>(row + at, size - at);
}

// The gradients contract the other axis of each weight: both are turned first, [rows][columns] to [columns][rows] for every
// adapter that has rows (a gradient of 4 bytes an element is written for every one of them, so this never dominates), by workgroups
// of the launch that forms x A^T, which does not need them: a launch less, and its time is hidden.
struct TurnArgs {
  const half_t *from[2];
  half_t *to[2];
  int64_t rows[2], columns[2];
  const int *parts_of;
  int pieces, adapters;  // of the grid
  bool wide;  // rows and columns of both are multiples of 8, 16-byte aligned
};

// workgroup `group` of a.pieces x adapters x 2; 64 x 72 of LDS
__device__ __forceinline__ void turn_weights(const TurnArgs &a, int group, half_t (*piece)[72]) {
  const int first = group % a.pieces, adapter = group / a.pieces % a.adapters, which = group / a.pieces / a.adapters, tid = threadIdx.x;
  if (a.parts_of[2 * adapter + 1] == 0) return;
  const int64_t rows = which ? a.rows[1] : a.rows[0], columns = which ? a.columns[1] : a.columns[0];
  const int64_t across = (columns + 63) / 64, pieces = (rows + 63) / 64 * across;
  const half_t *from = (which ? a.from[1] : a.from[0]) + adapter * rows * columns;
  half_t *to = (which ? a.to[1] : a.to[0]) + adapter * rows * columns;
  for (int64_t n = first; n < pieces; n += a.pieces) {
    const int64_t r0 = n / across * 64, c0 = n % across * 64;
    __syncthreads();
#pragma unroll
    for (int i = tid; i < 64 * 8; i += kThreads) {
      const int64_t r = r0 + i / 8, c = c0 + i % 8 * 8;
      if (r >= rows) continue;
      *(half8_t *)&piece[i / 8][i % 8 * 8] = a.wide ? load8<true>(from + r * columns + c, columns - c) : load8<false>(from + r * columns + c, columns - c);
    }
    __syncthreads();
#pragma unroll
    for (int i = tid; i < 64 * 8; i += kThreads) {
      const int64_t c = c0 + i / 8, r = r0 + i % 8 * 8;
      if (c >= columns) continue;
      half8_t v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = piece[i % 8 * 8 + j][i / 8];
      if (a.wide) {
        if (r < rows) *(half8_t *)(to + c * rows + r) = v;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (r + j < rows) to[c * rows + r + j] = v[j];
      }
    }
  }
}

struct DownArgs {
  const half_t *x, *w;  // w: [adapters][rank][features]
  int64_t x_stride;
  const AdapterTile *tiles;
  const int *tile_count, *order;
  float *v;     // [splits][rows][kRank]
  float *most;  // [splits][tiles]: largest magnitudes (NULL: nobody asks)
  int64_t rows, features, split;  // features of one split, a multiple of 128
  int rank, most_tiles, splits;
  TurnArgs turn;  // what the workgroups behind most_tiles x splits do
};

// kRank: rank rounded up to 32, 64 or 128; kTiles x 16 rows.  The four waves of a workgroup have a quarter of its features
// each, their binary32 sums meet in LDS.  v^T = A x^T: a lane ends with 4 consecutive ranks of one row.  The operands of the
// next 64 features are loaded before this step's products: a wave has little else to hide the latency with.
template <int kRank, int kTiles, bool kWide>
__global__ __launch_bounds__(kThreads, kRank * kTiles > 256 ? 1 : 2) void adapter_down_kernel(DownArgs a) {
  constexpr int kRankTiles = kRank / 16;
  extern __shared__ float shared[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
  const int split = blockIdx.x / a.most_tiles, index = blockIdx.x - split * a.most_tiles;
  if (split >= a.splits) {
    turn_weights(a.turn, blockIdx.x - a.splits * a.most_tiles, (half_t(*)[72])shared);
    return;
  }
  if (index >= *a.tile_count) return;
  const AdapterTile tile = a.tiles[index];
  if (tile.adapter < 0) return;
  const int64_t mine = a.split / kWaves, from = min(a.features, split * a.split + wave * mine), to = min(a.features, from + mine);
  const half_t *w = a.w + (int64_t)tile.adapter * a.rank * a.features;
  const half_t *x[kTiles], *wr[kRankTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) x[t] = a.x + (int64_t)a.order[tile.begin + min(t * 16 + m, tile.count - 1)] * a.x_stride;
#pragma unroll
  for (int r = 0; r < kRankTiles; ++r) wr[r] = w + (int64_t)min(r * 16 + m, a.rank - 1) * a.features;

  float4_t acc[kRankTiles][kTiles];
#pragma unroll
  for (int r = 0; r < kRankTiles; ++r)
#pragma unroll
    for (int t = 0; t < kTiles; ++t) acc[r][t] = float4_t{};
  // 64 features a step, so that a row's 128 bytes are asked for together.  Loads are made without conditions (of other
  // values of the row where it ends): a register that a load fills on one path only is copied, and the copy waits for it.
  half8_t xf[2][kTiles][2], wf[2][kRankTiles][2];
  const auto load = [&](int set, int64_t k) {
    k += g * 8;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) xf[set][t][u] = load8_any<kWide>(x[t], k + 32 * u, a.features);
#pragma unroll
    for (int r = 0; r < kRankTiles; ++r)
#pragma unroll
      for (int u = 0; u < 2; ++u) wf[set][r][u] = load8_any<kWide>(wr[r], k + 32 * u, a.features);
  };
  const auto multiply = [&](int set, int64_t k) {
    if (k + 64 > to) {  // values behind the range are zeros on both sides (`to` is a multiple of 8 or the row's end)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (k + 32 * u + g * 8 < to) continue;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) xf[set][t][u] = half8_t{};
#pragma unroll
        for (int r = 0; r < kRankTiles; ++r) wf[set][r][u] = half8_t{};
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < kRankTiles; ++r) {
        if (r * 16 >= a.rank) continue;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
          acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[set][r][u], xf[set][t][u], acc[r][t], 0, 0, 0);
      }
  };
  // Tiles start at different places of their range: rows are often a power of two apart, and tiles that walked their columns in
  // step would keep asking the same few memory channels (8192 rows of 16384: 87 us, 74 us so).
  const int steps = (int)((to - from + 63) / 64), turn = steps > 0 ? index * 5 % steps : 0;
  const auto place = [&](int i) {
    const int at = turn + min(i, steps - 1);
    return from + 64 * (int64_t)(at < steps ? at : at - steps);
  };
  if (steps > 0) {
    load(0, place(0));
    for (int i = 0; i < steps; i += 2) {
      load(1, place(i + 1));
      multiply(0, place(i));
      load(0, place(i + 2));
      if (i + 1 < steps) multiply(1, place(i + 1));
    }
  }
  // sum of the four waves, 16 rows at a time: [waves][16 rows][kRank + 4]
  float *v = a.v + ((int64_t)split * a.rows + tile.begin) * kRank;
  float most = 0.f;
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    if (t * 16 >= tile.count) break;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRankTiles; ++r) *(float4_t *)(shared + (wave * 16 + m) * (kRank + 4) + r * 16 + 4 * g) = acc[r][t];
    __syncthreads();
    for (int n = threadIdx.x; n < 4 * kRank; n += kThreads) {
      const int row = n / (kRank / 4), r = n % (kRank / 4) * 4;
      float4_t sum = {};
#pragma unroll
      for (int i = 0; i < kWaves; ++i) sum += *(const float4_t *)(shared + (i * 16 + row) * (kRank + 4) + r);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (r + j >= a.rank) sum[j] = 0.f;
        if (t * 16 + row < tile.count) most = fmaxf(most, fabsf(sum[j]));
      }
      if (t * 16 + row < tile.count) *(float4_t *)(v + (int64_t)(t * 16 + row) * kRank + r) = sum;
    }
  }
  if (a.most) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    __syncthreads();
    if (lane == 0) shared[wave] = most;
    __syncthreads();
    if (threadIdx.x == 0)
      a.most[(int64_t)split * a.most_tiles + index] = fmaxf(fmaxf(shared[0], shared[1]), fmaxf(shared[2], shared[3]));
  }
}

// two binary16 numbers whose sum is v to 22 bits of 1
__device__ __forceinline__ void split_of(float v, half_t &hi, half_t &lo) {
  hi = (half_t)v;
  lo = (half_t)(fabsf(v) < __builtin_inff() ? v - (float)hi : 0.f);
}

// the power of two that brings `most` into [1/2, 1), and its inverse (1 where there is nothing to bring there)
__device__ __forceinline__ float normal_power(float most, float &back) {
  int e = 0;
  if (most > 0.f && most < __builtin_inff()) (void)frexpf(most, &e);
  e = min(max(e, -100), 100);
  back = ldexpf(1.f, e);
  return ldexpf(1.f, -e);
}

// The epilogue on 8 values.  The tanh form of gelu is v s(2 u), s the logistic function: one exponential, where tanhf for
// each of a lane's 64 values would make the kernel's code outgrow the instruction cache.
__device__ __forceinline__ void activate(float (&v)[8], int act) {
  if (act == GQ_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];
  } else if (act == GQ_ACT_GELU_TANH) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float u = 0.7978845608028654f * (v[j] + 0.044715f * (v[j] * v[j] * v[j]));
      v[j] = v[j] / (1.f + __builtin_amdgcn_exp2f(-2.8853900817779268f * u));  // 2 log2(e)
    }
  }
}

// v summed over the splits, `p` a row's 4 ranks: four loads in flight
__device__ __forceinline__ float4_t sum_of_splits(const float *p, int64_t stride, int splits) {
  float4_t sum = {};
  int s = 0;
  for (; s + 4 <= splits; s += 4) {
    float4_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = *(const float4_t *)(p + (s + i) * stride);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += u[i];
  }
  for (; s < splits; ++s) sum += *(const float4_t *)(p + s * stride);
  return sum;
}

struct OuterSide {
  const half_t *x;  // [rows][features]
  int64_t x_stride, features;
  const float *v;     // [splits][rows][kRank]
  const float *most;  // [splits][tiles]
  int splits;
  half_t *operand;  // [row of operand_row / 32][hi, lo][16 ranks][lane][8]: 1 KiB for a wave's load
  float *back;      // [segments]
  float *grad;      // [adapters][rank][features], turned: [adapters][features][rank]
  float *parts;     // [parts], the same
  bool turned;
};

struct OuterArgs {
  OuterSide side[2];
  const AdapterTile *segments;
  const int *segment_count, *order, *parts_of;
  const float *scaling;
  int64_t rows;
  int rank, adapters, most_tiles, most_segments;
  bool large;
};

// Where a segment's rows begin in the operands: pieces of 64 rows, the segments apart (their rows are consecutive in the order,
// and 64 rows more for each keep rounded ones from meeting).
__device__ __forceinline__ int64_t operand_row(int segment, int begin) { return (int64_t)(begin / 64 + segment) * 64; }

// v of a segment as the other product's operand: 64 rows a workgroup, summed over the splits, scaled by the segment's power of
// two, split, transposed.  The power comes from the largest part times the number of splits, which is no less than the
// largest sum; what it is too large by costs that many of the 22 bits.
// Workgroup `group` of segments x pieces x 2; [2][kRank][72] of LDS.
template <int kRank>
__device__ __forceinline__ void make_operand(const OuterArgs &a, int group, half_t *shared) {
  constexpr int kRow = 64 + 8;
  half_t(*piece)[kRank][kRow] = (half_t(*)[kRank][kRow])shared;
  const int segment = group % a.most_segments, part = group / a.most_segments;
  const OuterSide &side = part & 1 ? a.side[1] : a.side[0];
  if (segment >= *a.segment_count) return;
  const AdapterTile seg = a.segments[segment];
  const int i0 = (part >> 1) * 64, tid = threadIdx.x, lane = tid & 63;
  if (i0 >= seg.count) return;
  const int per_tile = a.large ? kAdapterLargeTile : kAdapterSmallTile, tiles = (seg.count + per_tile - 1) / per_tile;
  const float *most_of = side.most + (a.large ? seg.first_large : seg.first);
  float most = 0.f;
  for (int n = lane; n < tiles * side.splits; n += 64) most = fmaxf(most, most_of[(int64_t)(n / tiles) * a.most_tiles + n % tiles]);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
  most *= side.splits;
  float back;
  const float power = normal_power(most, back);
  if (i0 == 0 && tid == 0) side.back[segment] = back * a.scaling[seg.adapter];
  for (int n = tid; n < 64 * kRank / 4; n += kThreads) {
    const int i = n / (kRank / 4), r = n % (kRank / 4) * 4;
    float4_t sum = {};
    if (i0 + i < seg.count) sum = sum_of_splits(side.v + (int64_t)(seg.begin + i0 + i) * kRank + r, a.rows * kRank, side.splits);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      half_t h, l;
      split_of(sum[j] * power, h, l);
      piece[0][r + j][i] = h, piece[1][r + j][i] = l;
    }
  }
  __syncthreads();
  half_t *to = side.operand + (operand_row(segment, seg.begin) + i0) * 2 * kRank;
  for (int n = tid; n < 2 * 2 * kRank * 4; n += kThreads) {
    const int m = n % 16, g = n / 16 % 4, r = n / 64 % (kRank / 16), which = n / (kRank * 4) % 2, step = n / (kRank * 8);
    *(half8_t *)(to + n * 8) = *(const half8_t *)&piece[which][r * 16 + m][step * 32 + g * 8];
  }
}

struct UpArgs {
  const float *v;   // [splits][rows][kRank]
  const half_t *w;  // [adapters][features][rank]
  const float *scaling;
  const half_t *y;  // out where there is none
  half_t *out;
  int64_t y_stride, out_stride;
  bool has_y;
  const AdapterTile *tiles;
  const int *tile_count, *order;
  int64_t rows, features, range;  // features of one workgroup, a multiple of 256
  int rank, splits, act;
  int ranges;
  OuterArgs outer;  // gradients: the workgroups behind tiles x ranges make its operand
  int most_tiles;
  bool skip_rows_without;  // out is y and there is no activation: rows without an adapter are done
};

// The workgroup sums its rows' v over the splits into LDS, where its waves take their operands from.  Then wave w takes 64
// features at a time: row 4 g' + i of operand tile f is feature 32 (f / 2) + 8 g' + 4 (f % 2) + i, so that a lane ends with 8
// consecutive features of one row in each half.  From there they go through the wave's own LDS to the lanes that have these rows
// of y, 8 to a row: loads and stores are whole lines (stored by halves of a line from the accumulators' own lanes, 6001 rows to 12288
// took 88 us, so 73).  The weights and y of the next piece are loaded before and among this one's products.
template <int kRank, int kTiles, bool kWide>
__global__ __launch_bounds__(kThreads, kRank * kTiles > 256 ? 1 : 2) void adapter_up_kernel(UpArgs a) {
  constexpr int kChunks = kRank / 32, kRow = kRank + 4, kTurned = 64 + 4;
  extern __shared__ float v[];  // [kTiles x 16 rows][kRow], then [waves][16 rows][kTurned]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
  const int range = blockIdx.x / a.most_tiles, index = blockIdx.x - range * a.most_tiles;
  if (range >= a.ranges) {
    make_operand<kRank>(a.outer, blockIdx.x - a.ranges * a.most_tiles, (half_t *)v);
    return;
  }
  if (index >= *a.tile_count) return;
  const AdapterTile tile = a.tiles[index];
  const bool with = tile.adapter >= 0;
  if (!with && a.skip_rows_without) return;
  const half_t *w = a.w + (int64_t)max(tile.adapter, 0) * a.rank * a.features;
  const float scaling = with ? a.scaling[tile.adapter] : 0.f;
  const int64_t from = range * a.range, to = min(a.features, from + a.range), first = from + wave * 64;
  // (tiles start at different pieces of the range and loads have no conditions, as in adapter_down_kernel)
  const int pieces = first < to ? (int)((to - first + kWaves * 64 - 1) / (kWaves * 64)) : 0, turn = pieces > 0 ? index * 5 % pieces : 0;
  const auto place = [&](int i) {
    if (pieces == 0) return (int64_t)0;  // (a wave without features still loads, and drops, the first ones)
    const int at = turn + min(i, pieces - 1);
    return first + (int64_t)(at < pieces ? at : at - pieces) * (kWaves * 64);
  };

  half8_t wf[2][4][kChunks], y[kTiles][2];
  int64_t row[kTiles][2];
  const auto load_weights = [&](int set, int64_t n0) {
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const half_t *p = w + min(n0 + 32 * (f >> 1) + 8 * (m >> 2) + 4 * (f & 1) + (m & 3), a.features - 1) * a.rank;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        wf[set][f][c] = load8_any<kWide>(p, c * 32 + g * 8, a.rank);
    }
  };
  const auto load_y = [&](int t, int64_t n0) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      y[t][half] = load8_any<kWide>(a.y + row[t][half] * a.y_stride, n0 + (lane & 7) * 8, a.features);
    }
  };
  load_weights(0, place(0));
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int half = 0; half < 2; ++half) row[t][half] = a.order[tile.begin + min(t * 16 + half * 8 + (lane >> 3), tile.count - 1)];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) load_y(t, place(0));

  half8_t hi[kTiles][kChunks] = {}, lo[kTiles][kChunks] = {};
  float back[kTiles] = {};
  if (with) {
    for (int n = threadIdx.x; n < tile.count * (kRank / 4); n += kThreads) {
      const int i = n / (kRank / 4), r = n % (kRank / 4) * 4;
      *(float4_t *)(v + i * kRow + r) = sum_of_splits(a.v + (int64_t)(tile.begin + i) * kRank + r, a.rows * kRank, a.splits);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const float *p = v + min(t * 16 + m, tile.count - 1) * kRow + g * 8;
      float most = 0.f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(p[c * 32 + j]));
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      const float power = normal_power(most, back[t]);
      back[t] *= scaling;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          half_t h, l;
          split_of(p[c * 32 + j] * power, h, l);
          hi[t][c][j] = h, lo[t][c][j] = l;
        }
    }
  }

  float *turned = v + kTiles * 16 * kRow + wave * 16 * kTurned;
  const uint32_t y_mask = a.has_y ? ~0u : 0u;
  const auto piece = [&](int set, int64_t n0, int64_t next) {
    load_weights(set ^ 1, next);
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      float4_t acc[4];
#pragma unroll
      for (int f = 0; f < 4; ++f) acc[f] = float4_t{};
      if (with) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          if (c * 32 >= a.rank) continue;
#pragma unroll
          for (int f = 0; f < 4; ++f) acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[set][f][c], hi[t][c], acc[f], 0, 0, 0);
#pragma unroll
          for (int f = 0; f < 4; ++f) acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[set][f][c], lo[t][c], acc[f], 0, 0, 0);
        }
      }
      // through LDS into the order of y: 8 lanes hold a row's 64 features, a line of memory each
#pragma unroll
      for (int f = 0; f < 4; ++f) *(float4_t *)(turned + m * kTurned + 32 * (f >> 1) + 8 * g + 4 * (f & 1)) = acc[f] * back[t];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      half8_t r[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const half8_t base = __builtin_bit_cast(half8_t, __builtin_bit_cast(uint4_t, y[t][half]) & y_mask);
        const float *p = turned + (half * 8 + (lane >> 3)) * kTurned + (lane & 7) * 8;
        const float4_t first4 = *(const float4_t *)p, second4 = *(const float4_t *)(p + 4);
        float sum[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] = (float)base[j] + (j < 4 ? first4[j & 3] : second4[j & 3]);
        activate(sum, a.act);
#pragma unroll
        for (int j = 0; j < 8; ++j) r[half][j] = (half_t)sum[j];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      load_y(t, next);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (t * 16 + half * 8 + (lane >> 3) >= tile.count) continue;
        const int64_t n = n0 + (lane & 7) * 8;
        half_t *o = a.out + row[t][half] * a.out_stride + n;
        if (kWide) {
          if (n < to) *(half8_t *)o = r[half];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (n + j < to) o[j] = r[half][j];
        }
      }
    }
  };
  for (int i = 0; i < pieces; i += 2) {
    piece(0, place(i), place(i + 1));
    if (i + 1 < pieces) piece(1, place(i + 1), place(i + 2));
  }
}

// 128 features of one segment's product; the four waves take every fourth 32 rows and meet in LDS.  The rows are loaded as
// they lie (8 features a lane, 8 rows) and paired in registers: operand c has feature 8 m + c, so that a lane ends with 8
// consecutive features of 4 ranks.  Rows are loaded two steps ahead, the operand one: one wave a SIMD with 512 registers keeps
// more bytes on their way than two with 256 (whose steps waited for the operand).
template <int kRank, bool kWide>
__global__ __launch_bounds__(kThreads, 1) void adapter_outer_kernel(OuterArgs a) {
  constexpr int kRankTiles = kRank / 16 < 4 ? kRank / 16 : 4;  // 64 ranks at most at a time: blockIdx.z
  constexpr int kRow = 128 + 4;
  __shared__ float shared[kWaves * 16 * kRow];  // at first the segment's rows
  int *order = (int *)shared;
  static_assert(sizeof(shared) >= kAdapterSegment * sizeof(int), "a segment's rows fit");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
  // dy before x and its last features first: what was read last may still be in a cache (8192 rows: 106 us, 101 us so)
  const bool second = !(blockIdx.z & 1);
  const int64_t f0 = (int64_t)(gridDim.y - 1 - blockIdx.y) * 128;
  const int rank0 = (blockIdx.z >> 1) * 64;
  const OuterSide &side = second ? a.side[1] : a.side[0];
  if ((int)blockIdx.x >= *a.segment_count || f0 >= side.features || rank0 >= a.rank) return;
  const AdapterTile seg = a.segments[blockIdx.x];
  for (int n = threadIdx.x; n < seg.count; n += kThreads) order[n] = a.order[seg.begin + n];
  __syncthreads();
  // (in the order of the loads: rows of it a power of two apart would all be asked of one memory channel)
  const half_t *operand = side.operand + operand_row(blockIdx.x, seg.begin) * 2 * kRank + rank0 * 32 + lane * 8;
  const int last_step = (seg.count - 1) / 32 * 32;
  const int64_t f = f0 + m * 8;

  float4_t acc[kRankTiles][8];
#pragma unroll
  for (int r = 0; r < kRankTiles; ++r)
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[r][c] = float4_t{};
  // Loads are made without conditions (of the last rows and operands again where there are no more), for a register that a load
  // fills on one path only is copied, and the copy waits for it.
  half8_t x[2][8], h[2][kRankTiles], l[2][kRankTiles];
  const auto load = [&](int set, int i0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // (rows behind the last have zeros in the other operand; features behind the last are not stored)
      const int i = min(i0 + g * 8 + j, seg.count - 1);
      x[set][j] = load8_any<kWide>(side.x + (int64_t)order[i] * side.x_stride, f, side.features);
    }
  };
  const auto load_operand = [&](int set, int i0) {
    const half_t *at = operand + (int64_t)min(i0, last_step) * 2 * kRank;
#pragma unroll
    for (int r = 0; r < kRankTiles; ++r) {
      h[set][r] = *(const half8_t *)(at + r * 512);
      l[set][r] = *(const half8_t *)(at + kRank * 32 + r * 512);
    }
  };
  constexpr int kStep = kWaves * 32;
  const auto multiply = [&](int set, int i0) {
    half8_t xf[8];
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) xf[c][j] = x[set][j][c];
    // (the operand first: loads arrive in order, and it is needed a step before these rows)
    load_operand(set ^ 1, i0 + kStep);
    load(set, i0 + 2 * kStep);
    if (i0 >= seg.count) return;
#pragma unroll
    for (int r = 0; r < kRankTiles; ++r) {
      if (rank0 + r * 16 >= a.rank) continue;
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h[set][r], xf[c], acc[r][c], 0, 0, 0);
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[set][r], xf[c], acc[r][c], 0, 0, 0);
    }
  };
  const int start = wave * 32;
  load_operand(0, start);
  load(0, start);
  load(1, start + kStep);
  for (int i0 = start; i0 < seg.count; i0 += 2 * kStep) {
    multiply(0, i0);
    multiply(1, i0 + kStep);
  }
  const float back = side.back[blockIdx.x];
  float *out = seg.part < 0 ? side.grad + (int64_t)seg.adapter * a.rank * side.features : side.parts + (int64_t)seg.part * a.rank * side.features;
#pragma unroll
  for (int r = 0; r < kRankTiles; ++r) {
    if (rank0 + r * 16 >= a.rank) continue;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float *to = shared + (wave * 16 + 4 * g + i) * kRow + m * 8;
      *(float4_t *)to = float4_t{acc[r][0][i], acc[r][1][i], acc[r][2][i], acc[r][3][i]};
      *(float4_t *)(to + 4) = float4_t{acc[r][4][i], acc[r][5][i], acc[r][6][i], acc[r][7][i]};
    }
    __syncthreads();
    for (int n = threadIdx.x; n < 16 * 128; n += kThreads) {
      // (a gradient [features][rank] is written 16 ranks of a feature at a time)
      const int rr = side.turned ? n % 16 : n / 128, ff = side.turned ? n / 16 : n % 128;
      const int rank = rank0 + r * 16 + rr;
      const int64_t feature = f0 + ff;
      if (rank >= a.rank || feature >= side.features) continue;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) sum += shared[(w * 16 + rr) * kRow + ff];
      out[side.turned ? feature * a.rank + rank : rank * side.features + feature] = sum * back;
    }
  }
}

// The parts of adapters of several segments, added in their order; zeros for adapters without rows.
__global__ __launch_bounds__(kThreads) void adapter_sum_kernel(OuterArgs a) {
  const OuterSide &side = blockIdx.z ? a.side[1] : a.side[0];
  const int adapter = blockIdx.y, first = a.parts_of[2 * adapter], segments = a.parts_of[2 * adapter + 1];
  if (segments == 1) return;
  const int64_t size = a.rank * side.features;
  float *grad = side.grad + adapter * size;
  const float *parts = side.parts + first * size;
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < size; n += (int64_t)gridDim.x * kThreads) {
    float sum = 0.f;
    for (int s = 0; s < segments; ++s) sum += parts[s * size + n];
    grad[n] = sum;
  }
}

// ----------------------------------------------------------------------------------------------------------- launches

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int rank_class(int64_t rank) { return rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

// Workgroups that fill the device twice over where the features allow it, each with at least 512 features (128 a wave).  With
// once, twice, four times as many: 31, 25, 32 us (6001 rows of 4096, rank 32), 127, 79, 81 us (8192 rows of 16384, rank 64).
int64_t down_splits(int64_t tiles, int64_t features) {
  const int64_t most = (features + 511) / 512, want = (512 + tiles - 1) / tiles;
  return want < most ? want : most > 0 ? most : 1;
}

// As many workgroups as are resident together, no more: each sums its tile's v anew, and a few behind the others cost as much as
// a whole turn of them (6001 rows to 12288, rank 32, 376 tiles: 2, 3, 6 ranges 74, 80, 77 us; 8192 rows to 4096, rank 64, 128
// tiles: 4, 8 ranges 43, 52 us; 150 rows to 16384, rank 64: 13, 16, 32 ranges 27, 24, 29 us).  It is a whole number, so a few
// tiles more can halve the workgroups: 4096 to 4096, rank 16, 8180 rows, 532, 542, 557, 602 tiles: 63, 65, 73, 71 us.  `tiles` counts
// the last one of every adapter: an eighth of them may be nobody's.
int64_t up_ranges(int64_t tiles, int64_t rank, bool large) {
  const int64_t resident = large || rank > 64 ? 512 : 1024, ranges = (resident + tiles / 8) / tiles;
  return ranges > 0 ? ranges : 1;
}

// Rows of a tile: 16 for decode batches, whose rows mostly have adapters of their own, and as long as tiles of 64 would not
// fill the device; 64 where an adapter's weights are worth reading once for more rows, the sooner the higher the rank (but ranks
// above 64 leave tiles of 64 rows one wave a SIMD).  Projection with 8 adapters, 4096 features to 4096 (* to 12288), us with
// tiles of 16 and 64: rank 16, rows 1024: 17 and 20, 4096: 34 and 43, 8192*: 130 and 126, rank 32, 32768: 229 and 209;
// rank 64, rows 512: 23 and 23, 1024: 31 and 28, 8192: 118 and 91; rank 128, rows 2048*: 121 and 134, 4096*: 196 and 181,
// 8192: 198 and 169.
bool large_tiles(int64_t rows, int64_t rank) { return rows >= (rank <= 32 ? 8192 : rank <= 64 ? 1024 : 4096); }

struct Batch {
  const PlanLayout plan;
  const int *words;
  bool large;
  const AdapterTile *tiles() const { return (const AdapterTile *)(words + (large ? plan.large : plan.small)); }
  int64_t most_tiles() const { return large ? plan.most_large : plan.most_small; }
};

template <int kRank, int kTiles, bool kWide>
int start_down(const DownArgs &a, int64_t turns, hipStream_t stream) {
  const size_t sums = (size_t)kWaves * 16 * (kRank + 4) * sizeof(float), turned = turns ? 64 * 72 * sizeof(half_t) : 0;
  adapter_down_kernel<kRank, kTiles, kWide>
      <<<(unsigned)((int64_t)a.most_tiles * a.splits + turns), kThreads, sums > turned ? sums : turned, stream>>>(a);
  return check_launch("adapter_down_kernel");
}

template <int kRank, int kTiles, bool kWide>
int start_up(const UpArgs &a, int64_t operands, hipStream_t stream) {
  const size_t rows = (size_t)(kTiles * 16 * (kRank + 4) + kWaves * 16 * (64 + 4)) * sizeof(float), operand = operands ? (size_t)2 * kRank * 72 * sizeof(half_t) : 0;
  adapter_up_kernel<kRank, kTiles, kWide>
      <<<(unsigned)((int64_t)a.most_tiles * a.ranges + operands), kThreads, rows > operand ? rows : operand, stream>>>(a);
  return check_launch("adapter_up_kernel");
}

#define GQ_BY_SHAPE(START, ...)                                                                                 \
  (kRankClass == 32    ? (large ? (wide ? START<32, 4, true>(__VA_ARGS__) : START<32, 4, false>(__VA_ARGS__))    \
                                : (wide ? START<32, 1, true>(__VA_ARGS__) : START<32, 1, false>(__VA_ARGS__)))   \
   : kRankClass == 64  ? (large ? (wide ? START<64, 4, true>(__VA_ARGS__) : START<64, 4, false>(__VA_ARGS__))    \
                                : (wide ? START<64, 1, true>(__VA_ARGS__) : START<64, 1, false>(__VA_ARGS__)))   \
                       : (large ? (wide ? START<128, 4, true>(__VA_ARGS__) : START<128, 4, false>(__VA_ARGS__))  \
                                : (wide ? START<128, 1, true>(__VA_ARGS__) : START<128, 1, false>(__VA_ARGS__))))

bool aligned16(const void *p) { return (uintptr_t)p % 16 == 0; }

int launch_down(const Batch &b, const half_t *x, int64_t x_stride, const half_t *w, int64_t features, int64_t rank, float *v, float *most,
                int64_t splits, const TurnArgs *turn, hipStream_t stream) {
  DownArgs a = {};
  a.x = x, a.w = w, a.x_stride = x_stride, a.tiles = b.tiles(), a.tile_count = b.words + b.plan.counts + (b.large ? 1 : 0);
  a.order = b.words + b.plan.order, a.v = v, a.most = most, a.rows = b.plan.rows, a.features = features, a.rank = (int)rank;
  a.split = round_up((features + splits - 1) / splits, 128), a.most_tiles = (int)b.most_tiles(), a.splits = (int)splits;
  if (turn) a.turn = *turn;
  const int64_t turns = turn ? (int64_t)turn->pieces * turn->adapters * 2 : 0;
  const bool large = b.large, wide = aligned16(x) && aligned16(w) && x_stride % 8 == 0 && features % 8 == 0;
  const int kRankClass = rank_class(rank);
  return GQ_BY_SHAPE(start_down, a, turns, stream);
}

int launch_up(const Batch &b, const float *v, int64_t splits, const half_t *w, const float *scaling, const half_t *y, int64_t y_stride,
              half_t *out, int64_t out_stride, int64_t features, int64_t rank, int act, const OuterArgs *outer, hipStream_t stream) {
  UpArgs a = {};
  a.v = v, a.w = w, a.scaling = scaling, a.has_y = y != nullptr, a.out = out, a.out_stride = out_stride;
  a.y = y ? y : out, a.y_stride = y ? y_stride : out_stride;
  a.tiles = b.tiles(), a.tile_count = b.words + b.plan.counts + (b.large ? 1 : 0), a.order = b.words + b.plan.order;
  a.rows = b.plan.rows, a.features = features, a.rank = (int)rank, a.splits = (int)splits, a.act = act;
  a.skip_rows_without = y == out && y_stride == out_stride && act == GQ_ACT_NONE;
  const int64_t tiles = b.most_tiles(), most = (features + 255) / 256, want = up_ranges(tiles, rank, b.large), ranges = want < most ? want : most;
  a.range = round_up((features + ranges - 1) / ranges, 256);
  a.most_tiles = (int)tiles, a.ranges = (int)((features + a.range - 1) / a.range);
  if (outer) a.outer = *outer;
  const int64_t longest = b.plan.rows < kAdapterSegment ? b.plan.rows : kAdapterSegment;
  const int64_t operands = outer ? outer->most_segments * ((longest + 63) / 64) * 2 : 0;
  const bool large = b.large, wide = aligned16(y) && aligned16(out) && aligned16(w) && y_stride % 8 == 0 && out_stride % 8 == 0 &&
                                     features % 8 == 0 && rank % 8 == 0;
  const int kRankClass = rank_class(rank);
  return GQ_BY_SHAPE(start_up, a, operands, stream);
}

// Workgroups at most for one adapter's weights, where every adapter gets as many and only the device knows which have rows.
int64_t groups_of_adapter(int64_t adapters) { return adapters < 64 ? 512 : 32768 / adapters; }

template <int kRank>
int launch_outer(const OuterArgs &a, const PlanLayout &plan, bool wide, hipStream_t stream) {
  const int64_t features = a.side[0].features > a.side[1].features ? a.side[0].features : a.side[1].features;
  const dim3 grid((unsigned)plan.most_segments, (unsigned)((features + 127) / 128), 2 * (kRank > 64 ? 2 : 1));
  if (wide)
    adapter_outer_kernel<kRank, true><<<grid, kThreads, 0, stream>>>(a);
  else
    adapter_outer_kernel<kRank, false><<<grid, kThreads, 0, stream>>>(a);
  const int rc = check_launch("adapter_outer_kernel");
  if (rc != GQ_OK) return rc;
  const int64_t each = (a.rank * features + kThreads - 1) / kThreads, most = 2 * groups_of_adapter(a.adapters);
  adapter_sum_kernel<<<dim3((unsigned)(each < most ? each : most), (unsigned)a.adapters, 2), kThreads, 0, stream>>>(a);
  return check_launch("adapter_sum_kernel");
}

struct GradLayout {
  int64_t v, dv, most[2], turned[2], operand[2], back[2], parts[2], bytes;
  GradLayout(const PlanLayout &plan, int64_t most_tiles, int64_t in, int64_t out, int64_t rank, int64_t in_splits, int64_t out_splits) {
    const int64_t width = rank_class(rank);
    int64_t at = 0;
    const auto take = [&](int64_t n) {
      const int64_t here = at;
      at += round_up(n, 256);
      return here;
    };
    v = take(in_splits * plan.rows * width * 4), dv = take(out_splits * plan.rows * width * 4);
    for (int i = 0; i < 2; ++i) {
      most[i] = take((i ? out_splits : in_splits) * most_tiles * 4);
      turned[i] = take(plan.adapters * rank * (i ? out : in) * 2);
      operand[i] = take((plan.rows + 64 * (plan.most_segments + 1)) * 2 * width * 2), back[i] = take(plan.most_segments * 4);
      parts[i] = take(plan.most_parts * rank * (i ? out : in) * 4);
    }
    bytes = at;
  }
};

int64_t tiles_at_most(const PlanLayout &plan, int64_t rank) { return large_tiles(plan.rows, rank) ? plan.most_large : plan.most_small; }

}  // namespace

int64_t adapter_plan_bytes(int64_t rows, int64_t adapters) { return PlanLayout(rows, adapters).words * 4; }

int launch_adapter_plan(const int32_t *ids, int64_t rows, int64_t adapters, void *plan, hipStream_t stream) {
  const PlanLayout l(rows, adapters);
  const PlanArgs a = {ids, (int *)plan, l.counts, l.order, l.parts, l.small, l.large, l.segments, (int)rows, (int)adapters};
  const size_t lds = (size_t)kPlanWaves * (adapters + 1) * sizeof(int);
  constexpr size_t most = (size_t)kPlanWaves * (kMostAdapters + 1) * sizeof(int);
  if (const int rc = allow_lds<adapter_plan_kernel, most>(lds, "adapter_plan_kernel")) return rc;
  adapter_plan_kernel<<<1, kPlanThreads, lds, stream>>>(a);
  return check_launch("adapter_plan_kernel");
}

int64_t adapter_apply_workspace_bytes(int64_t rows, int64_t adapters, int64_t in, int64_t rank) {
  const PlanLayout plan(rows, adapters);
  return round_up(down_splits(tiles_at_most(plan, rank), in) * rows * rank_class(rank) * 4, 256);
}

int launch_adapter_apply(const gq_adapters &w, const void *plan, int64_t rows, const uint16_t *x, int64_t x_stride, const uint16_t *y,
                         int64_t y_stride, uint16_t *out, int64_t out_stride, int act, void *workspace, hipStream_t stream) {
  const Batch b = {PlanLayout(rows, w.n_adapters), (const int *)plan, large_tiles(rows, w.rank)};
  const int64_t splits = down_splits(b.most_tiles(), w.in_features);
  const int rc = launch_down(b, (const half_t *)x, x_stride, (const half_t *)w.down, w.in_features, w.rank, (float *)workspace, nullptr, splits, nullptr, stream);
  if (rc != GQ_OK) return rc;
  return launch_up(b, (const float *)workspace, splits, (const half_t *)w.up, w.scaling, (const half_t *)y, y_stride, (half_t *)out, out_stride,
                   w.out_features, w.rank, act, nullptr, stream);
}

int64_t adapter_grad_workspace_bytes(int64_t rows, int64_t adapters, int64_t in, int64_t out, int64_t rank) {
  const PlanLayout plan(rows, adapters);
  const int64_t tiles = tiles_at_most(plan, rank);
  return GradLayout(plan, tiles, in, out, rank, down_splits(tiles, in), down_splits(tiles, out)).bytes;
}

int launch_adapter_grad(const gq_adapters &w, const void *plan, int64_t rows, const uint16_t *x, int64_t x_stride, const uint16_t *dy,
                        int64_t dy_stride, const uint16_t *dx, int64_t dx_stride, uint16_t *dx_out, int64_t dx_out_stride, float *d_down,
                        float *d_up, void *workspace, hipStream_t stream) {
  const Batch b = {PlanLayout(rows, w.n_adapters), (const int *)plan, large_tiles(rows, w.rank)};
  const int64_t in = w.in_features, out = w.out_features, tiles = b.most_tiles();
  const int64_t in_splits = down_splits(tiles, in), out_splits = down_splits(tiles, out);
  const GradLayout l(b.plan, tiles, in, out, w.rank, in_splits, out_splits);
  char *ws = (char *)workspace;
  half_t *down_turned = (half_t *)(ws + l.turned[0]), *up_turned = (half_t *)(ws + l.turned[1]);
  const int64_t pieces = ((in > out ? in : out) + 63) / 64 * ((w.rank + 63) / 64);
  const int64_t most_pieces = groups_of_adapter(w.n_adapters);
  const TurnArgs turn = {{(const half_t *)w.down, (const half_t *)w.up}, {down_turned, up_turned}, {w.rank, out}, {in, w.rank},
                         b.words + b.plan.parts, (int)(pieces < most_pieces ? pieces : most_pieces), (int)w.n_adapters,
                         (w.rank | in | out) % 8 == 0 && aligned16(w.down) && aligned16(w.up)};
  int rc = launch_down(b, (const half_t *)x, x_stride, (const half_t *)w.down, in, w.rank, (float *)(ws + l.v), (float *)(ws + l.most[0]), in_splits,
                       &turn, stream);
  if (rc == GQ_OK)
    rc = launch_down(b, (const half_t *)dy, dy_stride, up_turned, out, w.rank, (float *)(ws + l.dv), (float *)(ws + l.most[1]), out_splits, nullptr,
                     stream);
  if (rc != GQ_OK) return rc;
  OuterArgs a;
  // dA: the rows of x with dv;  dB: the rows of dy with v
  for (int i = 0; i < 2; ++i) {
    OuterSide &s = a.side[i];
    s.x = (const half_t *)(i ? dy : x), s.x_stride = i ? dy_stride : x_stride, s.features = i ? out : in;
    s.v = (const float *)(ws + (i ? l.v : l.dv)), s.splits = (int)(i ? in_splits : out_splits);
    s.most = (const float *)(ws + l.most[i ? 0 : 1]);
    s.operand = (half_t *)(ws + l.operand[i]), s.back = (float *)(ws + l.back[i]), s.parts = (float *)(ws + l.parts[i]);
    s.grad = i ? d_up : d_down, s.turned = i == 1;
  }
  a.segments = (const AdapterTile *)(b.words + b.plan.segments), a.segment_count = b.words + b.plan.counts + 2;
  a.order = b.words + b.plan.order, a.parts_of = b.words + b.plan.parts, a.scaling = w.scaling;
  a.rows = rows, a.rank = (int)w.rank, a.adapters = (int)w.n_adapters, a.most_tiles = (int)tiles, a.most_segments = (int)b.plan.most_segments, a.large = b.large;
  rc = launch_up(b, (const float *)(ws + l.dv), out_splits, down_turned, w.scaling, (const half_t *)dx, dx_stride, (half_t *)dx_out, dx_out_stride,
                 in, w.rank, GQ_ACT_NONE, &a, stream);
  if (rc != GQ_OK) return rc;
  const bool wide = aligned16(x) && aligned16(dy) && (x_stride | dy_stride | in | out) % 8 == 0;
  return rank_class(w.rank) == 32   ? launch_outer<32>(a, b.plan, wide, stream)
         : rank_class(w.rank) == 64 ? launch_outer<64>(a, b.plan, wide, stream)
                                    : launch_outer<128>(a, b.plan, wide, stream);
}

}  // namespace gq

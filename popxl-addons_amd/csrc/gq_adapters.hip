// Low-rank adapters of many requests beside a shared projection:  y' = act(y + s_a (x A_a^T) B_a^T), each row its adapter a.
//   A [rank, in], B [out, rank] (the layouts that adapters are published in), s one binary32 number an adapter.
//
// adapter_plan_kernel  sorts a batch's rows by adapter once, for every projection that they pass: tiles of rows of ONE
//                      adapter, so that each product below is a plain matrix product over gathered rows.
// adapter_down_kernel  v = x A^T (contraction over the features): a split of the features per workgroup, binary32 parts.
// adapter_up_kernel    y' = act(y + s v B^T) (contraction over the rank).
//   The gradients are the same two products with the weights turned (`kTurned`: through LDS): dv = dy B, dx' = dx + s dv A, and
// adapter_outer_kernel dA = s dv^T x, dB = s dy^T v (contraction over rows; parts of 512 rows, added in order by
//                      adapter_sum_kernel; no atomics anywhere, so results do not depend on timing).
//
// v is held in 32 bits.  Where it enters a second product it is split into two binary16 numbers, v = hi + lo, after a power of
// two has brought the largest of its row (or segment) near 1: 22 bits of the largest, for twice the matrix instructions of a
// contraction over no more than 128.
//
// Bound by memory: x, y, y' and the adapters in use, each once; ranks of 8 ... 64 give 2 rank flops a byte of x.
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

// One workgroup.  Wave w takes the w-th stretch of rows: it counts them by kind (adapter, or none = the last kind), a scan over
// kinds and waves gives every (kind, wave) its place, and the wave puts its rows there in their order.
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
  // Parts are numbered like segments; an adapter of one segment leaves its number unused.  The numbers are compact enough:
  // only those of adapters with several segments are used, so they are counted apart.
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
    if (e >= each || kind >= kinds) continue;
    const int adapter = kind < a.adapters ? kind : -1, n = total[e], begin = before[0];
    for (int i = 0; i < n; i += kAdapterSmallTile)
      ((AdapterTile *)(a.plan + a.small))[before[1]++] = AdapterTile{adapter, begin + i, min(n - i, kAdapterSmallTile), -1};
    for (int i = 0; i < n; i += kAdapterLargeTile)
      ((AdapterTile *)(a.plan + a.large))[before[2]++] = AdapterTile{adapter, begin + i, min(n - i, kAdapterLargeTile), -1};
    if (adapter >= 0) {
      const int segments = (n + kAdapterSegment - 1) / kAdapterSegment;
      a.plan[a.parts + 2 * kind] = part, a.plan[a.parts + 2 * kind + 1] = segments;
      for (int i = 0; i < n; i += kAdapterSegment)
        ((AdapterTile *)(a.plan + a.segments))[before[3]++] =
            AdapterTile{adapter, begin + i, min(n - i, kAdapterSegment), segments > 1 ? part + i / kAdapterSegment : -1};
      if (segments > 1) part += segments;
    }
    int at = begin;
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

// 8 values from p, of which `valid` exist (the rest are zeros); kWide: all or none of them, 16-byte aligned
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

// Orders a wave's own LDS stores and loads (it does not share the piece with other waves, so no barrier).
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_wave_barrier();
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

__device__ __forceinline__ uint32_t pair_of(half_t a, half_t b) {
  return (uint32_t)__builtin_bit_cast(uint16_t, a) | (uint32_t)__builtin_bit_cast(uint16_t, b) << 16;
}

struct DownArgs {
  const half_t *x, *w;  // w: [adapters][rank][features], turned: [adapters][features][rank]
  int64_t x_stride;
  const AdapterTile *tiles;
  const int *tile_count, *order;
  float *v;  // [splits][rows][kRank]
  int64_t rows, features, split;  // features of one split, a multiple of 512
  int rank;
};

constexpr int kStep = 128;           // features that a wave takes at a time
constexpr int kTurnedRow = kStep + 8;  // binary16 a row of a turned piece in LDS: 16-byte rows, 4 banks apart

// kRank: rank rounded up to 32, 64 or 128; kTiles x 16 rows.  Wave w of a workgroup takes features 128 w + 512 i ... of the
// workgroup's split; the four binary32 sums meet in LDS.  v^T = A x^T: a lane ends with 4 consecutive ranks of one row.
template <int kRank, int kTiles, bool kWide, bool kTurned>
__global__ __launch_bounds__(kThreads) void adapter_down_kernel(DownArgs a) {
  constexpr int kRankTiles = kRank / 16;
  extern __shared__ float shared[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
  if ((int)blockIdx.x >= *a.tile_count) return;
  const AdapterTile tile = a.tiles[blockIdx.x];
  if (tile.adapter < 0) return;
  const int64_t from = blockIdx.y * a.split, to = min(a.features, from + a.split);
  const half_t *w = a.w + (int64_t)tile.adapter * a.rank * a.features;
  const half_t *x[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) x[t] = a.x + (int64_t)a.order[tile.begin + min(t * 16 + m, tile.count - 1)] * a.x_stride;
  half_t *turned = (half_t *)shared + wave * kRank * kTurnedRow;

  float4_t acc[kRankTiles][kTiles];
#pragma unroll
  for (int r = 0; r < kRankTiles; ++r)
#pragma unroll
    for (int t = 0; t < kTiles; ++t) acc[r][t] = float4_t{};
  for (int64_t k0 = from + wave * kStep; k0 < to; k0 += kWaves * kStep) {
    if (kTurned) {
      // this wave's piece [128 features][rank] to [rank][features]: two features' 8 ranks at a time, 4-byte stores
      const int columns = (a.rank + 7) / 8;
      for (int n = lane; n < kStep / 2 * columns; n += 64) {
        const int c = n % columns, f = n / columns * 2;
        const half_t *p = w + (k0 + f) * a.rank + c * 8;
        const int64_t left = a.rank - c * 8;
        const half8_t u0 = load8<kWide>(p, k0 + f < to ? left : 0), u1 = load8<kWide>(p + a.rank, k0 + f + 1 < to ? left : 0);
#pragma unroll
        for (int j = 0; j < 8; ++j) *(uint32_t *)(turned + (c * 8 + j) * kTurnedRow + f) = pair_of(u0[j], u1[j]);
      }
      wave_lds_fence();
    }
#pragma unroll
    for (int s = 0; s < kStep / 32; ++s) {
      const int64_t k = k0 + s * 32 + g * 8;
      half8_t xf[kTiles];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) xf[t] = load8<kWide>(x[t] + k, to - k);
#pragma unroll
      for (int r = 0; r < kRankTiles; ++r) {
        if (r * 16 >= a.rank) continue;
        half8_t wf;
        if (kTurned)
          wf = *(const half8_t *)(turned + min(r * 16 + m, (a.rank + 7) / 8 * 8 - 1) * kTurnedRow + s * 32 + g * 8);
        else
          wf = load8<kWide>(w + (int64_t)min(r * 16 + m, a.rank - 1) * a.features + k, to - k);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf, xf[t], acc[r][t], 0, 0, 0);
      }
    }
    if (kTurned) wave_lds_fence();
  }
  // sum of the four waves, 64 rows at most: [waves][16 rows][kRank + 4]
  float *v = a.v + ((int64_t)blockIdx.y * a.rows + tile.begin) * kRank;
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRankTiles; ++r) *(float4_t *)(shared + (wave * 16 + m) * (kRank + 4) + r * 16 + 4 * g) = acc[r][t];
    __syncthreads();
    for (int n = threadIdx.x; n < 16 * kRank; n += kThreads) {
      const int row = n / kRank, r = n % kRank;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) sum += shared[(i * 16 + row) * (kRank + 4) + r];
      if (t * 16 + row < tile.count) v[(int64_t)(t * 16 + row) * kRank + r] = r < a.rank ? sum : 0.f;
    }
  }
}

struct UpArgs {
  const float *v;  // [splits][rows][kRank]
  const half_t *w;  // [adapters][features][rank], turned: [adapters][rank][features]
  const float *scaling;
  const half_t *y;  // NULL: zeros
  half_t *out;
  int64_t y_stride, out_stride;
  const AdapterTile *tiles;
  const int *tile_count, *order;
  int64_t rows, features, range;  // features of one workgroup, a multiple of 256
  int rank, splits, act;
  bool skip_rows_without;  // out is y and there is no activation: rows without an adapter are done
};

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

// Wave w takes 64 features at a time: row 4 g' + i of operand tile t is feature 16 g' + 4 t + i, so that a lane ends with 16
// consecutive features of one row (two 16-byte loads and stores, 128 bytes a row for the wave).
template <int kRank, int kTiles, bool kWide, bool kTurned>
__global__ __launch_bounds__(kThreads) void adapter_up_kernel(UpArgs a) {
  constexpr int kChunks = kRank / 32, kRow = kRank + 8;
  extern __shared__ float shared[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
  if ((int)blockIdx.x >= *a.tile_count) return;
  const AdapterTile tile = a.tiles[blockIdx.x];
  const bool with = tile.adapter >= 0;
  if (!with && a.skip_rows_without) return;
  const half_t *w = a.w + (int64_t)max(tile.adapter, 0) * a.rank * a.features;
  const float scaling = with ? a.scaling[tile.adapter] : 0.f;

  half8_t hi[kTiles][kChunks], lo[kTiles][kChunks];
  float back[kTiles];
  int64_t row[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const int i = min(t * 16 + m, tile.count - 1);
    row[t] = a.order[tile.begin + i];
    back[t] = 0.f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) hi[t][c] = lo[t][c] = half8_t{};
    if (!with) continue;
    float v[kChunks][8], most = 0.f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] = 0.f;
    for (int s = 0; s < a.splits; ++s) {
      const float *from = a.v + ((int64_t)s * a.rows + tile.begin + i) * kRank;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const float4_t u0 = *(const float4_t *)(from + c * 32 + g * 8), u1 = *(const float4_t *)(from + c * 32 + g * 8 + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[c][j] += u0[j], v[c][4 + j] += u1[j];
      }
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(v[c][j]));
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    const float power = normal_power(most, back[t]);
    back[t] *= scaling;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        half_t h, l;
        split_of(v[c][j] * power, h, l);
        hi[t][c][j] = h, lo[t][c][j] = l;
      }
  }

  half_t *turned = (half_t *)shared + wave * 64 * kRow;
  const int64_t from = blockIdx.y * a.range, to = min(a.features, from + a.range);
  for (int64_t n0 = from + wave * 64; n0 < to; n0 += kWaves * 64) {
    float4_t acc[kTiles][4];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int f = 0; f < 4; ++f) acc[t][f] = float4_t{};
    if (with) {
      if (kTurned) {
        // [rank][64 features] to [features][rank], two ranks at a time; ranks behind the last are zeros
        for (int n = lane; n < kRank / 2 * 8; n += 64) {
          const int c = n % 8, r = n / 8 * 2;
          const half_t *p = w + r * a.features + n0 + c * 8;
          const int64_t left = to - n0 - c * 8;
          const half8_t u0 = load8<kWide>(p, r < a.rank ? left : 0), u1 = load8<kWide>(p + a.features, r + 1 < a.rank ? left : 0);
#pragma unroll
          for (int j = 0; j < 8; ++j) *(uint32_t *)(turned + (c * 8 + j) * kRow + r) = pair_of(u0[j], u1[j]);
        }
        wave_lds_fence();
      }
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int feature = 16 * (m >> 2) + 4 * f + (m & 3);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          if (c * 32 >= a.rank) continue;
          half8_t wf;
          if (kTurned) {
            wf = *(const half8_t *)(turned + feature * kRow + c * 32 + g * 8);
          } else {
            const int64_t n = min(n0 + feature, a.features - 1);
            wf = load8<kWide>(w + n * a.rank + c * 32 + g * 8, a.rank - (c * 32 + g * 8));
          }
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            acc[t][f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf, hi[t][c], acc[t][f], 0, 0, 0);
            acc[t][f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf, lo[t][c], acc[t][f], 0, 0, 0);
          }
        }
      }
      if (kTurned) wave_lds_fence();
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      if (t * 16 + m >= tile.count) continue;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int64_t n = n0 + 16 * g + 8 * half;
        if (n >= to) continue;
        half8_t y = {};
        if (a.y) y = load8<kWide>(a.y + row[t] * a.y_stride + n, to - n);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          // (tile f, row 4 g + i of the accumulators is feature 16 g + 4 f + i)
          const float sum = (float)y[j] + acc[t][2 * half + j / 4][j % 4] * back[t];
          y[j] = (half_t)apply_activation(sum, a.act);
        }
        half_t *o = a.out + row[t] * a.out_stride + n;
        if (kWide) {
          *(half8_t *)o = y;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (n + j < to) o[j] = y[j];
        }
      }
    }
  }
}

struct OuterSide {
  const half_t *x;  // [rows][features]
  int64_t x_stride, features;
  const float *v;  // [splits][rows][kRank]
  int splits;
  half_t *operand;  // [segments][hi, lo][kRank][512]
  float *back;      // [segments]
  float *grad;      // [adapters][rank][features], turned: [adapters][features][rank]
  float *parts;     // [parts][rank][features]
  bool turned;
};

struct OuterArgs {
  OuterSide side[2];
  const AdapterTile *segments;
  const int *segment_count, *order, *parts_of;
  const float *scaling;
  int64_t rows;
  int rank, adapters;
};

// v of a segment as the other product's operand: summed over the splits, scaled by a power of two, split, transposed
template <int kRank>
__global__ __launch_bounds__(kThreads) void adapter_operand_kernel(OuterArgs a) {
  __shared__ float wave_most[kWaves];
  const OuterSide &side = a.side[blockIdx.y];
  if ((int)blockIdx.x >= *a.segment_count) return;
  const AdapterTile seg = a.segments[blockIdx.x];
  const int tid = threadIdx.x;
  half_t *hi = side.operand + (int64_t)blockIdx.x * 2 * kRank * kAdapterSegment, *lo = hi + kRank * kAdapterSegment;
  const auto value = [&](int i, int r) {
    float sum = 0.f;
    for (int s = 0; s < side.splits; ++s) sum += side.v[((int64_t)s * a.rows + seg.begin + i) * kRank + r];
    return sum;
  };
  float most = 0.f;
  for (int n = tid; n < seg.count * kRank; n += kThreads) most = fmaxf(most, fabsf(value(n / kRank, n % kRank)));
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
  if ((tid & 63) == 0) wave_most[tid >> 6] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) most = fmaxf(most, wave_most[w]);
  float back;
  const float power = normal_power(most, back);
  if (tid == 0) side.back[blockIdx.x] = back * a.scaling[seg.adapter];
  for (int n = tid; n < kAdapterSegment * kRank; n += kThreads) {
    const int i = n / kRank, r = n % kRank;
    half_t h = (half_t)0.f, l = (half_t)0.f;
    if (i < seg.count) split_of(value(i, r) * power, h, l);
    hi[r * kAdapterSegment + i] = h, lo[r * kAdapterSegment + i] = l;
  }
}

// 128 features of one segment's product; the four waves take every fourth 32 rows and meet in LDS.  The rows are loaded as
// they lie (8 features a lane, 8 rows) and paired in registers: operand c has feature 8 m + c, so that a lane ends with 8
// consecutive features of 4 ranks.
template <int kRank, bool kWide>
__global__ __launch_bounds__(kThreads) void adapter_outer_kernel(OuterArgs a) {
  constexpr int kRankTiles = kRank / 16 < 4 ? kRank / 16 : 4;  // 64 ranks at most at a time: blockIdx.z
  __shared__ float shared[16 * (128 + 4) * kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
  const bool second = blockIdx.z & 1;
  const int rank0 = (blockIdx.z >> 1) * 64;
  const OuterSide &side = second ? a.side[1] : a.side[0];
  if ((int)blockIdx.x >= *a.segment_count || (int64_t)blockIdx.y * 128 >= side.features) return;
  const AdapterTile seg = a.segments[blockIdx.x];
  const half_t *hi = side.operand + (int64_t)blockIdx.x * 2 * kRank * kAdapterSegment, *lo = hi + kRank * kAdapterSegment;
  const int64_t f = (int64_t)blockIdx.y * 128 + m * 8;

  float4_t acc[kRankTiles][8];
#pragma unroll
  for (int r = 0; r < kRankTiles; ++r)
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[r][c] = float4_t{};
  for (int i0 = wave * 32; i0 < seg.count; i0 += kWaves * 32) {
    half8_t x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + g * 8 + j;
      x[j] = half8_t{};
      if (i < seg.count) x[j] = load8<kWide>(side.x + (int64_t)a.order[seg.begin + i] * side.x_stride + f, side.features - f);
    }
    half8_t xf[8];
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) xf[c][j] = x[j][c];
#pragma unroll
    for (int r = 0; r < kRankTiles; ++r) {
      if (rank0 + r * 16 >= a.rank) continue;
      const int64_t at = (int64_t)(rank0 + r * 16 + m) * kAdapterSegment + i0 + g * 8;
      const half8_t h = *(const half8_t *)(hi + at), l = *(const half8_t *)(lo + at);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, xf[c], acc[r][c], 0, 0, 0);
        acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l, xf[c], acc[r][c], 0, 0, 0);
      }
    }
  }
  const float back = side.back[blockIdx.x];
  const bool direct = seg.part < 0;
  float *out = direct ? side.grad + (int64_t)seg.adapter * a.rank * side.features : side.parts + (int64_t)seg.part * a.rank * side.features;
#pragma unroll
  for (int r = 0; r < kRankTiles; ++r) {
    if (rank0 + r * 16 >= a.rank) continue;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 8; ++c) shared[(wave * 16 + 4 * g + i) * 132 + m * 8 + c] = acc[r][c][i];
    __syncthreads();
    for (int n = threadIdx.x; n < 16 * 128; n += kThreads) {
      // (a gradient [features][rank] is written rank by rank)
      const int rr = direct && side.turned ? n % 16 : n / 128, ff = direct && side.turned ? n / 16 : n % 128;
      const int rank = rank0 + r * 16 + rr;
      const int64_t feature = (int64_t)blockIdx.y * 128 + ff;
      if (rank >= a.rank || feature >= side.features) continue;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) sum += shared[(w * 16 + rr) * 132 + ff];
      out[direct && side.turned ? feature * a.rank + rank : rank * side.features + feature] = sum * back;
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
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < size; n += (int64_t)gridDim.x * kThreads) {
    const int64_t at = side.turned ? n % a.rank * side.features + n / a.rank : n;
    float sum = 0.f;
    for (int s = 0; s < segments; ++s) sum += side.parts[(first + s) * size + at];
    grad[n] = sum;
  }
}

// ----------------------------------------------------------------------------------------------------------- launches

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int rank_class(int64_t rank) { return rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

// Workgroups that fill the device twice over where the features allow it, each with at least 512 features (128 a wave)
int64_t down_splits(int64_t tiles, int64_t features) {
  const int64_t most = (features + kWaves * kStep - 1) / (kWaves * kStep), want = (512 + tiles - 1) / tiles;
  return want < most ? want : most > 0 ? most : 1;
}

// Rows of a tile: 16 for decode batches, whose rows mostly have adapters of their own; 64 where an adapter's weights are worth
// reading once for more rows.
bool large_tiles(int64_t rows) { return rows >= 1024; }

struct Batch {
  const PlanLayout plan;
  const int *words;
  bool large;
  const AdapterTile *tiles() const { return (const AdapterTile *)(words + (large ? plan.large : plan.small)); }
  int64_t most_tiles() const { return large ? plan.most_large : plan.most_small; }
};

// A kernel has to be told of more than 64 KiB of LDS, on each device.
int allow_lds(const void *kernel, size_t bytes, const char *who) {
  if (bytes <= 64 << 10) return GQ_OK;
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  return e == hipSuccess ? GQ_OK : fail((int)e, "%s: %s", who, hipGetErrorString(e));
}

template <int kRank, int kTiles, bool kWide, bool kTurned>
int start_down(const DownArgs &a, int64_t tiles, int64_t splits, hipStream_t stream) {
  const size_t sums = (size_t)kWaves * 16 * (kRank + 4) * sizeof(float);
  const size_t turned = kTurned ? (size_t)kWaves * kRank * kTurnedRow * sizeof(half_t) : 0;
  const size_t lds = sums > turned ? sums : turned;
  if (int rc = allow_lds((const void *)adapter_down_kernel<kRank, kTiles, kWide, kTurned>, lds, "adapter_down_kernel")) return rc;
  adapter_down_kernel<kRank, kTiles, kWide, kTurned><<<dim3((unsigned)tiles, (unsigned)splits), kThreads, lds, stream>>>(a);
  return check_launch("adapter_down_kernel");
}

template <int kRank, int kTiles, bool kWide, bool kTurned>
int start_up(const UpArgs &a, int64_t tiles, int64_t ranges, hipStream_t stream) {
  const size_t lds = kTurned ? (size_t)kWaves * 64 * (kRank + 8) * sizeof(half_t) : 0;
  if (int rc = allow_lds((const void *)adapter_up_kernel<kRank, kTiles, kWide, kTurned>, lds, "adapter_up_kernel")) return rc;
  adapter_up_kernel<kRank, kTiles, kWide, kTurned><<<dim3((unsigned)tiles, (unsigned)ranges), kThreads, lds, stream>>>(a);
  return check_launch("adapter_up_kernel");
}

#define GQ_BY_SHAPE(START, TURNED, ...)                                                                                   \
  (kRankClass == 32    ? (large ? (wide ? START<32, 4, true, TURNED>(__VA_ARGS__) : START<32, 4, false, TURNED>(__VA_ARGS__))    \
                                : (wide ? START<32, 1, true, TURNED>(__VA_ARGS__) : START<32, 1, false, TURNED>(__VA_ARGS__)))   \
   : kRankClass == 64  ? (large ? (wide ? START<64, 4, true, TURNED>(__VA_ARGS__) : START<64, 4, false, TURNED>(__VA_ARGS__))    \
                                : (wide ? START<64, 1, true, TURNED>(__VA_ARGS__) : START<64, 1, false, TURNED>(__VA_ARGS__)))   \
                       : (large ? (wide ? START<128, 4, true, TURNED>(__VA_ARGS__) : START<128, 4, false, TURNED>(__VA_ARGS__))  \
                                : (wide ? START<128, 1, true, TURNED>(__VA_ARGS__) : START<128, 1, false, TURNED>(__VA_ARGS__))))

bool aligned16(const void *p) { return (uintptr_t)p % 16 == 0; }

int launch_down(const Batch &b, const half_t *x, int64_t x_stride, const half_t *w, bool turned, int64_t features, int64_t rank,
                float *v, int64_t splits, hipStream_t stream) {
  DownArgs a;
  a.x = x, a.w = w, a.x_stride = x_stride, a.tiles = b.tiles(), a.tile_count = b.words + b.plan.counts + (b.large ? 1 : 0);
  a.order = b.words + b.plan.order, a.v = v, a.rows = b.plan.rows, a.features = features, a.rank = (int)rank;
  a.split = round_up((features + splits - 1) / splits, kWaves * kStep);
  const bool large = b.large, wide = aligned16(x) && aligned16(w) && x_stride % 8 == 0 && features % 8 == 0 && (!turned || rank % 8 == 0);
  const int kRankClass = rank_class(rank);
  return turned ? GQ_BY_SHAPE(start_down, true, a, b.most_tiles(), splits, stream)
                : GQ_BY_SHAPE(start_down, false, a, b.most_tiles(), splits, stream);
}

int launch_up(const Batch &b, const float *v, int64_t splits, const half_t *w, bool turned, const float *scaling, const half_t *y,
              int64_t y_stride, half_t *out, int64_t out_stride, int64_t features, int64_t rank, int act, hipStream_t stream) {
  UpArgs a;
  a.v = v, a.w = w, a.scaling = scaling, a.y = y, a.out = out, a.y_stride = y_stride, a.out_stride = out_stride;
  a.tiles = b.tiles(), a.tile_count = b.words + b.plan.counts + (b.large ? 1 : 0), a.order = b.words + b.plan.order;
  a.rows = b.plan.rows, a.features = features, a.rank = (int)rank, a.splits = (int)splits, a.act = act;
  a.skip_rows_without = y == out && y_stride == out_stride && act == GQ_ACT_NONE;
  const int64_t tiles = b.most_tiles(), most = (features + 255) / 256, want = (1024 + tiles - 1) / tiles;
  a.range = round_up((features + (want < most ? want : most) - 1) / (want < most ? want : most), 256);
  const int64_t ranges = (features + a.range - 1) / a.range;
  const bool large = b.large;
  const bool wide = aligned16(y) && aligned16(out) && aligned16(w) && y_stride % 8 == 0 && out_stride % 8 == 0 && features % 8 == 0 &&
                    (turned || rank % 8 == 0);
  const int kRankClass = rank_class(rank);
  return turned ? GQ_BY_SHAPE(start_up, true, a, tiles, ranges, stream) : GQ_BY_SHAPE(start_up, false, a, tiles, ranges, stream);
}

template <int kRank>
int launch_outer(const OuterArgs &a, const PlanLayout &plan, bool wide, hipStream_t stream) {
  const int64_t features = a.side[0].features > a.side[1].features ? a.side[0].features : a.side[1].features;
  adapter_operand_kernel<kRank><<<dim3((unsigned)plan.most_segments, 2), kThreads, 0, stream>>>(a);
  int rc = check_launch("adapter_operand_kernel");
  if (rc != GQ_OK) return rc;
  const dim3 grid((unsigned)plan.most_segments, (unsigned)((features + 127) / 128), 2 * (kRank > 64 ? 2 : 1));
  if (wide)
    adapter_outer_kernel<kRank, true><<<grid, kThreads, 0, stream>>>(a);
  else
    adapter_outer_kernel<kRank, false><<<grid, kThreads, 0, stream>>>(a);
  rc = check_launch("adapter_outer_kernel");
  if (rc != GQ_OK) return rc;
  const int64_t each = (a.rank * features + kThreads - 1) / kThreads;
  adapter_sum_kernel<<<dim3((unsigned)(each < 512 ? each : 512), (unsigned)a.adapters, 2), kThreads, 0, stream>>>(a);
  return check_launch("adapter_sum_kernel");
}

struct GradLayout {
  int64_t v, dv, operand[2], back[2], parts[2], bytes;
  GradLayout(const PlanLayout &plan, int64_t in, int64_t out, int64_t rank, int64_t in_splits, int64_t out_splits) {
    const int64_t width = rank_class(rank);
    int64_t at = 0;
    const auto take = [&](int64_t n) {
      const int64_t here = at;
      at += round_up(n, 256);
      return here;
    };
    v = take(in_splits * plan.rows * width * 4), dv = take(out_splits * plan.rows * width * 4);
    for (int i = 0; i < 2; ++i) {
      operand[i] = take(plan.most_segments * 2 * width * kAdapterSegment * 2), back[i] = take(plan.most_segments * 4);
      parts[i] = take(plan.most_parts * rank * (i ? out : in) * 4);
    }
    bytes = at;
  }
};

int64_t tiles_at_most(const PlanLayout &plan) { return large_tiles(plan.rows) ? plan.most_large : plan.most_small; }

}  // namespace

int64_t adapter_plan_bytes(int64_t rows, int64_t adapters) { return PlanLayout(rows, adapters).words * 4; }

int launch_adapter_plan(const int32_t *ids, int64_t rows, int64_t adapters, void *plan, hipStream_t stream) {
  const PlanLayout l(rows, adapters);
  const PlanArgs a = {ids, (int *)plan, l.counts, l.order, l.parts, l.small, l.large, l.segments, (int)rows, (int)adapters};
  const size_t lds = (size_t)kPlanWaves * (adapters + 1) * sizeof(int);
  if (int rc = allow_lds((const void *)adapter_plan_kernel, lds, "adapter_plan_kernel")) return rc;
  adapter_plan_kernel<<<1, kPlanThreads, lds, stream>>>(a);
  return check_launch("adapter_plan_kernel");
}

int64_t adapter_apply_workspace_bytes(int64_t rows, int64_t adapters, int64_t in, int64_t rank) {
  const PlanLayout plan(rows, adapters);
  return round_up(down_splits(tiles_at_most(plan), in) * rows * rank_class(rank) * 4, 256);
}

int launch_adapter_apply(const gq_adapters &w, const void *plan, int64_t rows, const uint16_t *x, int64_t x_stride, const uint16_t *y,
                         int64_t y_stride, uint16_t *out, int64_t out_stride, int act, void *workspace, hipStream_t stream) {
  const Batch b = {PlanLayout(rows, w.n_adapters), (const int *)plan, large_tiles(rows)};
  const int64_t splits = down_splits(b.most_tiles(), w.in_features);
  const int rc = launch_down(b, (const half_t *)x, x_stride, (const half_t *)w.down, false, w.in_features, w.rank, (float *)workspace, splits, stream);
  if (rc != GQ_OK) return rc;
  return launch_up(b, (const float *)workspace, splits, (const half_t *)w.up, false, w.scaling, (const half_t *)y, y_stride, (half_t *)out,
                   out_stride, w.out_features, w.rank, act, stream);
}

int64_t adapter_grad_workspace_bytes(int64_t rows, int64_t adapters, int64_t in, int64_t out, int64_t rank) {
  const PlanLayout plan(rows, adapters);
  return GradLayout(plan, in, out, rank, down_splits(tiles_at_most(plan), in), down_splits(tiles_at_most(plan), out)).bytes;
}

int launch_adapter_grad(const gq_adapters &w, const void *plan, int64_t rows, const uint16_t *x, int64_t x_stride, const uint16_t *dy,
                        int64_t dy_stride, const uint16_t *dx, int64_t dx_stride, uint16_t *dx_out, int64_t dx_out_stride, float *d_down,
                        float *d_up, void *workspace, hipStream_t stream) {
  const Batch b = {PlanLayout(rows, w.n_adapters), (const int *)plan, large_tiles(rows)};
  const int64_t in_splits = down_splits(b.most_tiles(), w.in_features), out_splits = down_splits(b.most_tiles(), w.out_features);
  const GradLayout l(b.plan, w.in_features, w.out_features, w.rank, in_splits, out_splits);
  char *ws = (char *)workspace;
  int rc = launch_down(b, (const half_t *)x, x_stride, (const half_t *)w.down, false, w.in_features, w.rank, (float *)(ws + l.v), in_splits, stream);
  if (rc == GQ_OK)
    rc = launch_down(b, (const half_t *)dy, dy_stride, (const half_t *)w.up, true, w.out_features, w.rank, (float *)(ws + l.dv), out_splits, stream);
  if (rc == GQ_OK)
    rc = launch_up(b, (const float *)(ws + l.dv), out_splits, (const half_t *)w.down, true, w.scaling, (const half_t *)dx, dx_stride,
                   (half_t *)dx_out, dx_out_stride, w.in_features, w.rank, GQ_ACT_NONE, stream);
  if (rc != GQ_OK) return rc;
  OuterArgs a;
  // dA: the rows of x with dv;  dB: the rows of dy with v
  for (int i = 0; i < 2; ++i) {
    OuterSide &s = a.side[i];
    s.x = (const half_t *)(i ? dy : x), s.x_stride = i ? dy_stride : x_stride, s.features = i ? w.out_features : w.in_features;
    s.v = (const float *)(ws + (i ? l.v : l.dv)), s.splits = (int)(i ? in_splits : out_splits);
    s.operand = (half_t *)(ws + l.operand[i]), s.back = (float *)(ws + l.back[i]), s.parts = (float *)(ws + l.parts[i]);
    s.grad = i ? d_up : d_down, s.turned = i == 1;
  }
  a.segments = (const AdapterTile *)(b.words + b.plan.segments), a.segment_count = b.words + b.plan.counts + 2;
  a.order = b.words + b.plan.order, a.parts_of = b.words + b.plan.parts, a.scaling = w.scaling;
  a.rows = rows, a.rank = w.rank, a.adapters = (int)w.n_adapters;
  const bool wide = aligned16(x) && aligned16(dy) && (x_stride | dy_stride | w.in_features | w.out_features) % 8 == 0;
  return rank_class(w.rank) == 32   ? launch_outer<32>(a, b.plan, wide, stream)
         : rank_class(w.rank) == 64 ? launch_outer<64>(a, b.plan, wide, stream)
                                    : launch_outer<128>(a, b.plan, wide, stream);
}

}  // namespace gq

// Append to and read back from the 8-bit key/value cache (layout: gq_kv.h).
//
// Quantisation.  A block that starts with these tokens takes scale = amax / 127.  A block that has tokens keeps its scale s
// where amax / 127 <= s; otherwise s grows by the least power of two that covers the new tokens and the codes that are there
// are scaled down by it (rint).  Growth by powers of two bounds what repeated rounding can add up to: a code is rounded by at
// most 1/2 of its own step, then by 1/2 of each later step, and the steps at least double: |value - x| < s (1/2 + 1/4 + ...)
// < s.  (With s following amax / 127 itself, every token that sets a new maximum would add another half step.)
// Codes are rint(x / s) with the correctly rounded quotient: a plain binary32 program gets the same codes.
//
// Bound by HBM: 2 bytes read and 1 written an element.  A workgroup owns one (block, head) of the keys or of the values: the
// scale is a maximum over all of it, and no other workgroup writes there.  Its 256 threads hold the new tokens in registers
// as pieces of 4 tokens x 8 dims: 16-byte loads that are contiguous over the row, 8-byte stores of key codes, and for the
// transposed value codes a 4-byte word of 4 tokens for each dim, which goes through LDS to 16-byte stores.
#include "gq_kv.h"
#include "gq_rotary.h"

namespace gq {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;
constexpr int kPieces = 16 * (kMaxDim / 8) / kThreads;  // pieces of 4 tokens x 8 dims a thread holds at most

struct AppendArgs {
  KvCache cache;
  KvBatch batch;
  const half_t *x[2];  // keys, values
  int64_t token[2], head[2];
  const double *turns;  // NULL: keys are stored as they come
  float factor;
  int rotary_dim;
  bool half_layout;
};

// Where a workgroup's (sequence, block) lies: rows [row, row + count) go to slots [slot, slot + count) of block `id`.
struct Place {
  int row, slot, count, position, id;
};

__device__ __forceinline__ bool find_place(const KvCache &cache, const KvBatch &batch, uint32_t unit, Place &p) {
  int b;
  uint32_t base;
  KvSequence s;
  const auto units = [&](const KvSequence &s) {
    const int from = max(s.first, 0);
    return (uint32_t)(s.length > from ? (s.length - 1) / kBlock - from / kBlock + 1 : 0);
  };
  if (!kv_locate(batch, unit, units, b, s, base)) return false;
  const int from = max(s.first, 0), block = from / kBlock + (int)(unit - base);
  p.position = max(from, block * kBlock);
  p.slot = p.position - block * kBlock;
  p.count = min(s.length, (block + 1) * kBlock) - p.position;
  p.row = s.begin + (p.position - s.first);
  p.id = batch.table[(int64_t)b * batch.width + block];
  return p.id >= 0 && p.id < cache.n_blocks;
}

__device__ __forceinline__ uint32_t quantise(half_t x, float scale) {
  if (!(scale > 0.f)) return 128;  // a block of zeros
  const float q = rintf((float)x / scale);
  return (uint32_t)(int)(fminf(fmaxf(q, -127.f), 127.f) + 128.f);  // (fmaxf maps a NaN, of an infinite block, to -127)
}

__global__ __launch_bounds__(kThreads) void kv_append_kernel(AppendArgs a) {
  __shared__ uint32_t words[kMaxDim * 16];  // value codes transposed: [dim][token quad], columns of 8 dims swizzled
  __shared__ uint32_t wave_max[kThreads / 64];
  const int tid = threadIdx.x, h = blockIdx.y;
  const bool values = blockIdx.z != 0;
  Place p;
  if (!find_place(a.cache, a.batch, blockIdx.x, p)) return;
  const int dim = a.cache.dim, columns = dim / 8;
  const int64_t place = (int64_t)p.id * a.cache.heads + h;
  const half_t *x = (values ? a.x[1] : a.x[0]) + h * (values ? a.head[1] : a.head[0]);
  const int64_t stride = values ? a.token[1] : a.token[0];
  const int rotary_dim = values || !a.turns ? 0 : a.rotary_dim;

  // the pieces: token quad q (slots 4q ... 4q+3), column c (dims 8c ... 8c+7); the largest magnitude as bits, where NaN > inf
  half8_t piece[kPieces][4];
  uint32_t most = 0;
#pragma unroll
  for (int n = 0; n < kPieces; ++n) {
    const int q = (tid + n * kThreads) / columns, c = (tid + n * kThreads) % columns;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int token = 4 * q + i - p.slot;
      half8_t v = {};
      if (q < 16 && token >= 0 && token < p.count) {
        const half_t *row = x + (p.row + token) * stride;
        v = *(const half8_t *)(row + c * 8);
        if (c * 8 < rotary_dim) {
          const int position = p.position + token;
          if (a.half_layout) {
            const int pairs = rotary_dim / 2, at = c * 8 < pairs ? c * 8 : c * 8 - pairs;
            const half8_t other = *(const half8_t *)(row + (c * 8 < pairs ? c * 8 + pairs : at));
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 cs = rotary_turn(position, a.turns[at + j], a.factor, false);
              half_t lo, hi;
              if (c * 8 < pairs)
                rotary_pair((float)v[j], (float)other[j], cs, lo, hi);
              else
                rotary_pair((float)other[j], (float)v[j], cs, lo, hi);
              v[j] = c * 8 < pairs ? lo : hi;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 cs = rotary_turn(position, a.turns[c * 4 + j], a.factor, false);
              half_t lo, hi;
              rotary_pair((float)v[2 * j], (float)v[2 * j + 1], cs, lo, hi);
              v[2 * j] = lo, v[2 * j + 1] = hi;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, (uint32_t)(__builtin_bit_cast(uint16_t, (half_t)v[j]) & 0x7fff));
      }
      piece[n][i] = v;
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, d));
  if ((tid & 63) == 0) wave_max[tid >> 6] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) most = max(most, wave_max[w]);
  const float need = (float)__builtin_bit_cast(half_t, (uint16_t)most) / 127.f;  // infinite or NaN where an input is

  float *scale_at = (values ? a.cache.v_scale : a.cache.k_scale) + place;
  const float old = p.slot > 0 ? *scale_at : 0.f;
  float scale = old, shrink = 1.f;
  if (!(need <= old) && old == old) {  // (a scale that is NaN stays)
    scale = need;
    if (old > 0.f && need < __builtin_inff()) {
      int e;
      if (frexpf(need / old, &e) == 0.5f) --e;
      scale = ldexpf(old, e);
      shrink = ldexpf(1.f, -e);
    }
  }
  // (every thread has read the old scale before one replaces it)
  __syncthreads();
  if (tid == 0 && (scale != old || p.slot == 0)) *scale_at = scale;

  uint8_t *codes = (values ? a.cache.v_codes : a.cache.k_codes) + place * kBlock * dim;
  if (shrink != 1.f) {  // tokens that were there: slots [0, slot)
    if (!values) {
      for (int n = tid; n < p.slot * dim / 4; n += kThreads) {
        uint32_t w = ((uint32_t *)codes)[n], r = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) r |= (uint32_t)(int)(rintf((float)((int)(w >> 8 * j & 255) - 128) * shrink) + 128.f) << 8 * j;
        ((uint32_t *)codes)[n] = r;
      }
    } else {
      for (int n = tid; n < dim * 16; n += kThreads) {
        const int t0 = n % 16 * 4;
        if (t0 >= p.slot) continue;
        uint32_t w = ((uint32_t *)codes)[n], r = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t byte = w >> 8 * j & 255;
          r |= (t0 + j < p.slot ? (uint32_t)(int)(rintf((float)((int)byte - 128) * shrink) + 128.f) : byte) << 8 * j;
        }
        ((uint32_t *)codes)[n] = r;
      }
      __syncthreads();  // (a word may hold bytes of new tokens too, stored below)
    }
  }

  const int end = p.slot + p.count;
  const bool few = p.count < 8;  // value codes of few tokens are stored byte by byte, each row of 64 tokens apart
#pragma unroll
  for (int n = 0; n < kPieces; ++n) {
    const int q = (tid + n * kThreads) / columns, c = (tid + n * kThreads) % columns;
    if (q >= 16 || 4 * q + 3 < p.slot || 4 * q >= end) continue;
    if (!values) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int slot = 4 * q + i;
        if (slot < p.slot || slot >= end) continue;
        uint2_t w = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j / 4] |= quantise(piece[n][i][j], scale) << 8 * (j % 4);
        *(uint2_t *)(codes + slot * dim + c * 8) = w;
      }
    } else if (few) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int slot = 4 * q + i;
        if (slot < p.slot || slot >= end) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j) codes[(c * 8 + j) * kBlock + slot] = (uint8_t)quantise(piece[n][i][j], scale);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= quantise(piece[n][i][j], scale) << 8 * i;
        words[(c * 8 + j) * 16 + (q ^ (c & 15))] = w;
      }
    }
  }
  if (values && !few) {
    __syncthreads();
    for (int n = tid; n < dim * 4; n += kThreads) {
      const int d = n / 4, q0 = n % 4 * 4, t0 = q0 * 4;
      if (t0 + 15 < p.slot || t0 >= end) continue;
      uint4_t w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = words[d * 16 + ((q0 + j) ^ (d / 8 & 15))];
      uint8_t *to = codes + d * kBlock + t0;
      if (t0 >= p.slot && t0 + 16 <= end) {
        *(uint4_t *)to = w;
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (t0 + j >= p.slot && t0 + j < end) to[j] = (uint8_t)(w[j / 4] >> 8 * (j % 4));
      }
    }
  }
}

struct GatherArgs {
  KvCache cache;
  KvBatch batch;
  half_t *out[2];
};

// The values of a batch's new tokens as binary16, [tokens][heads][dim]: one rounding of code * scale.
__global__ __launch_bounds__(kThreads) void kv_gather_kernel(GatherArgs a) {
  const int tid = threadIdx.x, h = blockIdx.y;
  const bool values = blockIdx.z != 0;
  Place p;
  if (!find_place(a.cache, a.batch, blockIdx.x, p)) return;
  const int dim = a.cache.dim, columns = dim / 8;
  const int64_t place = (int64_t)p.id * a.cache.heads + h;
  const float scale = (values ? a.cache.v_scale : a.cache.k_scale)[place];
  const uint8_t *codes = (values ? a.cache.v_codes : a.cache.k_codes) + place * kBlock * dim;
  half_t *out = (values ? a.out[1] : a.out[0]) + h * dim;
  const int64_t stride = (int64_t)a.cache.heads * dim;
  const int end = p.slot + p.count;
  for (int n = tid; n < 16 * columns; n += kThreads) {
    const int q = values ? n % 16 : n / columns, c = values ? n / 16 : n % columns;
    if (4 * q + 3 < p.slot || 4 * q >= end) continue;
    uint32_t byte[4][2];  // [token][8 dims]
    if (!values) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint2_t w = *(const uint2_t *)(codes + (4 * q + i) * dim + c * 8);
        byte[i][0] = w[0], byte[i][1] = w[1];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) byte[i][0] = byte[i][1] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w = *(const uint32_t *)(codes + (c * 8 + j) * kBlock + 4 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) byte[i][j / 4] |= (w >> 8 * i & 255) << 8 * (j % 4);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int slot = 4 * q + i;
      if (slot < p.slot || slot >= end) continue;
      half8_t v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (half_t)((float)((int)(byte[i][j / 4] >> 8 * (j % 4) & 255) - 128) * scale);
      *(half8_t *)(out + (p.row + slot - p.slot) * stride + c * 8) = v;
    }
  }
}

// (sequence, block) pairs at most: a sequence of n new tokens reaches into (n + 62) / 64 + 1 blocks
unsigned most_places(const KvBatch &b) { return (unsigned)(b.tokens / kBlock + 2 * b.sequences); }

}  // namespace

int launch_kv_append(const KvCache &cache, const KvBatch &batch, const uint16_t *k, int64_t k_token, int64_t k_head,
                     const uint16_t *v, int64_t v_token, int64_t v_head, const gq_rotary *rotary, hipStream_t stream) {
  AppendArgs a = {};
  a.cache = cache, a.batch = batch;
  a.x[0] = (const half_t *)k, a.token[0] = k_token, a.head[0] = k_head;
  a.x[1] = (const half_t *)v, a.token[1] = v_token, a.head[1] = v_head;
  if (rotary) {
    a.turns = rotary->turns, a.factor = rotary->factor, a.rotary_dim = rotary->rotary_dim;
    a.half_layout = rotary->layout == GQ_ROTARY_HALF;
  }
  kv_append_kernel<<<dim3(most_places(batch), cache.heads, 2), kThreads, 0, stream>>>(a);
  return check_launch("kv_append_kernel");
}

int launch_kv_gather(const KvCache &cache, const KvBatch &batch, uint16_t *k, uint16_t *v, hipStream_t stream) {
  GatherArgs a = {cache, batch, {(half_t *)k, (half_t *)v}};
  kv_gather_kernel<<<dim3(most_places(batch), cache.heads, 2), kThreads, 0, stream>>>(a);
  return check_launch("kv_gather_kernel");
}

}  // namespace gq

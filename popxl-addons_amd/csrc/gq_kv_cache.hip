// Append to and read back from the 8-bit key/value cache (layout: gq_kv.h).
//
// Quantisation.  A block that starts with these tokens takes scale = amax / 127.  A block that has tokens keeps its scale s
// where amax / 127 <= s; otherwise s grows by the least power of two that covers the new tokens and the codes that are there
// are scaled down by it (rint), or, under a scale of 0, cleared.  Growth by powers of two bounds what repeated rounding can add up to: a code is rounded by at
// most 1/2 of its own step, then by 1/2 of each later step, and the steps at least double: |value - x| < s (1/2 + 1/4 + ...)
// < s.  (With s following amax / 127 itself, every token that sets a new maximum would add another half step.)
// Codes are rint(x / s) with the correctly rounded quotient: a plain binary32 program gets the same codes.
//
// Bound by HBM: 2 bytes read and 1 written an element.  A workgroup owns a (block, head) of the keys or of the values: the
// scale is a maximum over all of it, and no other workgroup writes there.  The new tokens come by 16-byte loads that are
// contiguous over a row and wait in LDS, as binary16, for the scale; from there key codes go out 8 dims at a time, and value
// codes, which the cache holds transposed, 16 tokens of a dim at a time.  Keys that are turned on the way: the angles of the
// block's tokens are formed once in LDS.  (With the tokens held in registers instead the kernel had 160 of them and 23 KiB of
// code, and a decode step waited for its instructions: 19 us for 48 requests.)  Measured, 8 heads of 128, keys turned, 16383
// tokens: 25 us for the keys, 16 us for the values (2.5 and 4 TB/s; the angles and codes are what the keys wait for); a token
// for each of 48 requests, 16 heads of 256: 11 us, most of it a chain of dependent loads (offsets, table, scale, tokens, the old
// codes where the scale grows).
#include "gq_kv.h"
#include "gq_rotary.h"

namespace gq {
namespace {

constexpr int kThreads = 256;
constexpr int kFewOfBlock = 4;  // new tokens of a sequence, on average, up to which a workgroup is one wave
// New tokens of a block up to which their value codes are stored byte by byte.  With 2 in its place up to 4 tokens of 48 sequences
// take 22 to 27 us, not 11 to 14; with 8 up to 16 tokens of 48 sequences 27, not 25, up to 8 of 8 sequences 11, not 10.
constexpr int kFew = 16;

struct AppendArgs {
  KvCache cache;
  KvBatch batch;
  const half_t *x[2];  // keys, values
  int64_t token[2], head[2];
  const double *turns;  // NULL: keys are stored as they come
  float factor;
  int rotary_dim;
  int first;  // blockIdx.y + first: 0 keys, 1 values
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

typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));

// What turns values into codes at one scale: rint of the correctly rounded binary32 quotient.  The product with the reciprocal
// is within 3 2^-24 |q| <= 2.3e-5 of that quotient, so it rounds to the same integer unless it is nearer than that to a tie;
// then (of normal binary16 values one wave's 512 in 11 to 14, exact ties among them) the quotients are taken in binary64.  That is exact: the product with the binary64
// reciprocal is within 2^-52 of x / s, relatively, and a quotient of an 11-bit and a 24-bit number is never half way between
// two binary32 numbers (25 bits) nor nearer to that than 2^-49, so rounding the product rounds the quotient.
struct Coder {
  float scale, inverse;
  // (the least scale of a value is 2^-24 / 127; a smaller one, from elsewhere, has only zeros to code, and may have no reciprocal)
  __device__ explicit Coder(float s) : scale(s), inverse(s > 1e-30f && s < __builtin_inff() ? 1.f / s : 0.f) {}
  __device__ uint2_t operator()(half8_t x) const {
    uint2_t word = {0x80808080u, 0x80808080u};
    if (inverse == 0.f) return word;  // a block of zeros, or one that is not finite (its scale says so)
    float q[8], off = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = (float)x[i] * inverse;
      q[i] = rintf(t);
      off = fmaxf(off, fabsf(t - q[i]));
    }
    if (off > 0.49997f) {
      const double exact = 1. / (double)scale;
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = rintf((float)((double)x[i] * exact));
    }
    word = uint2_t{0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) word[i / 4] = __builtin_amdgcn_cvt_pk_u8_f32(q[i] + 128.f, i % 4, word[i / 4]);
    return word;
  }
};

__device__ __forceinline__ uint32_t scaled_down(uint32_t word, float by) {
  uint32_t r = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) r = __builtin_amdgcn_cvt_pk_u8_f32(rintf((float)((int)(word >> 8 * j & 255) - 128) * by) + 128.f, j, r);
  return r;
}

__device__ __forceinline__ uint32_t magnitudes(half8_t v, uint32_t most) {
  const uint4_t bits = __builtin_bit_cast(uint4_t, v) & 0x7fff7fffu;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t two = bits[j], had = most;  // (a bit cast of the vector's element itself takes element 0)
    most = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2_t, two), __builtin_bit_cast(ushort2_t, had)));
  }
  return most;
}

// kSize threads: one wave where blocks get few tokens, four otherwise
template <int kSize>
__global__ __launch_bounds__(kSize) void kv_append_kernel(AppendArgs a) {
  constexpr int kAhead = 4;
  extern __shared__ uint4_t append_shared[];  // rows: binary16 [token][dim]; turn: cosine and sine [token][pair]
  __shared__ uint32_t wave_max[kSize / 64];
  const int tid = threadIdx.x;
  const bool values = blockIdx.y + a.first != 0;
  // (heads run fastest: the workgroups under way together then cover whole rows of the tokens, not one head's stretch of each)
  const int dim = a.cache.dim, columns = dim / 8, heads = a.cache.heads, h = blockIdx.x % heads;
  Place p;
  if (!find_place(a.cache, a.batch, blockIdx.x / heads, p)) return;
  const int rotary_dim = values || !a.turns ? 0 : a.rotary_dim, pairs = rotary_dim / 2;
  const int64_t stride = values ? a.token[1] : a.token[0], place = (int64_t)p.id * heads + h;
  const half_t *x = (values ? a.x[1] : a.x[0]) + p.row * stride + h * (values ? a.head[1] : a.head[0]);
  half_t *rows = (half_t *)append_shared;
  float2 *turn = (float2 *)(rows + p.count * dim);
  const int twos = a.half_layout ? pairs / 8 : 0, per_token = columns - twos;  // (half layout: units of two pieces)
  const int end = p.slot + p.count, units = p.count * per_token;
  // n / columns = n * per_column >> 16 for n < 2048 and columns <= 32, likewise for units
  const uint32_t per_column = (65536 + columns - 1) / columns, per_unit = (65536 + per_token - 1) / per_token;
  // a unit's pairs lie apart, pair j of unit u at j * stretch + u: neighbouring threads read neighbouring angles
  const int per = a.half_layout ? 8 : 4, stretch = pairs / per;
  if (pairs > 0) {  // (a thread keeps its pair, where it would wait for another one's turns with every angle)
    const int together = max(kSize / pairs, 1);
    for (int i = tid % pairs; i < pairs; i += kSize) {
      const double turns = a.turns[i];
      const int at = i % per * stretch + i / per;
      for (int token = tid / pairs; token < p.count && tid < together * pairs; token += together)
        turn[token * pairs + at] = rotary_turn(p.position + token, turns, a.factor, false);
    }
  }

  float *scale_at = (values ? a.cache.v_scale : a.cache.k_scale) + place;
  const float old = p.slot > 0 ? *scale_at : 0.f;
  if (rotary_dim > 0) __syncthreads();  // (the angles are there)
  uint32_t most = 0;  // the largest magnitudes, as two 16-bit patterns: NaN above infinity above all numbers
  const auto put = [&](int token, int d, half8_t w) {
    most = magnitudes(w, most);
    *(half8_t *)(rows + token * dim + d) = w;
  };
  for (int n0 = tid; n0 < units; n0 += kAhead * kSize) {
    half8_t v[kAhead], other[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      // a unit is 8 dims, or, among the first of a token, 8 dims and those they are turned with (the last unit again behind it)
      const int n = min(n0 + i * kSize, units - 1), token = n * per_unit >> 16, u = n - token * per_token;
      v[i] = *(const half8_t *)(x + token * stride + (u < twos ? u : u + twos) * 8);
      if (twos > 0) other[i] = *(const half8_t *)(x + token * stride + (u < twos ? pairs + u * 8 : 0));
    }
#pragma unroll 1
    for (int i = 0; i < kAhead; ++i) {
      const int n = n0 + i * kSize, token = n * per_unit >> 16, u = n - token * per_token;
      if (n >= units) break;
      half8_t w = v[0];
      if (u < twos) {
        half8_t w2;
        const float2 *cs = turn + token * pairs + u;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          half_t lo, hi;
          rotary_pair((float)w[j], (float)other[0][j], cs[j * stretch], lo, hi);
          w[j] = lo, w2[j] = hi;
        }
        put(token, pairs + u * 8, w2);
      } else if (twos == 0 && u * 8 < rotary_dim) {
        const float2 *cs = turn + token * pairs + u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          half_t lo, hi;
          rotary_pair((float)w[2 * j], (float)w[2 * j + 1], cs[j * stretch], lo, hi);
          w[2 * j] = lo, w[2 * j + 1] = hi;
        }
      }
      put(token, (u < twos ? u : u + twos) * 8, w);
#pragma unroll
      for (int k = 0; k + 1 < kAhead; ++k) v[k] = v[k + 1], other[k] = other[k + 1];  // (one copy of this code for the four)
    }
  }
  most = max(most & 0xffff, most >> 16);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, d));
  if ((tid & 63) == 0) wave_max[tid >> 6] = most;
  __syncthreads();  // (every thread has read the old scale, too)
#pragma unroll
  for (int w = 0; w < kSize / 64; ++w) most = max(most, wave_max[w]);
  const float need = (float)__builtin_bit_cast(half_t, (uint16_t)most) / 127.f;  // infinite or NaN where an input is
  float scale = old, shrink = 1.f;
  if (!(need <= old) && old == old) {  // (a scale that is NaN stays)
    scale = need;
    if (old > 0.f && need < __builtin_inff()) {
      // (by mantissas and exponents: the quotient of a scale of 1e-40, which a cache made elsewhere may have, is infinite)
      int e_need, e_old;
      const float m_need = frexpf(need, &e_need), m_old = frexpf(old, &e_old);
      const int e = e_need - e_old + (m_need > m_old ? 1 : 0);
      scale = ldexpf(old, e);
      shrink = ldexpf(1.f, -e);
    } else if (old == 0.f && p.slot > 0) {
      shrink = 0.f;  // tokens under a scale of 0 are zeros whatever their codes (a cache made elsewhere), and stay it
    }
  }
  if (tid == 0 && (scale != old || p.slot == 0)) *scale_at = scale;

  uint8_t *codes = (values ? a.cache.v_codes : a.cache.k_codes) + place * kBlock * dim;
  if (shrink != 1.f) {  // tokens that were there: slots [0, slot)
    for (int n = tid; n < (values ? dim * 16 : p.slot * dim / 4); n += kSize) {
      const int t0 = values ? n % 16 * 4 : 0;
      if (values && t0 >= p.slot) continue;
      const uint32_t w = ((uint32_t *)codes)[n], keep = values && t0 + 4 > p.slot ? 0xffffffffu << 8 * (p.slot - t0) : 0u;
      ((uint32_t *)codes)[n] = (scaled_down(w, shrink) & ~keep) | (w & keep);
    }
    if (values) __syncthreads();  // (a word may hold bytes of new tokens too, stored below)
  }

  const Coder code(scale);
  if (!values || p.count < kFew) {
#pragma unroll 2
    for (int n = tid; n < p.count * columns; n += kSize) {
      const int token = n * per_column >> 16, c = n - token * columns;
      const half8_t v = *(const half8_t *)(rows + token * dim + c * 8);
      const uint2_t w = code(v);
      if (!values) {
        *(uint2_t *)(codes + (p.slot + token) * dim + c * 8) = w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) codes[(c * 8 + j) * kBlock + p.slot + token] = (uint8_t)(w[j / 4] >> 8 * (j % 4));
      }
    }
  } else {
    for (int n = tid; n < dim * 2; n += kSize) {  // two dims, 16 slots
      const int d = n / 4 * 2, t0 = n % 4 * 16;  // (a row's 64 bytes by four lanes)
      if (t0 + 15 < p.slot || t0 >= end) continue;
      const half_t *column = rows + (t0 - p.slot) * dim + d;
      uint4_t w[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {  // 8 slots
        half8_t v[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const half2_t two = *(const half2_t *)(column + (min(max(t0 + 8 * q + i, p.slot), end - 1) - t0) * dim);
          v[0][i] = two[0], v[1][i] = two[1];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint2_t eight = code(v[i]);
          w[i][2 * q] = eight[0], w[i][2 * q + 1] = eight[1];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint8_t *to = codes + (d + i) * kBlock + t0;
        if (t0 >= p.slot && t0 + 16 <= end) {
          *(uint4_t *)to = w[i];
        } else {
          for (int j = max(p.slot - t0, 0); j < min(end - t0, 16); ++j) {
            const uint32_t word = j < 4 ? w[i][0] : j < 8 ? w[i][1] : j < 12 ? w[i][2] : w[i][3];
            to[j] = (uint8_t)(word >> 8 * (j & 3));
          }
        }
      }
    }
  }
}

struct GatherArgs {
  KvCache cache;
  KvBatch batch;
  half_t *out[2];
};

// The values of a batch's new tokens as binary16, [tokens][heads][dim]: one rounding of code * scale.  A thread takes 4 tokens x 8
// dims, so that values, which lie the other way round in the cache, are turned in registers.  Bound by memory: 1 byte read, 2
// written an element; 16383 tokens, 8 heads of 128: 15.5 us, 6.5 TB/s (the codes are still in a cache behind the append).
__global__ __launch_bounds__(kThreads) void kv_gather_kernel(GatherArgs a) {
  const int tid = threadIdx.x, h = blockIdx.x % a.cache.heads;
  const bool values = blockIdx.y != 0;
  Place p;
  if (!find_place(a.cache, a.batch, blockIdx.x / a.cache.heads, p)) return;
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

// A block's tokens of 256 dims and the angles of 128 pairs.
constexpr size_t kMostLds = kBlock * (256 * sizeof(half_t) + 128 * sizeof(float2));

// (sequence, block) pairs at most: a sequence of n new tokens reaches into (n + 62) / 64 + 1 blocks
int64_t most_places(const KvBatch &b) { return b.tokens / kBlock + 2 * (int64_t)b.sequences; }

// 2^24 rows and 2^20 sequences of 1024 heads would be more workgroups than a grid has
bool too_many(const KvCache &cache, const KvBatch &batch) { return most_places(batch) * cache.heads > 0x7fffffff / kThreads; }

}  // namespace

int launch_kv_append(const KvCache &cache, const KvBatch &batch, const uint16_t *k, int64_t k_token, int64_t k_head,
                     const uint16_t *v, int64_t v_token, int64_t v_head, const gq_rotary *rotary, hipStream_t stream) {
  if (too_many(cache, batch)) return fail(GQ_ERR_UNSUPPORTED, "gq_kv_append_f16: too many rows, sequences and heads for one launch");
  AppendArgs a = {};
  a.cache = cache, a.batch = batch;
  a.x[0] = (const half_t *)k, a.token[0] = k_token, a.head[0] = k_head;
  a.x[1] = (const half_t *)v, a.token[1] = v_token, a.head[1] = v_head;
  if (rotary) {
    a.turns = rotary->turns, a.factor = rotary->factor, a.rotary_dim = rotary->rotary_dim;
    a.half_layout = rotary->layout == GQ_ROTARY_HALF;
  }
  const int64_t places = most_places(batch);
  const int rows = batch.tokens < kBlock ? batch.tokens : kBlock;
  const size_t codes = (size_t)rows * cache.dim * sizeof(half_t), angles = rotary ? (size_t)rows * rotary->rotary_dim / 2 * sizeof(float2) : 0;
  // Blocks of few tokens: one wave each (48 sequences of 1, about 2, about 4 tokens, 16 heads of 256: 11, 15, 27 us, with four waves
  // 14, 17, 21; 8 sequences of 1, about 8 tokens, 8 heads of 128: 5.5 and 11, with four waves 10 and 12).
  if (batch.tokens < kFewOfBlock * batch.sequences) {
    if (const int rc = allow_lds<kv_append_kernel<64>, kMostLds>(codes + angles, "kv_append_kernel")) return rc;
    kv_append_kernel<64><<<dim3((unsigned)(places * cache.heads), 2), 64, codes + angles, stream>>>(a);
  } else {
    // Keys and values apart: the angles take as much LDS as the rows or twice that, which only the keys' workgroups need.
    // (Sharing the angles between four heads of a workgroup took 47 us where this takes 43, for 16383 tokens, 8 heads of 128, and
    // 45 where this takes 28, for 48 sequences of about 8 tokens, 16 heads of 256.)
    if (const int rc = allow_lds<kv_append_kernel<kThreads>, kMostLds>(codes + angles, "kv_append_kernel")) return rc;
    kv_append_kernel<kThreads><<<(unsigned)(places * cache.heads), kThreads, codes + angles, stream>>>(a);
    a.first = 1;
    kv_append_kernel<kThreads><<<(unsigned)(places * cache.heads), kThreads, codes, stream>>>(a);
  }
  return check_launch("kv_append_kernel");
}

int launch_kv_gather(const KvCache &cache, const KvBatch &batch, uint16_t *k, uint16_t *v, hipStream_t stream) {
  if (too_many(cache, batch)) return fail(GQ_ERR_UNSUPPORTED, "gq_kv_gather_f16: too many rows, sequences and heads for one launch");
  GatherArgs a = {cache, batch, {(half_t *)k, (half_t *)v}};
  kv_gather_kernel<<<dim3((unsigned)(most_places(batch) * cache.heads), 2), kThreads, 0, stream>>>(a);
  return check_launch("kv_gather_kernel");
}

}  // namespace gq

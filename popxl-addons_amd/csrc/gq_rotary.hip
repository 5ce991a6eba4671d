// Rotary positions (GQ_ROTARY_* layouts) on a strided [tokens, heads, head_dim] tensor.
//
//   interleaved: pair i is (t[2i], t[2i+1]);  half: pair i is (t[i], t[i + r/2]);  i < r/2, r = rotary_dim <= head_dim
//   out = (a c - b s, a s + b c) with (c, s) = factor * (cos, sin)(2 pi p turns[i]), dims behind r copied.
//
// Bound by HBM: 4 bytes an element and little arithmetic.  A workgroup takes one token and some of its heads: the r/2
// angles are formed once in LDS and serve all of these heads.  Measured: 16381 tokens x 40 heads of 128, half layout, the
// gradient: 62.6 us, 5.4 TB/s (a plain copy of 1 GiB moves 5.1); 4 tokens x 32 heads of 256: 3.1 us, a launch with one chain of
// loads.
#include "gq_rotary.h"

namespace gq {
namespace {

constexpr int kThreads = 256;

struct RotaryArgs {
  const half_t *t;
  int64_t t_token, t_head;
  const int *positions;
  const double *turns;
  half_t *out;
  int64_t o_token, o_head;
  int heads, head_dim, rotary_dim, heads_per_group;
  float factor;
  bool half_layout, inverse;
};

// VEC: every row is 16-byte aligned and the pairs of an 8-element piece lie in it (interleaved, r % 8 == 0) or in one
// other piece (half, r % 16 == 0).  A thread keeps its piece of the row and walks over heads.  (16381 tokens x 40 heads of 128:
// 61 us; one element to the side, element by element, 144 us.)
template <bool VEC>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  __shared__ float2 turn[128];  // rotary_dim <= 256
  const int token = blockIdx.x, tid = threadIdx.x, pairs = a.rotary_dim / 2;
  const int h0 = blockIdx.y * a.heads_per_group, h1 = min(a.heads, h0 + a.heads_per_group);
  if (tid < pairs) turn[tid] = rotary_turn(a.positions[token], a.turns[tid], a.factor, a.inverse);
  __syncthreads();
  const half_t *row = a.t + token * a.t_token;
  half_t *dst = a.out + token * a.o_token;
  const bool in_place = row == dst;
  if (VEC) {
    // pieces of a row: those that a thread turns (half: with the piece r/2 behind), then those that are copied
    const int turned = a.half_layout ? pairs / 8 : a.rotary_dim / 8;
    const int copied = in_place ? 0 : (a.head_dim - a.rotary_dim) / 8;
    const int pieces = turned + copied, step = kThreads / pieces;
    const int piece = tid % pieces;
    if (tid >= step * pieces) return;
    for (int h = h0 + tid / pieces; h < h1; h += step) {
      const half_t *src = row + h * a.t_head;
      half_t *to = dst + h * a.o_head;
      if (piece >= turned) {
        const int d = a.rotary_dim + (piece - turned) * 8;
        *(half8_t *)(to + d) = *(const half8_t *)(src + d);
      } else if (a.half_layout) {
        const half8_t x = *(const half8_t *)(src + piece * 8), y = *(const half8_t *)(src + pairs + piece * 8);
        half8_t rx, ry;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          half_t p, q;
          rotary_pair((float)x[i], (float)y[i], turn[piece * 8 + i], p, q);
          rx[i] = p, ry[i] = q;
        }
        *(half8_t *)(to + piece * 8) = rx;
        *(half8_t *)(to + pairs + piece * 8) = ry;
      } else {
        const half8_t x = *(const half8_t *)(src + piece * 8);
        half8_t rx;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          half_t p, q;
          rotary_pair((float)x[2 * i], (float)x[2 * i + 1], turn[piece * 4 + i], p, q);
          rx[2 * i] = p, rx[2 * i + 1] = q;
        }
        *(half8_t *)(to + piece * 8) = rx;
      }
    }
  } else {
    const int units = pairs + (in_place ? 0 : a.head_dim - a.rotary_dim);
    for (int64_t n = tid; n < (int64_t)(h1 - h0) * units; n += kThreads) {
      const int h = h0 + (int)(n / units), u = (int)(n % units);
      const half_t *src = row + h * a.t_head;
      half_t *to = dst + h * a.o_head;
      if (u >= pairs) {
        to[a.rotary_dim + u - pairs] = src[a.rotary_dim + u - pairs];
        continue;
      }
      const int x = a.half_layout ? u : 2 * u, y = a.half_layout ? u + pairs : 2 * u + 1;
      half_t p, q;
      rotary_pair((float)src[x], (float)src[y], turn[u], p, q);
      to[x] = p, to[y] = q;
    }
  }
}

}  // namespace

int launch_rotary(const uint16_t *t, int64_t t_token, int64_t t_head, const int32_t *positions, const gq_rotary &rotary,
                  bool inverse, uint16_t *out, int64_t o_token, int64_t o_head, int64_t tokens, int64_t heads,
                  int64_t head_dim, hipStream_t stream) {
  RotaryArgs a;
  a.t = (const half_t *)t, a.t_token = t_token, a.t_head = t_head;
  a.positions = positions, a.turns = rotary.turns, a.factor = rotary.factor;
  a.out = (half_t *)out, a.o_token = o_token, a.o_head = o_head;
  a.heads = (int)heads, a.head_dim = (int)head_dim, a.rotary_dim = rotary.rotary_dim;
  a.half_layout = rotary.layout == GQ_ROTARY_HALF, a.inverse = inverse;
  const bool vec = (((uintptr_t)t | (uintptr_t)out) % 16 == 0) && (t_token | t_head | o_token | o_head | head_dim) % 8 == 0 &&
                   rotary.rotary_dim % (a.half_layout ? 16 : 8) == 0;
  // heads of a token are spread over workgroups until the device has two for each compute unit
  const int pieces = (int)head_dim / 8 > 0 ? (int)head_dim / 8 : 1;
  const int least = pieces >= kThreads ? 1 : kThreads / pieces;
  int64_t groups = (512 + tokens - 1) / tokens;
  const int64_t most = (heads + least - 1) / least;
  groups = groups < most ? groups : most;
  a.heads_per_group = (int)((heads + groups - 1) / groups);
  const unsigned across = (unsigned)((heads + a.heads_per_group - 1) / a.heads_per_group);
  constexpr int64_t kMostTokens = 1 << 23;  // of a launch: a grid has fewer than 2^32 threads along an axis
  for (int64_t first = 0; first < tokens; first += kMostTokens) {
    const dim3 grid((unsigned)(tokens - first < kMostTokens ? tokens - first : kMostTokens), across);
    if (vec)
      rotary_kernel<true><<<grid, kThreads, 0, stream>>>(a);
    else
      rotary_kernel<false><<<grid, kThreads, 0, stream>>>(a);
    if (const int rc = check_launch("rotary_kernel")) return rc;
    a.t += kMostTokens * t_token, a.out += kMostTokens * o_token, a.positions += kMostTokens;
  }
  return GQ_OK;
}

}  // namespace gq

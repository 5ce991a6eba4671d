// The rotation of rotary positions, shared by gq_rotary.hip and the cache's append (gq_kv_cache.hip).
#pragma once
#include "gq_common.h"

namespace gq {

// cos and sin of the angle of pair `turns` (turns a position) at `position`, times the factor.  The angle is formed in
// binary64 and reduced to an eighth of a turn about a multiple of a quarter there: at position 10^6 a binary32 angle would be
// off by 0.06 rad.  What is left, x in [-pi/4, pi/4], goes into the series of sine and cosine to x^9 and x^8, whose next terms
// are below 2^-25.  About 30 instructions, where the general function (whose own reduction has nothing left to do) is 80.
__device__ __forceinline__ float2 rotary_turn(int position, double turns, float factor, bool inverse) {
  double a = (double)position * turns;
  a -= rint(a);
  const double quarter = rint(4. * a);
  const float x = (float)((a - 0.25 * quarter) * 6.283185307179586), z = x * x;
  float s = __builtin_fmaf(z, 1.f / 362880.f, -1.f / 5040.f);
  s = __builtin_fmaf(z, s, 1.f / 120.f);
  s = __builtin_fmaf(z, s, -1.f / 6.f);
  s = __builtin_fmaf(z * x, s, x);
  float c = __builtin_fmaf(z, 1.f / 40320.f, -1.f / 720.f);
  c = __builtin_fmaf(z, c, 1.f / 24.f);
  c = __builtin_fmaf(z, c, -0.5f);
  c = __builtin_fmaf(z, c, 1.f);
  const int q = (int)quarter;  // -2 ... 2: cosine and sine change places every quarter, their signs every other
  const float cosine = q & 1 ? s : c, sine = q & 1 ? c : s;
  const bool minus_cosine = ((q + 1) & 2) != 0, minus_sine = ((q & 2) != 0) != inverse;
  return make_float2(minus_cosine ? -cosine * factor : cosine * factor, minus_sine ? -sine * factor : sine * factor);
}

// The same two operations wherever a pair is turned, so that the separate call and the append agree bit for bit.
__device__ __forceinline__ void rotary_pair(float a, float b, float2 cs, half_t &ra, half_t &rb) {
  ra = (half_t)(a * cs.x - b * cs.y);
  rb = (half_t)(a * cs.y + b * cs.x);
}

}  // namespace gq

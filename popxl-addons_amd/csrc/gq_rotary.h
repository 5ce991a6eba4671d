// The rotation of rotary positions, shared by gq_rotary.hip and the cache's append (gq_kv_cache.hip).
#pragma once
#include "gq_common.h"

namespace gq {

// cos and sin of the angle of pair `turns` (turns a position) at `position`, times the factor.  The angle is formed in
// binary64 and reduced to [-1/2, 1/2] turns there: at position 10^6 a binary32 angle would be off by 0.06 rad.  What is
// left fits binary32, where sincospif is good to about one unit in the last place.
__device__ __forceinline__ float2 rotary_turn(int position, double turns, float factor, bool inverse) {
  double a = (double)position * turns;
  a -= rint(a);
  float s, c;
  sincospif(2.f * (float)a, &s, &c);
  return make_float2(c * factor, (inverse ? -s : s) * factor);
}

// The same two operations wherever a pair is turned, so that the separate call and the append agree bit for bit.
__device__ __forceinline__ void rotary_pair(float a, float b, float2 cs, half_t &ra, half_t &rb) {
  ra = (half_t)(a * cs.x - b * cs.y);
  rb = (half_t)(a * cs.y + b * cs.x);
}

}  // namespace gq

// Rotary positions: the arguments that kernels take and the angles.
#pragma once

#include "dsa_common.h"

namespace dsa {

constexpr int RP_MAX_R = 256;  // frequencies
constexpr int RP_MAX_AXES = 4;

// What the angles are made of: frequency i turns by p[axis(i)] inv_freq[i], p the token's position on that axis.
struct RopeAngles {
  const int* positions;   // [axes][T]; null: a position that the kernel knows
  const float* inv_freq;  // [R]
  int R;
  int axes;
  float factor;           // of the rotated values
  float turn;             // 1, or -1 for the inverse rotation
  uint32_t axis[RP_MAX_R / 16];  // 2 bits a frequency
};

__device__ __forceinline__ int rope_axis(const RopeAngles& a, int i) { return (a.axis[i >> 4] >> (2 * (i & 15))) & 3; }

// (cos, sin) of position x frequency, times the factor. The angle is taken in 64 bits, where the product of an int32 and an
// fp32 is off by 2^-54 of itself at most, and reduced to half a turn there; what is left is exact enough in 32 (a position
// of a million in 32 bits would leave 0.03 radians).
__device__ __forceinline__ float2 rope_angle(const RopeAngles& a, int pos, int i) {
  const double turns = (double)pos * (double)a.inv_freq[i] * 0.15915494309189533577;
  float s, c;
  sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
  return make_float2(c * a.factor, s * a.factor * a.turn);
}

// A pair turned: one product and one fma each, the same in every kernel.
__device__ __forceinline__ void turn_pair(float& a, float& b, float2 cs) {
  const float x = a, y = b, ys = -y * cs.y, xs = x * cs.y;
  a = fmaf(x, cs.x, ys);
  b = fmaf(y, cs.x, xs);
}

}  // namespace dsa

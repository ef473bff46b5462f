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

// (cos, sin) of a number of turns up to a half: the nearest quarter turn off (exactly), then the series of both about 0 for
// at most an eighth of a turn, whose first terms left out are 2e-9 (sin) and 2e-10 (cos).
__device__ __forceinline__ float2 cos_sin_turns(float turns) {
  const float q = rintf(4.0f * turns), x = 6.28318530717958648f * fmaf(-0.25f, q, turns), y = x * x;
  float s = fmaf(y, 2.75573192e-6f, -1.98412698e-4f), c = fmaf(y, -2.75573192e-7f, 2.48015873e-5f);
  s = fmaf(y, s, 8.33333333e-3f), c = fmaf(y, c, -1.38888889e-3f);
  s = fmaf(y, s, -1.66666667e-1f), c = fmaf(y, c, 4.16666667e-2f);
  s = fmaf(y * x, s, x), c = fmaf(y, c, -0.5f);
  c = fmaf(y, c, 1.0f);
  const int n = (int)q;  // (-2 .. 2) quarter turns on top: (c, s) -> (-s, c) each
  const float a = n & 1 ? s : c, b = n & 1 ? c : s;
  return make_float2(n == 1 || n == 2 || n == -2 ? -a : a, n < 0 || n == 2 ? -b : b);
}

// (cos, sin) of position x frequency, times the factor. The angle is taken in 64 bits, where the product of an int32 and an
// fp32 is off by 2^-54 of itself at most, and reduced to half a turn there; what is left is exact enough in 32 (a position
// of a million in 32 bits would leave 0.03 radians).
__device__ __forceinline__ float2 rope_angle(const RopeAngles& a, int pos, int i) {
  const double turns = (double)pos * (double)a.inv_freq[i] * 0.15915494309189533577;
  const float2 cs = cos_sin_turns((float)(turns - rint(turns)));
  return make_float2(cs.x * a.factor, cs.y * a.factor * a.turn);
}

// A pair turned: one product and one fma each, the same in every kernel.
__device__ __forceinline__ void turn_pair(float& a, float& b, float2 cs) {
  const float x = a, y = b, ys = -y * cs.y, xs = x * cs.y;
  a = fmaf(x, cs.x, ys);
  b = fmaf(y, cs.x, xs);
}

}  // namespace dsa

// Rotary positions: pair i of a head at position p is turned by the angle p * f_i and multiplied by a magnitude m,
//   (a, b) -> (m a cos - m b sin, m a sin + m b cos).
// The angle is kept in turns: f_i / (2 pi) comes as a 64-bit fixed-point fraction of a turn, so that p * f_i modulo one turn is the low
// word of an integer product, exact to |p| * 2^-65 turns at any position (in 32-bit floating point the fastest pair is off by 0.03
// radians at position 2^20), without a table of positions, double precision or a reduction of the angle.
#pragma once

#include "ma_common.cuh"

namespace ma {

constexpr int kMaxPairs = 128;  // of a head: widths up to 256

struct RotaryArgs {
  int pairs;        // rotated pairs of a head; 0: nothing is rotated
  int interleaved;  // pair i = features (2i, 2i + 1), else (i, pairs + i)
  float magnitude;
  float sign;       // -1: the transpose, which turns back (backward pass)
  unsigned long long turns[kMaxPairs];
};

// m * (cos, sin) of pair i at position p.
__device__ __forceinline__ float2 rotary_turn(const RotaryArgs& r, int i, long long p) {
  const unsigned long long phase = (unsigned long long)p * r.turns[i];
  // the upper half word is the angle in units of 2^-31 half turns, in [-1, 1)
  const float half_turns = (float)(int)(phase >> 32) * 4.656612873077393e-10f;
  float s, c;
  sincospif(half_turns, &s, &c);
  return make_float2(r.magnitude * c, r.magnitude * r.sign * s);
}

// Host: checks the definition of the caller and copies it into kernel arguments; nullptr if it is fine.
const char* rotary_args(const ma_b200_rotary* r, int width, RotaryArgs* a);
cudaError_t launch_rotary(const ma_b200_rotation* p, const RotaryArgs& rotary, cudaStream_t stream);

}  // namespace ma

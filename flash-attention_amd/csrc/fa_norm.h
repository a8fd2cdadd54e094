// One head's vector of queries or keys, normalised by its root mean square, weighted and turned by its position:
//   y = R_t (w * x r),  r = 1 / sqrt(mean(x^2) + eps)
// and the gradient's way back through it.  A vector's D elements lie 8 to a lane over D / 8 neighbouring lanes (16 bytes each), so that the
// two sums over a vector are additions between lanes of at most 16, which DPP operands make without LDS.
// Everything between the one read and the one rounding is in fp32.
#pragma once

#include <type_traits>

#include "fa_common.h"

namespace fa {

// Workgroups of `waves` waves each that walk over rows, for the whole device: whole ones a compute unit, about `most` waves of them.
inline int walking_workgroups(int waves, int most) {
  const int each = (most + waves / 2) / waves;
  return 256 * (each > 0 ? each : 1);
}

// Sum over the CH lanes (2, 4, 8 or 16, aligned) that hold a vector, in each of them.
template <int CH>
FA_DEVICE float vector_sum(float x) {
  const auto other = [](float v, auto ctrl) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  x += other(x, std::integral_constant<int, 0xB1>{});                          // lane ^ 1
  if constexpr (CH >= 4) x += other(x, std::integral_constant<int, 0x4E>{});   // lane ^ 2
  if constexpr (CH >= 8) x += other(x, std::integral_constant<int, 0x141>{});  // 7 - lane of 8: the other quad
  if constexpr (CH >= 16) x += other(x, std::integral_constant<int, 0x140>{}); // 15 - lane of 16: the other eight
  return x;
}

template <typename T>
FA_DEVICE void load_weights(const void* w, bool fp32, int ch, float (&out)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++)
    out[i] = fp32 ? reinterpret_cast<const float*>(w)[ch * 8 + i] : (float)reinterpret_cast<const T*>(w)[ch * 8 + i];
}

template <int CH>
FA_DEVICE float inverse_rms(const float (&x)[8], float eps) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++) ss = __builtin_fmaf(x[i], x[i], ss);
  return rsqrtf(vector_sum<CH>(ss) * (1.f / (8 * CH)) + eps);
}

// Pairs (x[2e], x[2e+1]) turned by the angles of c4, s4 (rotate8 of fa_common.h on fp32 values); turn_back: by the opposite ones.
template <typename V4>
FA_DEVICE void turn(float (&x)[8], V4 c4, V4 s4) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float a = x[2 * e], b = x[2 * e + 1], c = (float)c4[e], s = (float)s4[e];
    x[2 * e] = a * c - b * s;
    x[2 * e + 1] = b * c + a * s;
  }
}
template <typename V4>
FA_DEVICE void turn_back(float (&x)[8], V4 c4, V4 s4) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float a = x[2 * e], b = x[2 * e + 1], c = (float)c4[e], s = (float)s4[e];
    x[2 * e] = a * c + b * s;
    x[2 * e + 1] = b * c - a * s;
  }
}

}  // namespace fa

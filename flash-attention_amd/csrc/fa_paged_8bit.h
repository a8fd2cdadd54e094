// Caches in 8 bits.  A row (the D values of a slot and key head) is held as e4m3 values y_i and one exponent e, and stands for y_i 2^e:
//   e = the smallest with max |x_i| <= 448 2^e (finite x_i), inside [least, most];   y_i = e4m3(x_i 2^-e), to nearest, ties to even;   inf and NaN: NaN.
// Eight bits with an exponent field lose the same 2^-4 of a value whatever the scale is, so a power of two serves as well as any and costs one byte (e + 127) a row;
// and what a row stands for, four significant bits, is exact in fp16 and bf16: reading it back rounds nothing.  least and most keep it so.  fp16: e4m3's last
// step 2^-9 times 2^-15 is fp16's; bf16: values below 2^-109 go.  At e = most a value of 256 would be more than the type holds: 240 is the largest there.
#pragma once

#include "fa_paged.h"

namespace fa {

template <typename T>
struct RowExponent;
template <>
struct RowExponent<_Float16> {
  static constexpr int least = -15, most = 8;
};
template <>
struct RowExponent<__bf16> {
  static constexpr int least = -100, most = 120;
};

FA_DEVICE float power_of_two(int byte) { return __uint_as_float((uint32_t)byte << 23); }  // 2^(byte - 127)
// 2^(127 - byte); 255, which is nobody's exponent but may lie behind a sequence's end, gives 0 and not infinity
FA_DEVICE float power_of_minus(uint32_t byte) { return __uint_as_float(__builtin_elementwise_sub_sat(254u, byte) << 23); }

// Eight e4m3 values times 2^(byte - 127), `scale` being that power; exact.  The instruction takes the scale's exponent for nothing.
FA_DEVICE f16x8 dequant8(u32x2 w, float scale, f16x8*) {
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  f16x8 y;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const v2 x = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i >> 1], scale, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i >> 1], scale, false);
    y[2 * i] = x[0];
    y[2 * i + 1] = x[1];
  }
  return y;
}
FA_DEVICE bf16x8 dequant8(u32x2 w, float scale, bf16x8*) {
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  bf16x8 y;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const v2 x = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i >> 1], scale, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i >> 1], scale, false);
    y[2 * i] = x[0];
    y[2 * i + 1] = x[1];
  }
  return y;
}
template <typename T>
FA_DEVICE typename Elem<T>::vec8 dequant8(u32x2 w, float scale) {
  return dequant8(w, scale, static_cast<typename Elem<T>::vec8*>(nullptr));
}

// The largest finite magnitude of eight values, as bits (of numbers that are not negative they are in order).  Infinities and NaN are rare: looked for once for the wave.
FA_DEVICE uint32_t finite_top(const float (&x)[8]) {
  constexpr uint32_t kInf = 0x7f800000u;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
    top = u > top ? u : top;
  }
  if (__builtin_expect(__any(top >= kInf), 0)) {
    top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
      top = u < kInf && u > top ? u : top;
    }
  }
  return top;
}
// The byte of a row whose largest finite magnitude has the bits u (448 = 7/8 * 2^9)
template <typename T>
FA_DEVICE int row_exponent(uint32_t u) {
  int e = (int)(u >> 23) - 135 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < RowExponent<T>::least ? RowExponent<T>::least : e;  // (zeros, too)
  return (e > RowExponent<T>::most ? RowExponent<T>::most : e) + 127;
}
// Eight values of a row with that byte.  Finite ones are 448 at most, and what is not becomes NaN as it is converted.
template <typename T>
FA_DEVICE u32x2 quant8(const float (&x)[8], int byte) {
  const float down = power_of_two(254 - byte);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; i++) y[i] = x[i] * down;
  if (__builtin_expect(__any(byte == RowExponent<T>::most + 127), 0)) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float z = __builtin_amdgcn_fmed3f(y[i], -240.f, 240.f);
      if (byte == RowExponent<T>::most + 127 && __builtin_fabsf(y[i]) < INFINITY) y[i] = z;
    }
  }
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
    w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], lo, true);
  }
  return w;
}

// One direct-to-LDS wave instruction from addresses of each lane's own (dma16 of fa_stage.h: from one base)
FA_DEVICE void dma16_from(const void* lane_src, unsigned char* lds_dst) {
  const uint32_t lds_addr = (uint32_t)(uintptr_t)(FA_LDS void*)lds_dst;
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(lane_src), "s"(lds_addr)
               : "memory", "m0");
}

// A tile of rows of D bytes in LDS, chunks of 16 bytes permuted as those of fa_stage.h are: a line of the LDS (256 bytes, 16 lanes of 16 bytes or 32 of 8 a
// cycle) holds 256 / D rows.  K, row fragments: 16 lanes read the same chunk of 16 rows.  V, transposed reads: 32 lanes read two neighbouring chunks of the eight
// rows 4 hf + {0 .. 3, 8 .. 11} (D = 32: two lanes meet in a bank, the rows being too few for a line).
template <int D, int KIND>
FA_DEVICE int tile_swz8(int r) {
  constexpr int CH = D / 16;
  if (CH == 1) return 0;
  if (KIND == kSwzRow) return (r / (256 / D)) % CH;
  if (CH == 8) return 2 * (((r >> 1) & 1) | ((r >> 3) & 1) << 1);
  if (CH == 4) return 2 * ((r >> 3) & 1);
  return 0;
}

// Stages 16 consecutive keys (or values), as GroupStager does those of 16 bits.
template <int D, int KIND, bool kStream = false>
struct GroupStager8 {
  static constexpr int CH = D / 16;
  static constexpr int RPI = 64 / CH < 16 ? 64 / CH : 16;  // rows per instruction (d < 64: some lanes have none)
  static constexpr int NI = 16 / RPI;
  static constexpr int kBytes = 16 * D;
  uint32_t off[NI];
  int rl, pch;

  FA_DEVICE void init(int lane, int64_t rsb) {
    rl = lane / CH;
    pch = lane % CH;
#pragma unroll
    for (int i = 0; i < NI; i++) off[i] = (uint32_t)((i * RPI + rl) * rsb) + 16u * (uint32_t)(pch ^ tile_swz8<D, KIND>(i * RPI + rl));
  }
  // (last: as in GroupStager)
  FA_DEVICE void issue(const char* base, int64_t rsb, int last, unsigned char* dst) const {
    if (64 / CH > 16 && rl >= 16) return;
    if (__builtin_expect(last >= 15, 1)) {
#pragma unroll
      for (int i = 0; i < NI; i++) dma16<kStream>(base, off[i], dst + i * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const int r = i * RPI + rl;
        dma16<kStream>(base, (uint32_t)((r < last ? r : last) * rsb) + 16u * (uint32_t)(pch ^ tile_swz8<D, KIND>(r)), dst + i * 1024);
      }
    }
  }
};

// Transposed read of bytes: among 16 lanes, lane j gives the address of 8 bytes, and lane i receives byte i % 8 of what lanes 2 r + i / 8 point at, r = 0 .. 7.
FA_DEVICE u32x2 lds_read_tr8(const unsigned char* lds_ptr) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  return bitcast<u32x2>(__builtin_amdgcn_ds_read_tr8_b64_v2i32((FA_LDS i32x2*)(lds_ptr)));
}

}  // namespace fa

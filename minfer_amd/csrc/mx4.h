// Microscaled numbers of 4 and 6 bits: the two formats, how they are stored, and what turns values into them.
//
// 32 neighbouring values of a row (a block) share a power of two, stored as e + 127 in a byte (255: the block is NaN).
//   E2M1, 4 bits, for matrices: 0 0.5 1 1.5 2 3 4 6 and their negatives.
//   E2M3, 6 bits, for the rows that are multiplied with them: 0 to 2 in steps of 1/8, to 4 in steps of 1/4, to 7.5 in steps of 1/2.
// The power is the smallest with which the block's largest magnitude is at most 7 (which becomes 6, half a step off) or 7.5, so no value
// is off by more than half a step of the list.  With |largest| = 1.f 2^x that is x - 2, or x - 1 where the mantissa is above 1.75 or 1.875:
// an addition to the bits that carries into the exponent there (`mx_power`).  From 2^-127 on; a block of zeros has that one.
//
// Why 6 bits for the rows: the matrix cores multiply 6-bit by 4-bit operands at twice the rate of 8-bit by 4-bit ones (32x32x64, operands in
// registers: 8,700 / 4,890 TFLOP/s measured), E2M3 has the three mantissa bits that E4M3 has, and within a block the range of E4M3 is not
// needed.  The sums also come out better: products of E4M3's 15 octaves lose what lies some 16 bits below the largest of an instruction
// (4.5e-5 of the sum measured), those of E2M3 with E2M1 span 10 bits and are added exactly (1e-8, what 32 bits give).
//
// Matrices, `[rows][k]`: codes [ceil(rows / 16)][ceil(k / 128)][64][16 bytes]: place 16 g + r of a tile holds row r's values
// 32 g .. 32 g + 31 of the tile's 128, two a byte, the lower one in the low half: what lane 16 g + r of a wave feeds to
// the 16x16x128 instruction, so a wave's load of a tile is one kilobyte without a gap.  Powers [ceil(rows / 16)][ceil(k / 512)][64][4 bytes]:
// byte s of place 16 g + r is that of the block of tile 4 S + s: one load serves four steps.  Past the rows and past k: zeros.
// Rows in 6 bits (scratch of a product), `[m][k]`: per 32 rows and 128 k three kilobytes: [4 g][32 r][16 bytes], the first 21 values and a third
// of one, then [4 g][32 r][8 bytes]; powers [ceil(m / 32)][ceil(k / 512)][4 g][32 r][4 bytes].
#pragma once
#include "common.h"

typedef int intx8 __attribute__((ext_vector_type(8)));
typedef unsigned uintx6 __attribute__((ext_vector_type(6)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x32 __attribute__((ext_vector_type(32)));
typedef float floatx2 __attribute__((ext_vector_type(2)));

constexpr unsigned MX_E2M1_CARRY = 0x1FFFFF, MX_E2M3_CARRY = 0x0FFFFF;       // mantissas above 1.75, above 1.875
constexpr int MX_FP6 = 2, MX_FP4 = 4;                                        // operand formats of the matrix instructions

// the stored power of a block whose largest magnitude has these bits (of a 32-bit float, without the sign)
__device__ __forceinline__ unsigned mx_power(unsigned largest, unsigned carry) {
  if (largest >= 0x7F800000u) return 255;
  return (unsigned)max((int)((largest + carry) >> 23) - 2, 0);
}
// ... as the float that the conversion instructions divide by (2^-127 has no normal one)
__device__ __forceinline__ float mx_unit(unsigned power) { return __uint_as_float(max(power << 23, 0x00400000u)); }

typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));
// the larger of the magnitudes in both halves of packed bfloat16 pairs (the bits of magnitudes are in the order of their values, NaN above all)
__device__ __forceinline__ unsigned max_pairs(unsigned a, unsigned b) {
  const ushortx2 x = __builtin_bit_cast(ushortx2, a), y = __builtin_bit_cast(ushortx2, b);
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(x, y));
}

// A block of 32 values in registers -> its power and its codes in E2M3.  `words`: 16 pairs of bfloat16, or 32 floats.
__device__ __forceinline__ uintx6 mx6_block(const unsigned (&words)[16], unsigned& power) {
  unsigned m = words[0] & 0x7FFF7FFFu;
#pragma unroll
  for (int i = 1; i < 16; ++i) m = max_pairs(m, words[i] & 0x7FFF7FFFu);
  power = mx_power(max(m & 0xFFFF0000u, m << 16), MX_E2M3_CARRY);
  bf16x32 v;
  __builtin_memcpy(&v, words, 64);
  return __builtin_amdgcn_cvt_scalef32_pk32_fp6_bf16(v, mx_unit(power));
}
__device__ __forceinline__ uintx6 mx6_block(const unsigned (&words)[32], unsigned& power) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = max(m, words[i] & 0x7FFFFFFFu);
  power = mx_power(m, MX_E2M3_CARRY);
  floatx16 even, odd;                              // the instruction takes its values from two operands in turn
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    even[i] = __uint_as_float(words[2 * i]);
    odd[i] = __uint_as_float(words[2 * i + 1]);
  }
  return __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, mx_unit(power));
}

__device__ __forceinline__ intx8 mx6_operand(const uintx6& c) {
  return intx8{(int)c[0], (int)c[1], (int)c[2], (int)c[3], (int)c[4], (int)c[5], 0, 0};
}
__device__ __forceinline__ intx8 mx4_operand(const uint4& c) { return intx8{(int)c.x, (int)c.y, (int)c.z, (int)c.w, 0, 0, 0, 0}; }

// The words of the block of 32 values of a row that begins at value k0, zeros from k_end on.  VEC: rows and k_end allow 16-byte loads of whole ones.
template <bool VEC, int W, typename T>
__device__ __forceinline__ void mx_load_block(const T* __restrict__ row, int k0, int k_end, unsigned (&words)[W]) {
  constexpr int PER = 16 / sizeof(T);              // values of a 16-byte load
#pragma unroll
  for (int i = 0; i < 32 / PER; ++i) {
    uint4 v = uint4{0, 0, 0, 0};
    const int k = k0 + i * PER;
    if (VEC) {
      if (k < k_end) v = *reinterpret_cast<const uint4*>(row + k);
    } else {
      alignas(16) T raw[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) raw[j] = k + j < k_end ? row[k + j] : (T)0.f;
      v = *reinterpret_cast<const uint4*>(raw);
    }
    words[4 * i] = v.x;
    words[4 * i + 1] = v.y;
    words[4 * i + 2] = v.z;
    words[4 * i + 3] = v.w;
  }
}

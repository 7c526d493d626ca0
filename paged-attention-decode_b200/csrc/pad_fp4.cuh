// pad_fp4.cuh -- the microscaled 4-bit cache format, shared by the kernels
// that write, read and attend over it.
//
// A row (one token of one KV head) is D/2 code bytes and 4 scale bytes. Code
// byte i holds dims 2i (low nibble) and 2i+1 (high nibble) as e2m1: sign, two
// exponent bits, one mantissa bit, i.e. 0 0.5 1 1.5 2 3 4 6 and their
// negatives. Scale byte j is the power of two 2^(byte - 127) of dims
// [32j, 32j + 32), 255 meaning NaN; bytes past D/32 are unused. The scale row
// is 4 bytes at every head dim so that it is one aligned word.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

namespace pad {

constexpr int kFp4Block = 32;       // dims that share a scale
constexpr int kFp4ScaleRow = 4;     // bytes of a scale row
constexpr int kFp4MinExp = -24;     // fp16 has no finer step: a smaller scale could only lose range
constexpr uint32_t kFp4NanScale = 255;

// 2^(byte - 127) in fp32 (byte 0 is the subnormal 2^-127, 255 is NaN).
__device__ __forceinline__ float fp4_scale_f32(uint32_t byte) {
  const uint32_t bits = byte == 255u ? 0x7fc00000u : (byte == 0u ? 0x00400000u : byte << 23);
  return __uint_as_float(bits);
}

// Byte `i` (0..3) of four code bytes -> (low nibble, high nibble) as fp16x2.
// One conversion instruction; exact, e2m1 being a subset of fp16.
__device__ __forceinline__ void fp4_unpack4(uint32_t w, uint32_t& h0, uint32_t& h1, uint32_t& h2, uint32_t& h3) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h0), "=r"(h1), "=r"(h2), "=r"(h3)
      : "r"(w));
}

// Two scale bytes (low 16 bits) -> 2^(byte - 127) as two bf16, exactly, 255 as NaN.
__device__ __forceinline__ uint32_t fp4_scale2_bf16(uint32_t two) {
  uint32_t y;
  asm("{\n\t.reg .b16 x;\n\tcvt.u16.u32 x, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, x;\n\t}" : "=r"(y) : "r"(two));
  return y;
}

// Eight fp32 values -> four code bytes, rounded to nearest even and saturated
// at +-6 (x[0] in the lowest nibble).
__device__ __forceinline__ uint32_t fp4_pack8(const float (&x)[8]) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return w;
}

}  // namespace pad

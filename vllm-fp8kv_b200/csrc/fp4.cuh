// fp4.cuh -- the 4-bit MLA row (fp4_ds_mla) and its conversions.
//
// Row format (416 bytes per KV slot):
//   [  0:256)  512 x e2m1          NoPE latent, element 2i in the low nibble of byte i
//   [256:288)   32 x float8_e4m3fn one scale per 16 latent values
//   [288:416)   64 x bfloat16      RoPE, raw
// A latent value is code * scale.  e2m1 has 2 significant bits and e4m3 has 4,
// so the product has at most 6 and lies in {0} u [2^-10, 2688] (a multiple of
// 2^-10): exact in fp16 and in bf16, subnormal scales included.  The kernels
// therefore feed the tensor cores fp16 latents without any rounding.
#pragma once
#include "common.cuh"

namespace fp8mla {
namespace fp4 {

constexpr int kFp4Group = 16;                   // latent values per scale
constexpr int kFp4CodeBytes = kNope / 2;        // 256
constexpr int kFp4ScaleOff = kFp4CodeBytes;        // 256
constexpr int kFp4RopeOff = kFp4ScaleOff + kNope / kFp4Group;  // 288
constexpr int kFp4RowBytes = kFp4RopeOff + 2 * kRope;       // 416
static_assert(kFp4RowBytes == FP8MLA_FP4_ROW_BYTES && kFp4ScaleOff == FP8MLA_FP4_SCALE_OFF &&
                  kFp4RopeOff == FP8MLA_FP4_ROPE_OFF && kFp4RowBytes % 16 == 0,
              "row geometry");

// 8 e2m1 codes -> 4 f16x2, element 2b in the low half of h[b]
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
      " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// 2 e4m3 bytes (low 16 bits of w) -> f16x2
__device__ __forceinline__ uint32_t e4m3x2_to_f16(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, l;\n}\n" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// The power of two, k, that a head's q is taken times on its way to fp16 (its rope in
// bf16 too: both products meet in one accumulator).  m and mr: the largest magnitudes
// (bf16 bits) of its latent part and of its rope; scale_log2: the factor from q . k
// to scores in log2 units.
//   * It brings the latents' largest value to [2^8, 2^9): what is lost below 2^-17 of
//     the scaled values is under 2^-33 of the largest.
//   * It is held to 2^24 / scale_log2.  A latent's rounding error (2^-25 at most) then
//     moves a score by less than 2^-48 a unit of cached latent, 2^-27 for a row full of
//     its largest, 2688: further bits of tiny latents would say nothing.  And a score is
//     at least 2^-24 of its accumulator, so sums are finite up to scores of 2^103,
//     however tiny the latents beside whatever rope.
//   * The rope itself stays below 2^127.
// 0 for latents of zeros, inf or NaN.  Exponents of bf16 and fp32 lie in [-127, 128],
// so k lies in [-119, 126]: 2^k and 2^-k are normal.
__device__ __forceinline__ int q_power(int m, int mr, float scale_log2) {
  const int em = (m >> 7) - 127, er = (mr >> 7) - 127;
  const int es = (int)((__float_as_uint(scale_log2) >> 23) & 255u) - 127;
  const int k = min(min(8 - em, es + 24), min(126, 126 - er));
  return m == 0 || m >= 0x7F80 ? 0 : k;
}
// Codes times scale in bf16, exact (at most 6 significant bits, and far from the
// ends of the range).  An fp16 code (normal or zero) moved three bits to the right
// under its sign is the bf16 code times 2^-112; the scale carries the 2^112.
__device__ __forceinline__ uint32_t bf16_scale(uint32_t e4m3) {
  const uint32_t h = e4m3x2_to_f16(e4m3);
  const float s = __half2float(__ushort_as_half((unsigned short)(h & 0xFFFFu))) * 0x1p112f;
  return pack_bf16x2(s, s);
}
__device__ __forceinline__ uint32_t scaled_bf16x2(uint32_t f16_codes, uint32_t scale) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(((f16_codes >> 3) & 0x0FFF0FFFu) | (f16_codes & 0x80008000u)), "r"(scale));
  return r;
}

}  // namespace fp4
}  // namespace fp8mla

// Rows held in 4 bits: groups of 64 channels with z = least value and s = bf16((most - least) / 15), a channel is the
// code n of s n + z.  A row of up to 64 channels has the width 64, a longer one is padded to whole blocks of 128.
// Eight codes make a 32-bit word: channel i of the eight is nibble (i >> 1) + 4 (i & 1), so that masking a shifted word
// with 0x000f000f leaves two neighbouring channels in the two halves of a register.  Word 2g + h of a block of 128 holds
// channels 64 h + 8 g .. + 7, so that a contiguous piece of a block has words of both groups; a block of 64 is word g for
// channels 8 g .. + 7.  `affine` is (s, z) per group in one 32-bit word, s in the low half.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "b200.cuh"

namespace q4 {

constexpr int kGroup = 64;

__host__ __device__ inline int row_width(int channels) { return channels <= 64 ? 64 : (channels + 127) / 128 * 128; }

// word of a row of `width` channels -> its first channel
__device__ __forceinline__ int word_channel(int word, int width) {
  if (width == 64) return word * 8;
  return (word >> 4) * 128 + (word & 1) * 64 + ((word >> 1) & 7) * 8;
}
// word -> its group
__device__ __forceinline__ int word_group(int word, int width) { return width == 64 ? 0 : (word >> 4) * 2 + (word & 1); }

__device__ __forceinline__ float scale_of(uint32_t affine) { return __uint_as_float(affine << 16); }
__device__ __forceinline__ float least_of(uint32_t affine) { return __uint_as_float(affine & 0xffff0000u); }

// the eight codes of a word in channel order
__device__ __forceinline__ void unpack(uint32_t word, float (&n)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = static_cast<float>((word >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u);
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Scale of a group from its least and largest value, as its bf16 bits: (most - least) / 15; NaN where the spread is no
// number or beyond fp32 (a NaN or an infinity in the group), 0 where it is below the least normal number.
__device__ __forceinline__ uint32_t scale_bits(float least, float most) {
  const float s = __bfloat162float(__float2bfloat16(__fdiv_rn(most - least, 15.f)));
  if (!(s <= 3.4e38f)) return 0x7fc0u;
  return s < 1.17549435e-38f ? 0u : __float_as_uint(s) >> 16;
}

// Code of x: (x - least) / s to the nearest whole number, ties to even, of the numbers themselves and not of their fp32
// quotient.  The quotient by the reciprocal is off by 4e-6 at most, so it decides wherever it is further than that from a
// border k + 1/2; near one the sign of x - least - (k + 1/2) s decides, which fp32 has exactly: the product has 13 bits
// and goes into one fused rounding, and what the difference x - least lost (it loses something only where the two are 2^16
// apart or more) is recovered and counts where the rest is zero.
__device__ __forceinline__ uint32_t code_of(float x, float least, float s, float inv) {
  const float d = x - least;
  const float q = d * inv;
  float n = rintf(q);
  if (fabsf(q - n) > 0.499f) {
    const float k = floorf(q);
    const float r = fmaf(-(k + 0.5f), s, d);
    const float back = d - x;
    const float lost = (x - (d - back)) - (least + back);
    const bool above = r > 0.f || (r == 0.f && (lost > 0.f || (lost == 0.f && (static_cast<int>(k) & 1))));
    n = above ? k + 1.f : k;
  }
  return static_cast<uint32_t>(fminf(n, 15.f));
}

// The word of eight channels of a group with the given affine pair.
__device__ __forceinline__ uint32_t pack(const float (&x)[8], uint32_t affine) {
  const float s = scale_of(affine), least = least_of(affine);
  if (!(s > 0.f)) return 0u;   // a constant group, or one without numbers
  const float inv = __frcp_rn(s);
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) word |= code_of(x[i], least, s, inv) << (4 * ((i >> 1) + 4 * (i & 1)));
  return word;
}

__device__ __forceinline__ void unpack_bf16(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// Values of a word as eight bf16, rounded once.
__device__ __forceinline__ uint4 values_bf16(uint32_t word, uint32_t affine) {
  const float s = scale_of(affine), z = least_of(affine);
  float n[8];
  unpack(word, n);
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = fmaf(n[i], s, z);
  return make_uint4(b200::pack_bf16x2(n[0], n[1]), b200::pack_bf16x2(n[2], n[3]), b200::pack_bf16x2(n[4], n[5]),
                    b200::pack_bf16x2(n[6], n[7]));
}

}  // namespace q4

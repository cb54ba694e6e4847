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

// Whether codes and pairs lie where the kernels may read them: codes in 16 bytes at a time, pairs in the 4 (rows of 64) or 8
// that a block has, so that a slice of a larger tensor between any two of its rows will do.
inline bool rows_aligned(const void* codes, const void* affine, int width) {
  return (reinterpret_cast<uintptr_t>(codes) & 15) == 0 && (reinterpret_cast<uintptr_t>(affine) & (width == 64 ? 3 : 7)) == 0;
}

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
// The quotient is x zh + x zl with zh + zl = 1 / 15 to 48 bits, one rounding after the fused sum (Brisebarre, Muller and
// Raina, "Accelerating Correctly Rounded Floating-Point Division When the Divisor Is Known in Advance", 2004); for 15 it is
// the correctly rounded one for every 24-bit significand.
__device__ __forceinline__ uint32_t scale_bits(float least, float most) {
  constexpr float zh = 0x1.111112p-4f, zl = -0x1.dddddep-29f;
  const float w = most - least;
  const float s = __bfloat162float(__float2bfloat16(fmaf(w, zh, w * zl)));
  if (!(s <= 3.4e38f)) return 0x7fc0u;
  return s < 1.17549435e-38f ? 0u : __float_as_uint(s) >> 16;
}

// Code of x: (x - least) / s to the nearest whole number, ties to even, of the numbers themselves and not of their fp32
// quotient: near a border k + 1/2 the sign of x - least - (k + 1/2) s decides, which fp32 has exactly: the product has 13
// bits and goes into one fused rounding, and what the difference x - least lost (it loses something only where the two are
// 2^16 apart or more) is recovered and counts where the rest is zero.
__device__ __forceinline__ float exact_code(float x, float least, float s, float inv) {
  const float d = x - least;
  const float k = floorf(d * inv);
  const float r = fmaf(-(k + 0.5f), s, d);
  const float back = d - x;
  const float lost = (x - (d - back)) - (least + back);
  const bool above = r > 0.f || (r == 0.f && (lost > 0.f || (lost == 0.f && (static_cast<int>(k) & 1))));
  return above ? k + 1.f : k;
}

// The word of eight channels of a group with the given affine pair.  Where the channels and the least are multiples of G =
// 2^-17 of the scale's power of two (all but groups of a very wide range are), the differences are exact, of 22 bits at most,
// and a quotient with one Newton step on the approximate reciprocal, off by little more than 2^-24 of itself, rounds to the
// right whole number: the borders (k + 1/2) s are multiples of G too, so what is not on a border is G away from it, 2^-22 of
// it at least, and what is on one comes out as k + 1/2 itself.  Codes come out of the low bits of q + 1.5 2^23, two to a byte by
// one multiply-add.
__device__ __forceinline__ uint32_t pack(const float (&x)[8], uint32_t affine) {
  using namespace b200;
  const float s = scale_of(affine), least = least_of(affine);
  if (!(s > 0.f)) return 0u;   // a constant group, or one without numbers
  const float inv = __fdividef(1.f, s);        // 2 ulp
  constexpr float magic = 12582912.f;
  // adding 1.5 2^23 G and taking it off again leaves multiples of G, and of what is larger no less (a bf16 above 2^7 G is one)
  const float grid = __uint_as_float((__float_as_uint(s) & 0x7f800000u)) * 96.f;
  const uint64_t inv2 = f2_pack(inv, inv), least2 = f2_pack(-least, -least), s2 = f2_pack(-s, -s);
  const uint64_t magic2 = f2_pack(magic, magic), minus2 = f2_pack(-magic, -magic);
  const uint64_t grid2 = f2_pack(grid, grid), ungrid2 = f2_pack(-grid, -grid);
  float n[8];
  bool coarse = (least + grid) - grid == least;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t x2 = f2_pack(x[i], x[i + 1]), d = f2_add(x2, least2), q = f2_mul(d, inv2);
    f2_unpack(f2_add(f2_add(f2_fma(f2_fma(q, s2, d), inv2, q), magic2), minus2), n[i], n[i + 1]);
    float u, v;
    f2_unpack(f2_add(f2_add(x2, grid2), ungrid2), u, v);
    coarse = coarse && u == x[i] && v == x[i + 1];
  }
  if (!coarse) {
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = exact_code(x[i], least, s, inv);
  }
  // nibbles 0 .. 7 are channels 0 2 4 6 1 3 5 7; none is above 15: s is at least 1 - 2^-8 of a fifteenth of the spread
  const uint32_t b0 = __float_as_uint(fmaf(n[2], 16.f, n[0]) + magic), b1 = __float_as_uint(fmaf(n[6], 16.f, n[4]) + magic);
  const uint32_t b2 = __float_as_uint(fmaf(n[3], 16.f, n[1]) + magic), b3 = __float_as_uint(fmaf(n[7], 16.f, n[5]) + magic);
  return __byte_perm(__byte_perm(b0, b1, 0x0040), __byte_perm(b2, b3, 0x0040), 0x5410);
}

__device__ __forceinline__ void unpack_bf16(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// Codes P of both halves of w as bf16 128 + n: one shift and one three-input operation (a & b) | c, whose constants are kept
// in registers (opaque_masks), since an instruction has room for one.
template <int P>
__device__ __forceinline__ uint32_t coded(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(P ? w >> (4 * P) : w), "r"(mask), "r"(magic));
  return r;
}
__device__ __forceinline__ void opaque_masks(uint32_t& mask, uint32_t& magic) {
  mask = 0x000f000fu;
  magic = 0x43004300u;
  asm volatile("" : "+r"(mask), "+r"(magic));
}

// Values of a word as eight bf16, rounded once (after fp32).
__device__ __forceinline__ uint4 values_bf16(uint32_t word, uint32_t affine, uint32_t mask, uint32_t magic) {
  const uint64_t s = b200::f2_pack(scale_of(affine), scale_of(affine)), z = b200::f2_pack(least_of(affine), least_of(affine));
  const uint64_t minus = b200::f2_pack(-128.f, -128.f);
  const uint32_t pair[4] = {coded<0>(word, mask, magic), coded<1>(word, mask, magic), coded<2>(word, mask, magic),
                            coded<3>(word, mask, magic)};
  uint32_t out[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint64_t n = b200::f2_add(b200::f2_pack(__uint_as_float(pair[p] << 16), __uint_as_float(pair[p] & 0xffff0000u)), minus);
    float u, v;
    b200::f2_unpack(b200::f2_fma(n, s, z), u, v);
    out[p] = b200::pack_bf16x2(u, v);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// n / d by a multiplication: n, d below 2^31 (Granlund and Montgomery, "Division by Invariant Integers using
// Multiplication", 1994, figure 4.1).
struct Divisor {
  uint32_t d, mul, shift;
  Divisor() = default;
  __host__ explicit Divisor(uint32_t by) : d(by) {
    shift = 0;
    while (shift < 32 && (1ull << shift) < by) ++shift;
    mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - by)) / by + 1);
  }
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return (__umulhi(mul, n) + n) >> shift; }
};

}  // namespace q4

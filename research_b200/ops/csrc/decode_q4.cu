// Attention of one new token per sequence over a K/V cache held in 4 bits (quant4.cuh), head-major pages of any size.
//   o[h] = sum_r p_r (s n_r + z) / sum_r p_r,  p = softmax(scale * q . (s n + z)),  rows max(lo, 0) <= r < min(len, capacity)
// A sequence without such a row gets zeros.
#include <math_constants.h>

#include "quant4.cuh"
#include "host_util.cuh"

namespace {

using namespace q4;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
  const __nv_bfloat16* q;             // [B, Hq, D], heads D apart
  long long q_batch;
  const uint32_t *k_codes, *k_affine, *v_codes, *v_affine;
  const int *lengths, *lo;
  __nv_bfloat16* out;                 // [B, Hq, D]
  int B, Hq, Hkv, pages, page_rows;
  float scale_log2;
};

// One warp per query head: a lane per word of the row (the lanes beyond it take other rows), one pass with a running
// maximum and sum.
template <int D>
__global__ void __launch_bounds__(32) decode_q4_kernel(const AttnParams p) {
  constexpr int WORDS = D / 8, ROWS = 32 / WORDS;
  const int b = blockIdx.x / p.Hq, hq = blockIdx.x % p.Hq, h = hq / (p.Hq / p.Hkv);
  const int lane = threadIdx.x, w = lane % WORDS, sub = lane / WORDS;
  b200::pdl_launch_dependents();
  b200::pdl_wait();
  const int first = p.lo ? max(p.lo[b], 0) : 0;
  const int end = static_cast<int>(min(static_cast<long long>(p.lengths[b]), static_cast<long long>(p.pages) * p.page_rows));
  const int c = word_channel(w, D), group = word_group(w, D);
  float q[8], acc[8] = {}, m = -CUDART_INF_F, l = 0.f;
  unpack_bf16(*reinterpret_cast<const uint4*>(p.q + b * p.q_batch + static_cast<long long>(hq) * D + c), q);
  for (int r0 = first; r0 < end; r0 += ROWS) {
    const int r = r0 + sub;
    const bool seen = r < end;
    const int at = seen ? r : first, pg = at / p.page_rows;
    const long long row = ((static_cast<long long>(b) * p.pages + pg) * p.Hkv + h) * p.page_rows + (at - pg * p.page_rows);
    float n[8], s = 0.f;
    uint32_t a = p.k_affine[row * (D / 64) + group];
    unpack(p.k_codes[row * WORDS + w], n);
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(q[i], fmaf(n[i], scale_of(a), least_of(a)), s);
#pragma unroll
    for (int off = WORDS / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (!seen) continue;    // no shuffles below
    s *= p.scale_log2;
    const float m_new = fmaxf(m, s), m_use = m_new == -CUDART_INF_F ? 0.f : m_new;
    const float alpha = exp2f(m - m_use), pr = exp2f(s - m_use);
    m = m_new;
    l = l * alpha + pr;
    a = p.v_affine[row * (D / 64) + group];
    unpack(p.v_codes[row * WORDS + w], n);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(acc[i], alpha, pr * fmaf(n[i], scale_of(a), least_of(a)));
  }
  __syncwarp();
  float mm = m;
#pragma unroll
  for (int off = 16; off >= WORDS; off >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, off));
  const float wgt = m == -CUDART_INF_F ? (l != l ? l : 0.f) : exp2f(m - mm);
  l *= wgt;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] *= wgt;
#pragma unroll
  for (int off = 16; off >= WORDS; off >>= 1) {
    l += __shfl_xor_sync(0xffffffffu, l, off);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], off);
  }
  if (sub == 0) {
    const float inv = end > first ? 1.f / l : 0.f;
    *reinterpret_cast<uint4*>(p.out + (static_cast<long long>(b) * p.Hq + hq) * D + c) =
        make_uint4(b200::pack_bf16x2(acc[0] * inv, acc[1] * inv), b200::pack_bf16x2(acc[2] * inv, acc[3] * inv),
                   b200::pack_bf16x2(acc[4] * inv, acc[5] * inv), b200::pack_bf16x2(acc[6] * inv, acc[7] * inv));
  }
}

}  // namespace

// q [B, Hq, D] bf16 (q_batch elements between sequences), caches [B, pages, Hkv, page_rows, ..] contiguous, lengths and lo
// int32 [B] (lo may be null), out [B, Hq, D] bf16.  D 64 or 128.
extern "C" int b200_q4_decode_attn(const void* q, long long q_batch, const void* k_codes, const void* k_affine,
                                   const void* v_codes, const void* v_affine, const void* lengths, const void* lo,
                                   void* out, int B, int Hq, int Hkv, int D, int pages, int page_rows, float scale,
                                   void* stream) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || pages <= 0 || page_rows <= 0 || (D != 64 && D != 128) ||
      (long long)pages * page_rows > 0x7fffffffll || (long long)B * Hq > 0x7fffffffll)
    return b200host::RC_BAD_SHAPE;
  if ((q_batch & 7) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_codes) |
                         reinterpret_cast<uintptr_t>(k_affine) | reinterpret_cast<uintptr_t>(v_codes) |
                         reinterpret_cast<uintptr_t>(v_affine) | reinterpret_cast<uintptr_t>(out)) & 15))
    return b200host::RC_BAD_ALIGNMENT;
  AttnParams p{(const __nv_bfloat16*)q, q_batch, (const uint32_t*)k_codes, (const uint32_t*)k_affine,
               (const uint32_t*)v_codes, (const uint32_t*)v_affine, (const int*)lengths, (const int*)lo,
               (__nv_bfloat16*)out, B, Hq, Hkv, pages, page_rows, scale * kLog2e};
  const bool pdl = b200host::pdl_enabled() != 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (D == 128) return static_cast<int>(b200host::launch_kernel(decode_q4_kernel<128>, dim3(B * Hq), dim3(32), 0, s, pdl, p));
  return static_cast<int>(b200host::launch_kernel(decode_q4_kernel<64>, dim3(B * Hq), dim3(32), 0, s, pdl, p));
}

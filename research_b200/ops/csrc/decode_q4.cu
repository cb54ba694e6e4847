// Attention of one new token per sequence over a K/V cache held in 4 bits (quant4.cuh), head-major pages of any size.
//   o[h] = sum_r p_r (s n_r + z) / sum_r p_r,  p = softmax(scale * q . (s n + z)),  rows max(lo, 0) <= r < min(len, capacity)
// A sequence without such a row gets zeros.
//
// Every cached row is read once for all query heads that share it.  A row of 128 has 72 bytes instead of 256, so what would
// be a stream for the memory becomes work for the SM: at the copy bandwidth 46 codes a clock and SM, too many for an FMA per
// code and head.  Both products therefore go through the tensor cores as m16n8k16 with the cache as the 16-row operand and
// up to eight query heads as the columns (a tcgen05 product would want the expanded rows in shared or tensor memory first,
// and its 128 x 16 tile has no more use for eight columns): a code c becomes the bf16 128 + c by one shift and one
// and-or per two codes, exact, and scales and least values are applied to the sums in fp32:
//   q . k_r = sum_groups s_r (sum q (128 + n) - 128 sum q) + z_r sum q
//   o       = sum_r (p_r s_r) (128 + n_r) - 136 sum_r (p_r s_r) + sum_r p_r (z_r + 8 s_r)      (centred: n - 8)
// p s enters the second product as two bf16 parts (up to four heads: in columns 4 .. 7 of the same product, else in a
// second one), which holds it to 2^-14; a single bf16 would cost as much as the rounding of the result does.
#include <math_constants.h>

#include "quant4.cuh"
#include "host_util.cuh"

namespace {

using namespace q4;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
  const __nv_bfloat16* q;             // [B, Hq, D], heads D apart
  long long q_batch;
  const uint8_t *k_codes, *k_affine, *v_codes, *v_affine;
  const int *lengths, *lo;
  __nv_bfloat16* out;                 // [B, Hq, D]
  float *part_o, *part_ml;            // [B, Hq, splits, D], [B, Hq, splits, 2]: (m in log2 units, l)
  int B, Hq, Hkv, pages, page_rows, splits;
  float scale_log2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// codes p of both halves of w as bf16 128 + n
template <int P>
__device__ __forceinline__ uint32_t coded(uint32_t w) { return ((w >> (4 * P)) & 0x000f000fu) | 0x43004300u; }

constexpr uint32_t kOnes = 0x3f803f80u;

// A warp works by itself on tiles of TR rows that it brings into a ring of its own in shared memory (cp.async, so pages may
// end anywhere); the warps of a block take turns, and their states are joined at the end.
//
// Fragments.  Lane (g, t) = (lane / 4, lane % 4).  In the products over the channels row m of the 16 is cache row pi(m) of the
// tile, pi(2 j) = j, pi(2 j + 1) = 7 - j (+ 8 for m >= 8): the lane's rows in the second product, whose index runs over the
// cache rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9, are then t, 7 - t, 8 + t, 15 - t, and neither product's reads from shared
// memory meet in a bank (rows of 128 with their 16-byte chunks swapped in pairs every second pair of rows).
template <int D, bool WIDE, int WARPS, int TR, int STAGES>
__global__ void __launch_bounds__(WARPS * 32) decode_q4_kernel(const __grid_constant__ AttnParams p) {
  constexpr int GROUPS = D / 64, KW = D / 32, STEPS = TR / 16;
  constexpr int CODE_BYTES = D / 2, PAIR_BYTES = D / 16;
  constexpr int OFF_V = TR * CODE_BYTES, OFF_KA = 2 * OFF_V, OFF_VA = OFF_KA + TR * PAIR_BYTES;
  constexpr int SLOT = OFF_VA + TR * PAIR_BYTES;
  static_assert(SLOT * STAGES >= (8 * D + 16) * 4, "the states of a warp go over its ring");
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % p.splits, bh = blockIdx.x / p.splits;
  const int b = bh / p.Hkv, h = bh - b * p.Hkv, G = p.Hq / p.Hkv;
  uint8_t* ring = smem + warp * (SLOT * STAGES);
  const uint32_t ring_s = b200::smem_u32(ring);

  b200::pdl_launch_dependents();
  b200::pdl_wait();
  const int capacity = p.pages * p.page_rows;
  const int first = p.lo ? max(p.lo[b], 0) : 0;
  const int end = min(p.lengths[b], capacity);
  const int tile_lo = first / TR, tile_hi = end > first ? (end + TR - 1) / TR : tile_lo;
  const int per = (tile_hi - tile_lo + p.splits - 1) / p.splits;
  const int t_begin = tile_lo + split * per, t_end = min(t_begin + per, tile_hi);
  const bool whole = p.page_rows % TR == 0;    // a tile never leaves its page

  auto fill = [&](int tile, int slot) {
    if (tile < t_end) {
      const uint32_t dst = ring_s + slot * SLOT;
      const int r0 = tile * TR;
      const int pg0 = r0 / p.page_rows, in0 = r0 - pg0 * p.page_rows;
      auto pool_row = [&](int j) {    // of row r0 + j
        int pg = pg0, in = in0 + j;
        if (!whole) {
          pg = (r0 + j) / p.page_rows;
          in = r0 + j - pg * p.page_rows;
        }
        return ((static_cast<long long>(b) * p.pages + pg) * p.Hkv + h) * p.page_rows + in;
      };
      constexpr int CHUNKS = CODE_BYTES / 16, ROWS = 32 / CHUNKS;
      const int c = lane % CHUNKS;
#pragma unroll
      for (int j0 = 0; j0 < TR; j0 += ROWS) {
        const int j = j0 + lane / CHUNKS;
        if (r0 + j >= first && r0 + j < end) {
          const long long src = pool_row(j) * CODE_BYTES + c * 16;
          const uint32_t to = dst + j * CODE_BYTES + ((D == 128 ? c ^ (j & 2) : c) * 16);
          cp_async16(to, p.k_codes + src);
          cp_async16(to + OFF_V, p.v_codes + src);
        }
      }
#pragma unroll
      for (int j0 = 0; j0 < TR; j0 += 32) {
        const int j = j0 + lane;
        if (j < TR && r0 + j >= first && r0 + j < end) {
          const long long src = pool_row(j) * PAIR_BYTES;
          cp_async_small<PAIR_BYTES>(dst + OFF_KA + j * PAIR_BYTES, p.k_affine + src);
          cp_async_small<PAIR_BYTES>(dst + OFF_VA + j * PAIR_BYTES, p.v_affine + src);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fill(t_begin + warp + i * WARPS, i);

  // queries: column g of the first product is head g (WIDE) or g % 4, whose second copy gives the low parts of p s
  uint32_t qf[KW][4];
  float qsum[GROUPS][2] = {};
  {
    const int hq = WIDE ? g : (g & 3);
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      const int c = D == 128 ? 64 * (j & 1) + 16 * t + 8 * (j >> 1) : 16 * t + 8 * j;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (hq < G) v = *reinterpret_cast<const uint4*>(p.q + b * p.q_batch + static_cast<long long>(h * G + hq) * D + c);
      qf[j][0] = v.x, qf[j][1] = v.y, qf[j][2] = v.z, qf[j][3] = v.w;
    }
#pragma unroll
    for (int gr = 0; gr < GROUPS; ++gr) {
      float c[4] = {};
#pragma unroll
      for (int j = 0; j < KW; ++j)
        if (GROUPS == 1 || (j & 1) == gr) {
          mma(c, kOnes, kOnes, kOnes, kOnes, qf[j][0], qf[j][1]);
          mma(c, kOnes, kOnes, kOnes, kOnes, qf[j][2], qf[j][3]);
        }
      qsum[gr][0] = c[0], qsum[gr][1] = c[1];
    }
  }

  const int pi = (g & 1) ? 7 - (g >> 1) : g >> 1;
  const float low = (!WIDE && t >= 2) ? 1.f : 0.f;
  float o[GROUPS * 4][4] = {}, zacc[GROUPS][2] = {}, m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {};
  int i = 0;
  for (int tile = t_begin + warp; tile < t_end; tile += WARPS, ++i) {
    cp_async_wait<STAGES - 2>();
    __syncwarp();
    fill(tile + (STAGES - 1) * WARPS, (i + STAGES - 1) % STAGES);
    const uint8_t* slot = ring + (i % STAGES) * SLOT;
    const int r0 = tile * TR;
    const bool edge = r0 < first || r0 + TR > end;

    float sc[STEPS][4];
#pragma unroll
    for (int mt = 0; mt < STEPS; ++mt) {
      const int ja = 16 * mt + pi, jb = ja + 8;
      uint32_t ka[KW], kb[KW], aa[GROUPS], ab[GROUPS];
      if constexpr (D == 128) {
        const uint4 va = *reinterpret_cast<const uint4*>(slot + ja * 64 + ((t ^ (ja & 2)) * 16));
        const uint4 vb = *reinterpret_cast<const uint4*>(slot + jb * 64 + ((t ^ (jb & 2)) * 16));
        ka[0] = va.x, ka[1] = va.y, ka[2] = va.z, ka[3] = va.w;
        kb[0] = vb.x, kb[1] = vb.y, kb[2] = vb.z, kb[3] = vb.w;
        const uint2 pa = *reinterpret_cast<const uint2*>(slot + OFF_KA + ja * 8);
        const uint2 pb = *reinterpret_cast<const uint2*>(slot + OFF_KA + jb * 8);
        aa[0] = pa.x, aa[1] = pa.y, ab[0] = pb.x, ab[1] = pb.y;
      } else {
        const uint2 va = *reinterpret_cast<const uint2*>(slot + ja * 32 + t * 8);
        const uint2 vb = *reinterpret_cast<const uint2*>(slot + jb * 32 + t * 8);
        ka[0] = va.x, ka[1] = va.y, kb[0] = vb.x, kb[1] = vb.y;
        aa[0] = *reinterpret_cast<const uint32_t*>(slot + OFF_KA + ja * 4);
        ab[0] = *reinterpret_cast<const uint32_t*>(slot + OFF_KA + jb * 4);
      }
      float acc[GROUPS][4];
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[gr][c] = -128.f * qsum[gr][c & 1];
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        float(&a)[4] = acc[GROUPS == 1 ? 0 : (j & 1)];
        mma(a, coded<0>(ka[j]), coded<0>(kb[j]), coded<1>(ka[j]), coded<1>(kb[j]), qf[j][0], qf[j][1]);
        mma(a, coded<2>(ka[j]), coded<2>(kb[j]), coded<3>(ka[j]), coded<3>(kb[j]), qf[j][2], qf[j][3]);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float s = 0.f;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) {
          const uint32_t a = c < 2 ? aa[gr] : ab[gr];
          s = fmaf(scale_of(a), acc[gr][c], fmaf(least_of(a), qsum[gr][c & 1], s));
        }
        sc[mt][c] = s * p.scale_log2;
      }
      if (edge) {
        const bool seen_a = r0 + ja >= first && r0 + ja < end, seen_b = r0 + jb >= first && r0 + jb < end;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (!(c < 2 ? seen_a : seen_b)) sc[mt][c] = -CUDART_INF_F;
      }
    }

    float alpha[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float mx = m[e];
#pragma unroll
      for (int mt = 0; mt < STEPS; ++mt) mx = fmaxf(mx, fmaxf(sc[mt][e], sc[mt][e + 2]));
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float use = mx == -CUDART_INF_F ? 0.f : mx;
      alpha[e] = b200::ex2_approx(m[e] - use);
      m[e] = mx;
      float sum = 0.f;
#pragma unroll
      for (int mt = 0; mt < STEPS; ++mt) {
        sc[mt][e] = b200::ex2_approx(sc[mt][e] - use);
        sc[mt][e + 2] = b200::ex2_approx(sc[mt][e + 2] - use);
        sum += sc[mt][e] + sc[mt][e + 2];
      }
      l[e] = fmaf(l[e], alpha[e], sum);
    }

    // p s in two parts, as the column operand of the second product
    uint32_t bh_[GROUPS][STEPS][2], bl_[WIDE ? GROUPS : 1][STEPS][2];
#pragma unroll
    for (int gr = 0; gr < GROUPS; ++gr) zacc[gr][0] *= alpha[0], zacc[gr][1] *= alpha[1];
#pragma unroll
    for (int mt = 0; mt < STEPS; ++mt) {
      const int ja = 16 * mt + pi, jb = ja + 8;
      uint32_t aa[GROUPS], ab[GROUPS];
      if constexpr (D == 128) {
        const uint2 pa = *reinterpret_cast<const uint2*>(slot + OFF_VA + ja * 8);
        const uint2 pb = *reinterpret_cast<const uint2*>(slot + OFF_VA + jb * 8);
        aa[0] = pa.x, aa[1] = pa.y, ab[0] = pb.x, ab[1] = pb.y;
      } else {
        aa[0] = *reinterpret_cast<const uint32_t*>(slot + OFF_VA + ja * 4);
        ab[0] = *reinterpret_cast<const uint32_t*>(slot + OFF_VA + jb * 4);
      }
      if (edge) {
        const bool seen_a = r0 + ja >= first && r0 + ja < end, seen_b = r0 + jb >= first && r0 + jb < end;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) {
          if (!seen_a) aa[gr] = 0;
          if (!seen_b) ab[gr] = 0;
        }
      }
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) {
        const float sa = scale_of(aa[gr]), sb = scale_of(ab[gr]);
        const float za = fmaf(8.f, sa, least_of(aa[gr])), zb = fmaf(8.f, sb, least_of(ab[gr]));
        zacc[gr][0] = fmaf(sc[mt][0], za, fmaf(sc[mt][2], zb, zacc[gr][0]));
        zacc[gr][1] = fmaf(sc[mt][1], za, fmaf(sc[mt][3], zb, zacc[gr][1]));
        const float u[4] = {sc[mt][0] * sa, sc[mt][1] * sa, sc[mt][2] * sb, sc[mt][3] * sb};
        float rest[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float hi = __uint_as_float(__float_as_uint(u[c]) & 0xffff0000u);
          rest[c] = WIDE ? u[c] - hi : fmaf(-low, hi, u[c]);
        }
        if constexpr (WIDE) {
          bh_[gr][mt][0] = transpose8(__byte_perm(__float_as_uint(u[0]), __float_as_uint(u[1]), 0x7632));
          bh_[gr][mt][1] = transpose8(__byte_perm(__float_as_uint(u[2]), __float_as_uint(u[3]), 0x7632));
          bl_[gr][mt][0] = transpose8(__byte_perm(__float_as_uint(rest[0]), __float_as_uint(rest[1]), 0x7632));
          bl_[gr][mt][1] = transpose8(__byte_perm(__float_as_uint(rest[2]), __float_as_uint(rest[3]), 0x7632));
        } else {
          bh_[gr][mt][0] = transpose8(__byte_perm(__float_as_uint(rest[0]), __float_as_uint(rest[1]), 0x7632));
          bh_[gr][mt][1] = transpose8(__byte_perm(__float_as_uint(rest[2]), __float_as_uint(rest[3]), 0x7632));
        }
      }
    }
    // a tile's sums start at -136 sum p s and are added to the running ones in fp32
    float acc[GROUPS * 4][4];
#pragma unroll
    for (int gr = 0; gr < GROUPS; ++gr) {
      float c[4] = {};
#pragma unroll
      for (int mt = 0; mt < STEPS; ++mt) {
        mma(c, kOnes, kOnes, kOnes, kOnes, bh_[gr][mt][0], bh_[gr][mt][1]);
        if constexpr (WIDE) mma(c, kOnes, kOnes, kOnes, kOnes, bl_[gr][mt][0], bl_[gr][mt][1]);
      }
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[gr * 4 + v][e] = -136.f * c[e & 1];
    }
#pragma unroll
    for (int mt = 0; mt < STEPS; ++mt) {
      uint32_t w[4][GROUPS];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = 16 * mt + (k >> 1) * 8 + ((k & 1) ? 7 - t : t);
        const uint8_t* row = slot + OFF_V + j * CODE_BYTES;
        if constexpr (D == 128) {
          const uint2 v = *reinterpret_cast<const uint2*>(row + (((g >> 1) ^ (j & 2)) * 16 + (g & 1) * 8));
          w[k][0] = v.x, w[k][1] = v.y;
        } else {
          w[k][0] = *reinterpret_cast<const uint32_t*>(row + g * 4);
        }
      }
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) {
        const uint32_t a0 = __byte_perm(w[0][gr], w[1][gr], 0x5410), a1 = __byte_perm(w[0][gr], w[1][gr], 0x7632);
        const uint32_t a2 = __byte_perm(w[2][gr], w[3][gr], 0x5410), a3 = __byte_perm(w[2][gr], w[3][gr], 0x7632);
        auto step = [&](float(&c)[4], uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3) {
          mma(c, x0, x1, x2, x3, bh_[gr][mt][0], bh_[gr][mt][1]);
          if constexpr (WIDE) mma(c, x0, x1, x2, x3, bl_[gr][mt][0], bl_[gr][mt][1]);
        };
        step(acc[gr * 4 + 0], coded<0>(a0), coded<0>(a1), coded<0>(a2), coded<0>(a3));
        step(acc[gr * 4 + 1], coded<1>(a0), coded<1>(a1), coded<1>(a2), coded<1>(a3));
        step(acc[gr * 4 + 2], coded<2>(a0), coded<2>(a1), coded<2>(a2), coded<2>(a3));
        step(acc[gr * 4 + 3], coded<3>(a0), coded<3>(a1), coded<3>(a2), coded<3>(a3));
      }
    }
#pragma unroll
    for (int v = 0; v < GROUPS * 4; ++v)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[v][e] = fmaf(o[v][e], alpha[e & 1], acc[v][e]);
  }
  cp_async_wait<0>();
  __syncwarp();

  // the warp's state over its ring: o [8][D], m [8], l [8]
  float* st = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], off);
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) zacc[gr][e] += __shfl_xor_sync(0xffffffffu, zacc[gr][e], off);
    }
    if (g == 0) {
      st[8 * D + 2 * t + e] = m[e];
      st[8 * D + 8 + 2 * t + e] = l[e];
    }
#pragma unroll
    for (int gr = 0; gr < GROUPS; ++gr) {
      const float z = low == 0.f ? zacc[gr][e] : 0.f;
#pragma unroll
      for (int v = 0; v < 4; ++v)
        *reinterpret_cast<float2*>(st + (2 * t + e) * D + 64 * gr + 8 * g + 2 * v) =
            make_float2(o[gr * 4 + v][e] + z, o[gr * 4 + v][e + 2] + z);
    }
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < G * D; idx += WARPS * 32) {
    const int hq = idx / D, d = idx - hq * D;
    float mm = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, reinterpret_cast<const float*>(smem + w * (SLOT * STAGES))[8 * D + hq]);
    float sum = 0.f, ls = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float* s = reinterpret_cast<const float*>(smem + w * (SLOT * STAGES));
      const float mw = s[8 * D + hq], lw = s[8 * D + 8 + hq];
      // a warp that saw no row has l = 0; one that saw no number has m = -inf and l = NaN, which counts
      const float wgt = mw == -CUDART_INF_F ? (lw == 0.f ? 0.f : 1.f) : b200::ex2_approx(mw - mm);
      float v = s[hq * D + d];
      if constexpr (!WIDE) v += s[(hq + 4) * D + d];
      sum = fmaf(v, wgt, sum);
      ls = fmaf(lw, wgt, ls);
    }
    const long long head = static_cast<long long>(b) * p.Hq + h * G + hq;
    if (p.splits == 1) {
      p.out[head * D + d] = __float2bfloat16(end > first ? sum / ls : 0.f);
    } else {
      p.part_o[(head * p.splits + split) * D + d] = sum;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (head * p.splits + split) * 2) = make_float2(mm, ls);
    }
  }
}

// Joins the splits of a head, as above.
template <int D>
__global__ void __launch_bounds__(D) decode_q4_merge_kernel(const __grid_constant__ AttnParams p) {
  const long long head = blockIdx.x;
  const int d = threadIdx.x;
  b200::pdl_launch_dependents();
  b200::pdl_wait();
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + head * p.splits;
  const float* part = p.part_o + head * p.splits * D + d;
  float mm = -CUDART_INF_F, sum = 0.f, ls = 0.f;
  bool any = false;
  for (int s = 0; s < p.splits; ++s) mm = fmaxf(mm, ml[s].x);
  for (int s = 0; s < p.splits; ++s) {
    const float2 v = ml[s];
    const bool none = v.x == -CUDART_INF_F && v.y == 0.f;
    const float wgt = v.x == -CUDART_INF_F ? (none ? 0.f : 1.f) : b200::ex2_approx(v.x - mm);
    any = any || !none;
    sum = fmaf(part[static_cast<long long>(s) * D], wgt, sum);
    ls = fmaf(v.y, wgt, ls);
  }
  p.out[head * D + d] = __float2bfloat16(any ? sum / ls : 0.f);
}

constexpr int kWarps = 4, kRows = 64, kStages = 3;

template <int D, bool WIDE>
int launch(const AttnParams& p, cudaStream_t s) {
  constexpr int bytes = kWarps * kStages * kRows * (D + D / 8);
  auto* kern = decode_q4_kernel<D, WIDE, kWarps, kRows, kStages>;
  static bool configured[b200host::kMaxDevices] = {};
  if (int rc = b200host::ensure_dynamic_smem(kern, bytes, configured)) return rc;
  const bool pdl = b200host::pdl_enabled() != 0;
  if (cudaError_t e = b200host::launch_kernel(kern, dim3(p.B * p.Hkv * p.splits), dim3(kWarps * 32), bytes, s, pdl, p))
    return static_cast<int>(e);
  if (p.splits == 1) return 0;
  return static_cast<int>(b200host::launch_kernel(decode_q4_merge_kernel<D>, dim3(p.B * p.Hq), dim3(D), 0, s, pdl, p));
}

}  // namespace

// Parts that a sequence's rows are cut into: as many as give each SM two blocks, of at least a tile a warp.
extern "C" int b200_q4_decode_attn_splits(int B, int Hkv, long long rows) {
  const long long base = (long long)B * Hkv, tiles = (rows + kRows - 1) / kRows;
  long long splits = base > 0 ? 2 * b200host::sm_count() / base : 1;
  if (splits > (tiles + kWarps - 1) / kWarps) splits = (tiles + kWarps - 1) / kWarps;
  if (splits > 64) splits = 64;
  return splits < 1 ? 1 : (int)splits;
}

// q [B, Hq, D] bf16 (q_batch elements between sequences), caches [B, pages, Hkv, page_rows, ..] contiguous, lengths and lo
// int32 [B] (lo may be null), out [B, Hq, D] bf16.  D 64 or 128, up to 8 query heads to a K/V head.  With more than one
// split: part_o [B, Hq, splits, D] and part_ml [B, Hq, splits, 2] fp32 of the call's own.
extern "C" int b200_q4_decode_attn(const void* q, long long q_batch, const void* k_codes, const void* k_affine,
                                   const void* v_codes, const void* v_affine, const void* lengths, const void* lo,
                                   void* out, void* part_o, void* part_ml, int B, int Hq, int Hkv, int D, int pages,
                                   int page_rows, int splits, float scale, void* stream) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > 8 || pages <= 0 || page_rows <= 0 || (D != 64 && D != 128) ||
      splits < 1 || (long long)pages * page_rows > 0x7fffff00ll || (long long)B * Hq * splits > 0x7fffffffll ||
      (splits > 1 && (!part_o || !part_ml)))
    return b200host::RC_BAD_SHAPE;
  if ((q_batch & 7) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_codes) |
                         reinterpret_cast<uintptr_t>(k_affine) | reinterpret_cast<uintptr_t>(v_codes) |
                         reinterpret_cast<uintptr_t>(v_affine) | reinterpret_cast<uintptr_t>(out)) & 15))
    return b200host::RC_BAD_ALIGNMENT;
  AttnParams p{(const __nv_bfloat16*)q, q_batch, (const uint8_t*)k_codes, (const uint8_t*)k_affine,
               (const uint8_t*)v_codes, (const uint8_t*)v_affine, (const int*)lengths, (const int*)lo,
               (__nv_bfloat16*)out, (float*)part_o, (float*)part_ml, B, Hq, Hkv, pages, page_rows, splits,
               scale * kLog2e};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool wide = Hq / Hkv > 4;
  if (D == 128) return wide ? launch<128, true>(p, s) : launch<128, false>(p, s);
  return wide ? launch<64, true>(p, s) : launch<64, false>(p, s);
}

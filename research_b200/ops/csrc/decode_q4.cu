// Attention of one new token per sequence over a K/V cache held in 4 bits (quant4.cuh), head-major pages of any size.
//   o[h] = sum_r p_r (s n_r + z) / sum_r p_r,  p = softmax(scale * q . (s n + z)),  rows max(lo, 0) <= r < min(len, capacity)
// A sequence without such a row gets zeros.
//
// Every cached row is read once for all query heads that share it.  A row of 128 has 72 bytes instead of 256, so what would
// be a stream for the memory becomes work for the SM: at the copy bandwidth 46 codes a clock and SM, too many for an FMA per
// code and head.  Both products therefore go through the tensor cores as m16n8k16 with the cache as the 16-row operand and
// up to eight query heads as the columns (a tcgen05 product would want the expanded rows in shared or tensor memory first,
// and its 128 x 16 tile has no more use for eight columns).  The bits 0 .. 255 are, as bf16, the numbers i 2^-133 (subnormals
// and the first binade are one straight line), so that a code needs no more than to be masked out: n at the low end of a
// half word, 16 n four bits further up, one shift for the word's other four.  The other operands make up for the size: queries
// are brought to 2^126 by a power of two of their head's own (and divided by 16 where the code is not), weights times scales
// to 2^100 by one that follows the largest scale.  Scales and least values are applied to the sums in fp32:
//   q . k_r = sum_groups s_r (sum q n) + z_r sum q
//   o       = sum_r (p_r s_r) n_r + sum_r p_r z_r
// p s enters the second product as two bf16 parts (up to four heads: in columns 4 .. 7 of the same product, else in a
// second one): the first is cut off, what it leaves is exact and below 2^-7 of the weight, and the second is that, rounded to
// 2^-8 of itself, to either side.  (Cut off as well, it takes 2^-17 from every weight on average, which shows in a result
// whose two sums nearly cancel: 64 sequences of 512 .. 4096 rows were 6e-4 away from the same in fp32, and are 7e-5 away;
// the rounding costs 1 to 2 % of the time.  A single bf16 would cost as much as the rounding of the result does.)
//
// Measured (inputs of several sets in turn, larger than L2), heads of 128: 64 sequences of 512 .. 4096 rows, 16 heads over 8,
// 47.6 us, of 16384 rows 139.9 us, 75 % of the copy bandwidth; 2 sequences of 32768 rows, 32 heads over 8, 22.0 us; one of 777
// rows 7.6 us, which are two launches and one tile's latency.  No unit is full (59 % of the issue slots, 58 % of the DRAM rate at
// 16384 rows): twelve warps an SM with one tile under way each wait for latency.  With codes as 128 + n (a second operation
// each, and the 128 taken off again) and a maximum followed tile by tile the first took 53 us.  That and the other comparisons
// below were taken with both parts of p s cut off.
#include <math.h>
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
  float *part_o, *part_ml;            // [slots, G, D], [slots, G, 2]: (m in log2 units, l)
  int B, Hq, Hkv, pages, page_rows, warps;
  float scale_log2;                   // above zero: a negative scale changes the queries' sign, one of zero leaves zeros of them
  uint32_t q_keep, q_flip;            // bits of two bf16
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
// the first product of a chain
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// 2^e, e clamped to what fp32 has as normal numbers
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(min(max(e, -126), 127) + 127) << 23); }

// codes 0 and 1 (of four) of each half of a word as bf16: n 2^-133 and 16 n 2^-133
__device__ __forceinline__ uint32_t low_codes(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t high_codes(uint32_t w) { return w & 0x00f000f0u; }

// Rows of sequence b that count: [first, end), in tiles of TR rows from tile_lo to tile_hi (none: tile_lo = tile_hi).
template <int TR>
struct Span {
  int first, end, tile_lo, tile_hi;
  __device__ __forceinline__ Span(const AttnParams& p, int b) {
    first = p.lo ? max(p.lo[b], 0) : 0;
    end = min(p.lengths[b], p.pages * p.page_rows);
    tile_lo = end > first ? first / TR : 0;
    tile_hi = end > first ? (end + TR - 1) / TR : 0;
  }
  __device__ __forceinline__ int tiles() const { return tile_hi - tile_lo; }
};

// The tiles of all (sequence, K/V head) pairs in their order are dealt to the warps of the grid in equal runs, so that ragged
// lengths leave no SM behind.  Warp i has tiles [i * share, (i + 1) * share); what it finds for pair bh goes to slot i + bh,
// which no other run and pair have (in that order either the warp or the pair goes up from one piece to the next).
struct Deal {
  long long total, share;
  __device__ __forceinline__ Deal(long long tiles, int warps) : total(tiles) {
    // the 64-bit quotient only where there are that many tiles
    share = tiles + warps <= 0x7fffffff ? (static_cast<int>(tiles) + warps - 1) / warps : (tiles + warps - 1) / warps;
  }
  __device__ __forceinline__ int run_of(long long tile) const {
    return total <= 0x7fffffff ? static_cast<int>(tile) / static_cast<int>(share) : static_cast<int>(tile / share);
  }
};

// Where a warp is: tile `tile` of pair (b, h).
template <int TR>
struct Cursor {
  int b, h, tile, first, end, tile_lo, tile_hi;
  __device__ __forceinline__ void load(const AttnParams& p) {
    const Span<TR> s(p, b);
    first = s.first, end = s.end, tile_lo = s.tile_lo, tile_hi = s.tile_hi;
  }
  __device__ __forceinline__ void next(const AttnParams& p) {
    if (++tile < tile_hi) return;
    if (++h == p.Hkv) {
      h = 0;
      do {
        if (++b >= p.B) return;
        load(p);
      } while (tile_lo == tile_hi);
    }
    tile = tile_lo;
  }
};

// A warp works by itself: it brings tiles of TR rows into a ring of its own in shared memory (cp.async, so pages may end
// anywhere) and keeps the state of a pair's heads in registers until its run leaves the pair.
//
// Fragments.  Lane (g, t) = (lane / 4, lane % 4).  In the products over the channels row m of the 16 is cache row pi(m) of the
// tile, pi(2 j) = j, pi(2 j + 1) = 7 - j (+ 8 for m >= 8): the lane's rows in the second product, whose index runs over the
// cache rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9, are then t, 7 - t, 8 + t, 15 - t, and neither product's reads from shared
// memory meet in a bank (rows of 128 with their 16-byte chunks swapped in pairs every second pair of rows).
template <int D, bool WIDE, int WARPS, int TR, int STAGES, int BLOCKS>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS) decode_q4_kernel(const __grid_constant__ AttnParams p) {
  constexpr int GROUPS = D / 64, KW = D / 32, STEPS = TR / 16;
  constexpr int CODE_BYTES = D / 2, PAIR_BYTES = D / 16;
  constexpr int OFF_V = TR * CODE_BYTES, OFF_KA = 2 * OFF_V, OFF_VA = OFF_KA + TR * PAIR_BYTES;
  constexpr int SLOT = OFF_VA + TR * PAIR_BYTES;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = p.Hq / p.Hkv;
  uint8_t* ring = smem + warp * (SLOT * STAGES);
  const uint32_t ring_s = b200::smem_u32(ring);

  // the dependent (the kernel below) may read the lengths before its own wait, so it is let in after this one
  b200::pdl_wait();
  b200::pdl_launch_dependents();
  // neighbouring runs go to different blocks, so that few tiles spread over the SMs
  const int run = warp * gridDim.x + blockIdx.x;
  const Span<TR> near(p, min(lane, p.B - 1));
  long long tiles = lane < p.B ? near.tiles() : 0;
  for (int b = lane + 32; b < p.B; b += 32) tiles += Span<TR>(p, b).tiles();
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, off);
  const Deal deal(tiles * p.Hkv, p.warps);
  const long long begin = run * deal.share;
  if (run >= p.warps || begin >= deal.total) return;
  const int count = static_cast<int>(min(deal.share, deal.total - begin));
  Cursor<TR> at;
  {
    long long before = 0;     // tiles of one head of the sequences before the 32 looked at
    for (int b0 = 0;; b0 += 32) {
      const Span<TR> span = b0 ? Span<TR>(p, min(b0 + lane, p.B - 1)) : near;
      const int n = b0 + lane < p.B ? span.tiles() : 0;
      long long sum = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += up;
      }
      const unsigned past = __ballot_sync(0xffffffffu, (before + sum) * p.Hkv > begin);
      if (past) {             // always in the last 32 at the latest: begin is below the total
        const int which = __ffs(past) - 1;
        const long long rest = begin - (before + __shfl_sync(0xffffffffu, sum - n, which)) * p.Hkv;
        at.b = b0 + which;
        at.first = __shfl_sync(0xffffffffu, span.first, which);
        at.end = __shfl_sync(0xffffffffu, span.end, which);
        at.tile_lo = __shfl_sync(0xffffffffu, span.tile_lo, which);
        at.tile_hi = __shfl_sync(0xffffffffu, span.tile_hi, which);
        const int per_head = at.tile_hi - at.tile_lo;
        at.h = static_cast<int>(rest / per_head);
        at.tile = at.tile_lo + static_cast<int>(rest - static_cast<long long>(at.h) * per_head);
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  const bool whole = p.page_rows % TR == 0;    // a tile never leaves its page: its rows are contiguous, and all there

  auto fill = [&](const Cursor<TR>& c, int slot) {
    const uint32_t dst = ring_s + slot * SLOT;
    const int r0 = c.tile * TR;
    constexpr int CHUNKS = CODE_BYTES / 16, ROWS = 32 / CHUNKS;
    const int chunk = lane % CHUNKS, row = lane / CHUNKS;      // of the first copy; the next ones are ROWS rows further
    const uint32_t to = dst + row * CODE_BYTES + ((D == 128 ? chunk ^ (row & 2) : chunk) * 16);
    if (whole) {
      const int pg = r0 / p.page_rows;
      const long long r = ((static_cast<long long>(c.b) * p.pages + pg) * p.Hkv + c.h) * p.page_rows + (r0 - pg * p.page_rows);
      const uint8_t *k = p.k_codes + r * CODE_BYTES + lane * 16, *v = p.v_codes + r * CODE_BYTES + lane * 16;
#pragma unroll
      for (int j = 0; j < TR / ROWS; ++j) {
        cp_async16(to + j * 512, k + j * 512);
        cp_async16(to + OFF_V + j * 512, v + j * 512);
      }
      const uint8_t *ka = p.k_affine + (r + lane) * PAIR_BYTES, *va = p.v_affine + (r + lane) * PAIR_BYTES;
#pragma unroll
      for (int j = 0; j < TR; j += 32) {
        cp_async_small<PAIR_BYTES>(dst + OFF_KA + (j + lane) * PAIR_BYTES, ka + j * PAIR_BYTES);
        cp_async_small<PAIR_BYTES>(dst + OFF_VA + (j + lane) * PAIR_BYTES, va + j * PAIR_BYTES);
      }
    } else {
      auto pool_row = [&](int r) {
        const int pg = r / p.page_rows;
        return ((static_cast<long long>(c.b) * p.pages + pg) * p.Hkv + c.h) * p.page_rows + (r - pg * p.page_rows);
      };
#pragma unroll 2
      for (int j = 0; j < TR / ROWS; ++j) {
        const int r = r0 + row + j * ROWS;
        if (r >= c.first && r < c.end) {
          const long long src = pool_row(r) * CODE_BYTES + chunk * 16;
          cp_async16(to + j * 512, p.k_codes + src);
          cp_async16(to + OFF_V + j * 512, p.v_codes + src);
        }
      }
#pragma unroll
      for (int j = lane; j < TR; j += 32) {
        const int r = r0 + j;
        if (r >= c.first && r < c.end) {
          const long long src = pool_row(r) * PAIR_BYTES;
          cp_async_small<PAIR_BYTES>(dst + OFF_KA + j * PAIR_BYTES, p.k_affine + src);
          cp_async_small<PAIR_BYTES>(dst + OFF_VA + j * PAIR_BYTES, p.v_affine + src);
        }
      }
    }
  };
  Cursor<TR> ahead = at;
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (i < count) {
      fill(ahead, i);
      ahead.next(p);
    }
    cp_async_commit();
  }

  const int pi = (g & 1) ? 7 - (g >> 1) : g >> 1;
  const float low = (!WIDE && t >= 2) ? 1.f : 0.f;
  const uint32_t half = (!WIDE && t >= 2) ? 0x8000u : 0u;     // of a low part's last place as bf16
  uint32_t qf[KW][4];
  float qsum[GROUPS][2], scale[2], before[2];  // sums of q, and log2(e) times the scale, in the units of the first product
  bool huge = false;                           // queries of 2^113 and more: the scale is in two factors
  float o[GROUPS * 4][4], zacc[GROUPS][2], m[2], l[2];
  int v_exp = 0;                               // of the largest scale of V so far, about
  float v_up = 1.f, v_limit = -1.f;            // 2^(100 - v_exp), and the scale from which v_exp has to go up
  bool fresh = true;
  for (int i = 0; i < count; ++i) {
    if (fresh) {
      // queries: column g of the first product is head g (WIDE) or g % 4, whose second copy gives the low parts of p s
      fresh = false;
      const int hq = WIDE ? g : (g & 3);
      uint32_t most = 0;                       // exponent bits of the head's largest value
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        const int c = D == 128 ? 64 * (j & 1) + 16 * t + 8 * (j >> 1) : 16 * t + 8 * j;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (hq < G)
          v = *reinterpret_cast<const uint4*>(p.q + at.b * p.q_batch + static_cast<long long>(at.h * G + hq) * D + c);
        qf[j][0] = v.x, qf[j][1] = v.y, qf[j][2] = v.z, qf[j][3] = v.w;
#pragma unroll
        for (int k = 0; k < 4; ++k) most = max(most, max(qf[j][k] & 0x7f80u, (qf[j][k] >> 16) & 0x7f80u));
      }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // q' = q 2^(126 - e): a sum of q' n 2^-133 stands for 2^(7 + e) times itself, of which what is above 2^119 goes to the
      // scores first.  A head with an infinity or a NaN has none; else the factor stays a number above zero, so that a masked
      // row's -inf does.
      const int e = static_cast<int>(most >> 7) - 127;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int ec = __shfl_sync(0xffffffffu, e, 8 * t + 4 * c) + 7;
        const float f = fminf(fmaxf(p.scale_log2 * pow2(min(ec, 119)), 1.17549435e-38f), 3.402823466e38f);
        scale[c] = ec == 135 ? CUDART_NAN_F : f;
        before[c] = pow2(max(ec - 119, 0));
      }
      huge = __any_sync(0xffffffffu, before[0] + before[1] > 2.f);
      // 2^(126 - e) may be more than one factor has room for
      const float up = pow2((126 - e) / 2), up2 = pow2(126 - e - (126 - e) / 2);
#pragma unroll
      for (int j = 0; j < KW; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float f = (k & 1) ? up2 * 0.0625f : up2;
          const uint32_t v = (qf[j][k] & p.q_keep) ^ p.q_flip;
          qf[j][k] = b200::pack_bf16x2(__uint_as_float(v << 16) * up * f, __uint_as_float(v & 0xffff0000u) * up * f);
        }
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) {    // sums of q': the product with a row of ones
        float c[4] = {};
#pragma unroll
        for (int j = 0; j < KW; ++j)
          if (GROUPS == 1 || (j & 1) == gr) {
            mma(c, 0x00010001u, 0x00010001u, 0x00100010u, 0x00100010u, qf[j][0], qf[j][1]);
            mma(c, 0x00010001u, 0x00010001u, 0x00100010u, 0x00100010u, qf[j][2], qf[j][3]);
          }
        qsum[gr][0] = c[0], qsum[gr][1] = c[1];
        zacc[gr][0] = zacc[gr][1] = 0.f;
      }
#pragma unroll
      for (int v = 0; v < GROUPS * 4; ++v)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[v][e] = 0.f;
      m[0] = m[1] = -CUDART_INF_F;
      l[0] = l[1] = 0.f;
    }
    cp_async_wait<STAGES - 2>();
    __syncwarp();
    if (i + STAGES - 1 < count) {
      fill(ahead, (i + STAGES - 1) % STAGES);
      ahead.next(p);
    }
    cp_async_commit();
    const uint8_t* slot = ring + (i % STAGES) * SLOT;
    const int r0 = at.tile * TR, first = at.first, end = at.end;
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
      for (int j = 0; j < KW; ++j) {
        const int gr = GROUPS == 1 ? 0 : (j & 1);
        const uint32_t wa = ka[j] >> 8, wb = kb[j] >> 8;
        if (j < GROUPS)
          mma_first(acc[gr], low_codes(ka[j]), low_codes(kb[j]), high_codes(ka[j]), high_codes(kb[j]), qf[j][0], qf[j][1]);
        else
          mma(acc[gr], low_codes(ka[j]), low_codes(kb[j]), high_codes(ka[j]), high_codes(kb[j]), qf[j][0], qf[j][1]);
        mma(acc[gr], low_codes(wa), low_codes(wb), high_codes(wa), high_codes(wb), qf[j][2], qf[j][3]);
      }
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) {
        const float sa = scale_of(aa[gr]), sb = scale_of(ab[gr]);
        const float za = least_of(aa[gr]), zb = least_of(ab[gr]);
#pragma unroll
        for (int c = 0; c < 4; ++c)
          sc[mt][c] = fmaf(c < 2 ? sa : sb, acc[gr][c],
                           gr ? fmaf(c < 2 ? za : zb, qsum[gr][c & 1], sc[mt][c]) : (c < 2 ? za : zb) * qsum[gr][c & 1]);
      }
      if (edge) {
        const bool seen_a = r0 + ja >= first && r0 + ja < end, seen_b = r0 + jb >= first && r0 + jb < end;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (!(c < 2 ? seen_a : seen_b)) sc[mt][c] = -CUDART_INF_F;
      }
    }

    if (huge) {
#pragma unroll
      for (int mt = 0; mt < STEPS; ++mt)
#pragma unroll
        for (int c = 0; c < 4; ++c) sc[mt][c] *= before[c & 1];
    }
    // Exponentials are taken relative to a reference that follows the maximum only where a score is 2^8 above it (or there
    // is none yet): what they add up to stays far inside fp32, and nothing has to be rescaled for most tiles.
    float top[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[e] = fmaxf(sc[0][e], sc[0][e + 2]);
#pragma unroll
      for (int mt = 1; mt < STEPS; ++mt) top[e] = fmaxf(top[e], fmaxf(sc[mt][e], sc[mt][e + 2]));
    }
    // the largest scale of the tile's V rows, two rows a lane (a scale that is no number counts for nothing here)
    float v_top = 0.f;
#pragma unroll
    for (int k = 0; k < TR / 32; ++k) {
      const int j = lane + 32 * k;
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) {
        const float s = scale_of(*reinterpret_cast<const uint32_t*>(slot + OFF_VA + j * PAIR_BYTES + gr * 4));
        if (!edge || (r0 + j >= first && r0 + j < end)) v_top = fmaxf(v_top, fabsf(s));
      }
    }
    if (__any_sync(0xffffffffu, fmaf(top[0], scale[0], -m[0]) > 8.f || fmaf(top[1], scale[1], -m[1]) > 8.f ||
                                    v_top > v_limit)) {
      v_top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v_top)));
      float down = 1.f;
      if (v_top > v_limit) {                   // weights go up to 2^8, scales to 2^9 above v_exp: far from 2^127 together
        const int now = max(static_cast<int>(__float_as_uint(v_top) >> 23) - 127, -27);
        down = v_limit < 0.f ? 1.f : pow2(v_exp - now);
        v_exp = now;
        v_up = pow2(100 - now);
        v_limit = pow2(now + 9);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = top[e];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        mx = fmaxf(m[e], mx * scale[e]);
        const float alpha = mx == -CUDART_INF_F ? 1.f : b200::ex2_approx(m[e] - mx);
        m[e] = mx;
        l[e] *= alpha;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) zacc[gr][e] *= alpha;
#pragma unroll
        for (int v = 0; v < GROUPS * 4; ++v) o[v][e] *= alpha * down, o[v][e + 2] *= alpha * down;
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float use = m[e] == -CUDART_INF_F ? 0.f : m[e];     // no number yet: nothing but zeros (or NaN) comes out
#pragma unroll
      for (int mt = 0; mt < STEPS; ++mt) {
        sc[mt][e] = b200::ex2_approx(fmaf(sc[mt][e], scale[e], -use));
        sc[mt][e + 2] = b200::ex2_approx(fmaf(sc[mt][e + 2], scale[e], -use));
        l[e] += sc[mt][e] + sc[mt][e + 2];
      }
    }

    // p s in two parts, as the column operand of the second product
    uint32_t bh_[GROUPS][STEPS][2], bl_[WIDE ? GROUPS : 1][STEPS][2];
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
        const float sa = scale_of(aa[gr]) * v_up, sb = scale_of(ab[gr]) * v_up;
        const float za = least_of(aa[gr]), zb = least_of(ab[gr]);
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
          bl_[gr][mt][0] = transpose8(b200::pack_bf16x2(rest[0], rest[1]));
          bl_[gr][mt][1] = transpose8(b200::pack_bf16x2(rest[2], rest[3]));
        } else {
          bh_[gr][mt][0] = transpose8(__byte_perm(__float_as_uint(rest[0]) + half, __float_as_uint(rest[1]) + half, 0x7632));
          bh_[gr][mt][1] = transpose8(__byte_perm(__float_as_uint(rest[2]) + half, __float_as_uint(rest[3]) + half, 0x7632));
        }
      }
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
        step(o[gr * 4 + 0], low_codes(a0), low_codes(a1), low_codes(a2), low_codes(a3));
        step(o[gr * 4 + 1], high_codes(a0), high_codes(a1), high_codes(a2), high_codes(a3));
        step(o[gr * 4 + 2], low_codes(a0 >> 8), low_codes(a1 >> 8), low_codes(a2 >> 8), low_codes(a3 >> 8));
        step(o[gr * 4 + 3], high_codes(a0 >> 8), high_codes(a1 >> 8), high_codes(a2 >> 8), high_codes(a3 >> 8));
      }
    }
    const int b = at.b, h = at.h;
    fresh = i + 1 == count || at.tile + 1 == at.tile_hi;
    at.next(p);
    if (!fresh) continue;
    // the run leaves the pair: its state goes to the pair's slot
    const float v_back = pow2(v_exp);          // and 2^33, or 2^29 where codes were 16 n
    v_limit = -1.f;
    const long long place = static_cast<long long>(run) + static_cast<long long>(b) * p.Hkv + h;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], off);
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) zacc[gr][e] += __shfl_xor_sync(0xffffffffu, zacc[gr][e], off);
      }
      const int hq = WIDE ? 2 * t + e : (2 * t + e) & 3;
      if (g == 0 && low == 0.f && hq < G)
        *reinterpret_cast<float2*>(p.part_ml + (place * G + hq) * 2) = make_float2(m[e], l[e]);
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float back = (v & 1) ? 536870912.f : 8589934592.f;
          float x = o[gr * 4 + v][e] * back * v_back, y = o[gr * 4 + v][e + 2] * back * v_back;
          if constexpr (!WIDE) {      // the low parts are two lanes further
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            y += __shfl_xor_sync(0xffffffffu, y, 2);
          }
          if (low == 0.f && hq < G)
            *reinterpret_cast<float2*>(p.part_o + (place * G + hq) * D + 64 * gr + 8 * g + 2 * v) =
                make_float2(x + zacc[gr][e], y + zacc[gr][e]);
        }
    }
  }
  cp_async_wait<0>();
}

// Joins the pieces of a head: out = sum_i w_i o_i / sum_i w_i l_i, w_i = 2^(m_i - max m); a piece that met no number has
// m = -inf and l = NaN, which counts.  The threads of a channel share the pieces.
template <int D, int TR, int THREADS>
__global__ void __launch_bounds__(THREADS) decode_q4_merge_kernel(const __grid_constant__ AttnParams p) {
  constexpr int PARTS = THREADS / (D / 4), WARPS = THREADS / 32;
  __shared__ long long s_sum[2][WARPS];
  __shared__ float s_max[WARPS], s_w[THREADS], s_l[WARPS];
  __shared__ __align__(16) float s_o[PARTS][D];
  const int b = blockIdx.x / p.Hq, hq = blockIdx.x - b * p.Hq, G = p.Hq / p.Hkv, h = hq / G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  b200::pdl_launch_dependents();
  long long sum[2] = {0, 0};    // tiles of one head: of all sequences, of those before b
  for (int i = threadIdx.x; i < p.B; i += THREADS) {
    const int n = Span<TR>(p, i).tiles();
    sum[0] += n;
    if (i < b) sum[1] += n;
  }
  const int tiles = Span<TR>(p, b).tiles();
  b200::pdl_wait();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], off);
    if (lane == 0) s_sum[k][warp] = sum[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    sum[k] = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) sum[k] += s_sum[k][w];
  }
  const int d = threadIdx.x % (D / 4) * 4, part = threadIdx.x / (D / 4);     // four channels, every PARTS-th piece
  uint2* out = reinterpret_cast<uint2*>(p.out + (static_cast<long long>(b) * p.Hq + hq) * D + d);
  if (tiles == 0) {
    if (part == 0) *out = make_uint2(0, 0);
    return;
  }
  const Deal deal(sum[0] * p.Hkv, p.warps);
  const long long from = sum[1] * p.Hkv + static_cast<long long>(h) * tiles;
  const int first = deal.run_of(from), pieces = deal.run_of(from + tiles - 1) - first + 1;
  const long long place = first + static_cast<long long>(b) * p.Hkv + h;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + place * G + (hq - h * G);
  const float* o = p.part_o + (place * G + (hq - h * G)) * D + d;
  // the first pieces' channels are on their way while the weights are made
  float4 ahead[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    ahead[k] = part + k * PARTS < pieces ? *reinterpret_cast<const float4*>(o + static_cast<long long>(part + k * PARTS) * G * D)
                                         : make_float4(0.f, 0.f, 0.f, 0.f);
  float mm = -CUDART_INF_F;
  float2 mine = make_float2(-CUDART_INF_F, 0.f);
  for (int i = threadIdx.x; i < pieces; i += THREADS) {
    const float2 v = ml[static_cast<long long>(i) * G];
    if (i < THREADS) mine = v;
    mm = fmaxf(mm, v.x);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, off));
  if (lane == 0) s_max[warp] = mm;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, s_max[w]);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  auto add = [&](const float4& v, float w) {
    acc.x = fmaf(v.x, w, acc.x);
    acc.y = fmaf(v.y, w, acc.y);
    acc.z = fmaf(v.z, w, acc.z);
    acc.w = fmaf(v.w, w, acc.w);
  };
  for (int i0 = 0; i0 < pieces; i0 += THREADS) {
    const int n = min(pieces - i0, THREADS);
    if (threadIdx.x < n) {
      const float2 v = i0 ? ml[static_cast<long long>(i0 + threadIdx.x) * G] : mine;
      const float w = v.x == -CUDART_INF_F ? (v.y == 0.f ? 0.f : 1.f) : b200::ex2_approx(v.x - mm);
      s_w[threadIdx.x] = w;
      l = fmaf(v.y, w, l);
    }
    __syncthreads();
    int i = part;
    if (i0 == 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k, i += PARTS)
        if (i < n) add(ahead[k], s_w[i]);
    }
#pragma unroll 4
    for (; i < n; i += PARTS) add(*reinterpret_cast<const float4*>(o + static_cast<long long>(i0 + i) * G * D), s_w[i]);
    __syncthreads();
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
  if (lane == 0) s_l[warp] = l;
  *reinterpret_cast<float4*>(&s_o[part][d]) = acc;
  __syncthreads();
  if (part == 0) {
    l = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) l += s_l[w];
#pragma unroll
    for (int k = 1; k < PARTS; ++k) add(*reinterpret_cast<const float4*>(&s_o[k][d]), 1.f);
    *out = make_uint2(b200::pack_bf16x2(acc.x / l, acc.y / l), b200::pack_bf16x2(acc.z / l, acc.w / l));
  }
}

// Warps of a block, rows of a tile, blocks an SM; the ring takes the shared memory.  64 sequences of 512 .. 4096 / 16384 rows,
// heads of 128: 64 rows and 3 blocks 46.6 / 136.5 us, 2 blocks 48.4 / 144.8, 32 rows and 4 blocks 50.8 / 154.5 (what a tile costs
// besides its rows weighs more than the fourth warp of a scheduler gives).
constexpr int kWarps = 4, kRows = 64, kBlocks = 3;
template <int D>
constexpr int stages() { return D == 128 ? 2 : 4; }

template <int D, bool WIDE>
int launch(const AttnParams& p, cudaStream_t s) {
  constexpr int bytes = kWarps * stages<D>() * kRows * (D + D / 8);
  auto* kern = decode_q4_kernel<D, WIDE, kWarps, kRows, stages<D>(), kBlocks>;
  static bool configured[b200host::kMaxDevices] = {};
  if (int rc = b200host::ensure_dynamic_smem(kern, bytes, configured)) return rc;
  const bool pdl = b200host::pdl_enabled() != 0;
  // fewer runs than the device has blocks: one warp of a block each, on as many SMs
  const int most = kBlocks * b200host::sm_count(), grid = p.warps < most ? p.warps : most;
  if (cudaError_t e = b200host::launch_kernel(kern, dim3(grid), dim3(kWarps * 32), bytes, s, pdl, p)) return static_cast<int>(e);
  // where a head has many pieces, more threads read them at once: 64 heads in 103 or 104 pieces each, both kernels,
  // 256 threads 23.1 us, 512 21.8, 1024 26.0; 7 pieces of 512 heads, 256 threads 46.6 us, and 512 find less room beside the
  // first kernel
  const bool many = p.warps > 32 * p.B * p.Hkv;
  auto* merge = many ? decode_q4_merge_kernel<D, kRows, 512> : decode_q4_merge_kernel<D, kRows, 256>;
  return static_cast<int>(b200host::launch_kernel(merge, dim3(p.B * p.Hq), dim3(many ? 512 : 256), 0, s, pdl, p));
}

}  // namespace

// Runs that the rows are dealt to for a cache of `rows` rows a sequence: one per warp of a wave of blocks, or one
// per tile where that is fewer.
extern "C" int b200_q4_decode_attn_runs(int B, int Hkv, long long rows) {
  const long long tiles = (rows + kRows - 1) / kRows * B * Hkv, most = (long long)kBlocks * b200host::sm_count() * kWarps;
  return (int)(tiles < 1 ? 1 : (tiles < most ? tiles : most));
}

// q [B, Hq, D] bf16 (q_batch elements between sequences), caches [B, pages, Hkv, page_rows, ..] contiguous, lengths and lo
// int32 [B] (lo may be null), out [B, Hq, D] bf16.  D 64 or 128, up to 8 query heads to a K/V head.  `runs` from
// b200_q4_decode_attn_runs (pages * page_rows rows); part_o and part_ml are the call's own: (runs + B * Hkv) * (Hq / Hkv) times
// D and 2 floats.
extern "C" int b200_q4_decode_attn(const void* q, long long q_batch, const void* k_codes, const void* k_affine,
                                   const void* v_codes, const void* v_affine, const void* lengths, const void* lo,
                                   void* out, void* part_o, void* part_ml, int B, int Hq, int Hkv, int D, int pages,
                                   int page_rows, int runs, float scale, void* stream) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > 8 || pages <= 0 || page_rows <= 0 || (D != 64 && D != 128) ||
      runs < 1 || (long long)pages * page_rows > 0x7fffff00ll || (long long)B * Hq > 0x7fffffffll || !part_o || !part_ml)
    return b200host::RC_BAD_SHAPE;
  if (runs > kBlocks * b200host::sm_count() * kWarps) return b200host::RC_BAD_SHAPE;
  if ((q_batch & 7) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) ||
      !rows_aligned(k_codes, k_affine, D) || !rows_aligned(v_codes, v_affine, D))
    return b200host::RC_BAD_ALIGNMENT;
  AttnParams p{(const __nv_bfloat16*)q, q_batch, (const uint8_t*)k_codes, (const uint8_t*)k_affine,
               (const uint8_t*)v_codes, (const uint8_t*)v_affine, (const int*)lengths, (const int*)lo,
               (__nv_bfloat16*)out, (float*)part_o, (float*)part_ml, B, Hq, Hkv, pages, page_rows, runs,
               scale == 0.f ? 1.f : fabsf(scale) * kLog2e, scale == 0.f ? 0u : ~0u, scale < 0.f ? 0x80008000u : 0u};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool wide = Hq / Hkv > 4;
  if (D == 128) return wide ? launch<128, true>(p, s) : launch<128, false>(p, s);
  return wide ? launch<64, true>(p, s) : launch<64, false>(p, s);
}

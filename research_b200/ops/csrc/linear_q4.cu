// y = x W^T with weights held in 4 bits (quant4.cuh): x [rows, K] bf16, W [N, K], y [rows, N] bf16 with fp32 sums.  Up to 16
// rows of x the codes themselves are multiplied, as follows; for more see linear_q4_many_kernel.  (With 16 rows of 28672 x 4096 /
// 2048 x 2048 this one takes 23.7 / 6.3 us, with 17 that one 27.1 / 5.7; this one rounds no weight.)
//
// The time is that of streaming the codes once (0.56 bytes a weight), as long as expanding them keeps up: at the copy
// bandwidth an SM gets 46 codes a clock, which is what the arrangement below is for.  Measured, 1 row: 2048 x 2048 5.6 us, a
// stage's latency; 28672 x 4096 22.4 us, 0.45 of the copy bandwidth, 0.55 us per stage of 256 channels and SM.
//
// The weights are the 128-row operand of tcgen05.mma, from tensor memory, the rows of x its 16 columns, both in e4m3.  The
// bytes 0 .. 15 are, as e4m3, the numbers n 2^-9 (subnormals and the first binade are one straight line), so that a word of
// eight codes becomes eight operands by two masks and a shift, a third of what bf16 operands take, in half the tensor memory.
// A row of x is brought to [128, 256) by a power of two and split into two e4m3 numbers, high + low, which go into one
// accumulator: the eight bits of a bf16 are two times four, so that is exact down to 2^-9 of the row's largest value, and
// below that off by 2^-17 of it at most.  The product of each group is taken by itself.  The sum X_g of x over a group gets
// into every lane as a product too, of fours with 32 e4m3 numbers that add up to a quarter of it (16 times its sixteenth, then
// what is left: to 2^-15 of the row's largest value); scales and least values are applied to both in fp32:
//   y = x_max (sum_g s_g (sum_k x'_k n_k) + z_g X'_g),   x' = x / x_max
// (weights rounded to bf16 instead would cost as much precision again as the result's own rounding; sums and scales of x from
// shared memory, the same word for all lanes, take one pass a word: 16 passes a column and 128 x 128 block, 85 us for 28672 x
// 4096 with 64 rows).  K is cut over the blocks of a cluster, which add up their partial sums in rank order: the same bits
// every time.
//
// Blocks of short slices split x themselves (see kOwnStages); else a first kernel does once for all blocks, while the second
// one, launched as its dependent, brings its first codes into L2.  The second one's warps:
//   warp 0     TMA: 256 channels of codes (128 x 128 bytes) and of the split x through a ring of stages
//   warp 1     MMA issuer: for each group the products with the high and the low parts
//   warps 2-5  a weight row per thread: expand the next half stage's codes, then scale and add up the current one's products
// An SM has up to four such blocks, which wait at different places: roles of their own for expanding and for adding up, in one
// block of 20 warps, took 33 us for 28672 x 4096 with 16 rows, most of it in handing over.
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <math_constants.h>
#include <type_traits>

#include "quant4.cuh"
#include "host_util.cuh"

namespace {

using namespace q4;
using namespace b200;

constexpr int kThreads = 192;
constexpr int kStage = 256;                    // channels of a stage
constexpr int kCodeBytes = 128 * kStage / 2;
constexpr int kMaxStages = 8;
constexpr int kFewRows = 16;                   // up to which the codes themselves are multiplied
// Stages of a slice of x up to which a block splits it itself: with 1 and 16 rows of 2048 x 2048 (one stage) 5.7 and 6.3 us
// instead of 6.4 and 7.0 with the kernel before, and 4 us less on the host.
constexpr int kOwnStages = 2;
constexpr int kFours = 32, kProducts = 48;     // tensor memory: half a stage's codes (128 bytes a row), 32 fours, products
constexpr int ERR_Q4_A = 41, ERR_Q4_D = 42;    // status codes: operands or products that never came

struct LinearParams {
  const uint8_t* affine;
  const float* xs;                    // [rows]: what a row of x was divided by; null: nothing
  __nv_bfloat16* out;
  long long ldo;
  int rows, N, width, cluster, stages, token_tiles;
  int* status;
  const __nv_bfloat16* x;             // where blocks split it themselves: [rows, K], `aligned` where 16 bytes may be read at once
  long long ldx;
  int K, aligned;
};

// D[tmem] (+)= A[tmem] * B[smem], both e4m3, fp32 accumulate; 32 channels
__device__ __forceinline__ void tc_mma_ts_e4m3(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// instruction descriptor: e4m3 operands (format 0), both K-major, fp32 result
__host__ __device__ constexpr uint32_t make_idesc_e4m3(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// A wait that looks a few times without the suspend hint of mbar_wait first: 46 clocks instead of 84 where the phase is
// complete, and no waking up where it is soon.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, const AbortCtx& ab, int code) {
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return mbar_wait(bar, parity, ab, code);
}
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, const AbortCtx& ab, int code) {
  return __all_sync(0xffffffffu, wait(bar, parity, ab, code));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
template <int COLS>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t* r) {
  if constexpr (COLS == 16) {
    tmem_ld_32x32b_x16(taddr, *reinterpret_cast<uint32_t(*)[16]>(r));
  } else {
    tmem_ld_32x32b_x32(taddr, *reinterpret_cast<uint32_t(*)[32]>(r));
  }
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t saddr, uint32_t rank) {
  uint32_t peer;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(peer)
               : "memory");
  return v;
}

constexpr int kStageBytes = kCodeBytes + (2 * 2 + 1) * kFewRows * 128;   // codes; [half][high, low] of x; its sums

// 16 channels of row r from channel c on, zeros where there are none
__device__ __forceinline__ void load16(const __nv_bfloat16* x, long long ldx, int rows, int K, int aligned, int r, int c,
                                       float (&f)[16]) {
  const bool there = r < rows;
  if (there && aligned && c + 16 <= K) {
    const uint4* at = reinterpret_cast<const uint4*>(x + r * ldx + c);
    float lo[8], hi[8];
    unpack_bf16(at[0], lo);
    unpack_bf16(at[1], hi);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = lo[k], f[8 + k] = hi[k];
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) f[k] = there && c + k < K ? __bfloat162float(x[r * ldx + c + k]) : 0.f;
  }
}

// What a row whose largest exponent bits are `most` is multiplied by, and what undoes it: 2^(7 - e) brings the largest to
// [128, 256).  A row with an infinity or a NaN counts as NaN.
__device__ __forceinline__ void row_scale(uint32_t most, float& up, float& back) {
  const int e = max(static_cast<int>(most >> 23), 8);
  up = e == 255 ? CUDART_NAN_F : __uint_as_float(static_cast<uint32_t>(261 - e) << 23);
  back = e == 255 ? CUDART_NAN_F : __uint_as_float(static_cast<uint32_t>(e - 7) << 23);
}

// 16 channels as two e4m3 parts, in the order in which a word's codes fall into its low and its high nibbles: 0 4 1 5 2 6 3 7.
__device__ __forceinline__ void split16(const float (&f)[16], uint4& high, uint4& low) {
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a0 = f[8 * h + order[2 * k]], a1 = f[8 * h + order[2 * k + 1]];
      const __nv_fp8x2_storage_t u = __nv_cvt_float2_to_fp8x2(make_float2(a0, a1), __NV_SATFINITE, __NV_E4M3);
      const __half2 back(__nv_cvt_fp8x2_to_halfraw2(u, __NV_E4M3));
      const __nv_fp8x2_storage_t l =
          __nv_cvt_float2_to_fp8x2(make_float2(a0 - __low2float(back), a1 - __high2float(back)), __NV_SATFINITE, __NV_E4M3);
      if (k & 1) {
        hi[2 * h + (k >> 1)] |= static_cast<uint32_t>(u) << 16;
        lo[2 * h + (k >> 1)] |= static_cast<uint32_t>(l) << 16;
      } else {
        hi[2 * h + (k >> 1)] = u;
        lo[2 * h + (k >> 1)] = l;
      }
    }
  }
  high = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  low = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// A group's sum as 32 e4m3 numbers that add up to a quarter of it: 16 times its sixteenth, then what is left, and zeros.
__device__ __forceinline__ void split_sum(float sum, uint4& first, uint4& second) {
  float rest = sum * 0.25f;
  uint32_t part[5];
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    const float of = k ? rest : rest * 0.0625f;
    const __nv_fp8_storage_t v = __nv_cvt_float_to_fp8(of, __NV_SATFINITE, __NV_E4M3);
    const float back = __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
    rest -= k ? back : 16.f * back;
    part[k] = v;
  }
  const uint32_t all = part[0] * 0x01010101u;
  first = make_uint4(all, all, all, all);
  second = make_uint4(part[1] | part[2] << 8 | part[3] << 16 | part[4] << 24, 0, 0, 0);
}

// x [rows, K] -> xq [high, low][kFewRows][width] e4m3, behind them the groups' sums [kFewRows][width / 64][32], and xs [kFewRows]
// fp32; a block per row.
__global__ void __launch_bounds__(512) linear_q4_split_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, int rows,
                                                              int K, int width, int aligned,
                                                              uint8_t* __restrict__ xq,
                                                              float* __restrict__ xs) {
  __shared__ uint32_t s_most[16];
  const int r = blockIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  uint32_t most = 0;
  for (int c = threadIdx.x * 16; c < width; c += 512 * 16) {
    float f[16];
    load16(x, ldx, rows, K, aligned, r, c, f);
#pragma unroll
    for (int k = 0; k < 16; ++k) most = max(most, __float_as_uint(f[k]) & 0x7f800000u);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 16; ++w) most = max(most, s_most[w]);
  float up, back;
  row_scale(most, up, back);
  if (threadIdx.x == 0) xs[r] = back;
  for (int c0 = 0; c0 < width; c0 += 512 * 16) {
    const int c = c0 + threadIdx.x * 16;       // four threads have a group; beyond the row they have zeros
    float f[16], sum = 0.f;
    load16(x, ldx, rows, K, aligned, r, c, f);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      f[k] *= up;
      sum += f[k];
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (c >= width) continue;                  // no shuffles below
    uint4 high, low;
    split16(f, high, low);
    uint8_t* to = xq + static_cast<long long>(r) * width + c;
    *reinterpret_cast<uint4*>(to) = high;
    *reinterpret_cast<uint4*>(to + static_cast<long long>(kFewRows) * width) = low;
    if ((threadIdx.x & 3) == 0) {
      uint4 first, second;
      split_sum(sum, first, second);
      uint8_t* at = xq + 2ll * kFewRows * width + (static_cast<long long>(r) * width + c) / 2;
      *reinterpret_cast<uint4*>(at) = first;
      *reinterpret_cast<uint4*>(at + 16) = second;
    }
  }
}

// Writes the block's part of the result: weight rows [rank, rank + 1) * 128 / cluster of every token of the tile, from the
// sums red[token][128] of the cluster's blocks, added in rank order.
template <int NT>
__device__ __forceinline__ void finish(float* red, const LinearParams& p, int tile, int tokens0, int rank, int threads) {
  pdl_wait();   // what the output replaces may still be read by the predecessor
  const int width = 128 / p.cluster, vecs = width >> 2;
  const int rows = min(p.rows - tokens0 * NT, NT);
  for (int it = threadIdx.x; it < rows * vecs; it += threads) {
    const int token = it / vecs, nl = rank * width + (it - token * vecs) * 4, n = tile * 128 + nl;
    if (n >= p.N) continue;
    const float* at = red + token * 128 + nl;
    float4 v = *reinterpret_cast<const float4*>(at);
    if (p.cluster > 1) {
      v = ld_cluster4(smem_u32(at), 0);
      for (int r = 1; r < p.cluster; ++r) {
        const float4 w = ld_cluster4(smem_u32(at), r);
        v.x += w.x;
        v.y += w.y;
        v.z += w.z;
        v.w += w.w;
      }
    }
    const float scale = p.xs ? p.xs[tokens0 * NT + token] : 1.f;
    v.x *= scale;
    v.y *= scale;
    v.z *= scale;
    v.w *= scale;
    __nv_bfloat16* dst = p.out + (tokens0 * NT + token) * p.ldo + n;
    if (((p.N | p.ldo) & 3) == 0) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    } else {
      const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) dst[i] = __float2bfloat16(e[i]);
    }
  }
  if (p.cluster > 1) {
    __syncwarp();
    cluster_sync();   // peers may still read this block's sums
  }
}

constexpr int kFewBlocks = 4;                  // an SM, by tensor memory (128 columns each) and shared memory

// SPLIT: x comes split from the kernel before.  Else the block's slice has no more stages than there are slots, and its workers
// split x themselves, with scales of the slice's own: a launch less.
template <bool SPLIT>
__global__ void __launch_bounds__(kThreads, kFewBlocks)
linear_q4_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                 const __grid_constant__ CUtensorMap tmS, const __grid_constant__ LinearParams p) {
  constexpr int NT = kFewRows, STAGE = kStageBytes;
  constexpr int UNIT = 2;                      // groups whose products are there at a time: NT columns, and NT of the fours'
  constexpr int TMEM_COLUMNS = 128;
  static_assert(kProducts + UNIT * 2 * NT <= TMEM_COLUMNS && TMEM_COLUMNS * kFewBlocks <= 512, "tensor memory");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], go[1], done[1];
  __shared__ uint32_t tmem_slot[1];
  __shared__ int abort_word;
  __shared__ float s_back[NT];                 // what undoes a token's scale, where it is the block's own
  pdl_launch_dependents();
  volatile int* abort_flag = &abort_word;
  const AbortCtx ab{abort_flag, p.status};
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = blockIdx.x % p.cluster;
  const int tokens0 = blockIdx.x / p.cluster % p.token_tiles, tile = blockIdx.x / p.cluster / p.token_tiles;
  const int blocks = (p.width + kStage - 1) / kStage, per = (blocks + p.cluster - 1) / p.cluster;
  const int kb0 = rank * per, n_kb = max(min(per, blocks - kb0), 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 4 + 1);             // the warps that read the codes, the MMA
    }
    mbar_init(go, 4);
    mbar_init(done, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLUMNS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  float* red = reinterpret_cast<float*>(smem);   // [token][128], over the ring once everything has been read

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&tmW);
      if (SPLIT) tma_prefetch_desc(&tmX);
      // what runs before may be what writes the weights: they are read after the wait, and only brought into L2 ahead of it
      for (int i = 0; i < min(n_kb, 4); ++i) tma_prefetch_l2_2d(&tmW, (kb0 + i) * (kStage / 2), tile * 128);
      pdl_wait();
      bool ok = true;
      for (int i = 0, s = 0, ph = 1; i < n_kb; ++i) {
        if (!wait(&empty[s], ph, ab, ERR_WAIT_EMPTY)) { ok = false; break; }
        uint8_t* to = smem + s * STAGE;
        mbar_expect_tx(&full[s], SPLIT ? STAGE : kCodeBytes);
        tma_load_2d(to, &tmW, &full[s], (kb0 + i) * (kStage / 2), tile * 128);
        if constexpr (!SPLIT) {
          if (++s == p.stages) s = 0, ph ^= 1;
          continue;
        }
        tma_load_2d(to + kCodeBytes, &tmX, &full[s], (kb0 + i) * kStage, tokens0 * 2 * NT);
        tma_load_2d(to + kCodeBytes + 2 * NT * 128, &tmX, &full[s], (kb0 + i) * kStage + 128, tokens0 * 2 * NT);
        tma_load_2d(to + kCodeBytes + 4 * NT * 128, &tmS, &full[s], (kb0 + i) * (kStage / 2), tokens0 * NT);
        if (++s == p.stages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (!ok) {
        // give copies already in flight time to land before the CTA's shared memory goes away
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc_e4m3(128, NT);
      bool ok = true;
      for (int i = 0, s = 0, ph = 0; i < n_kb && ok; ++i) {
        ok = wait(&full[s], ph, ab, ERR_WAIT_FULL);
        const uint64_t xdesc = make_smem_desc_sw128(smem_u32(smem + s * STAGE + kCodeBytes), 16, 1024);
#pragma unroll
        for (int u = 0; u < 4 / UNIT; ++u) {   // the codes are expanded and the last products have been read
          ok = ok && wait(go, (i * (4 / UNIT) + u) & 1, ab, ERR_Q4_A);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < UNIT; ++h) {
            const int g = u * UNIT + h;        // of the stage's four groups
            tc_mma_ts_e4m3(tmem + kProducts + (h * 2 + 1) * NT, tmem + kFours, xdesc + (uint64_t)((4 * NT * 128 + g * 32) >> 4),
                           idesc, 0u);
#pragma unroll
            for (int k = 0; k < 4; ++k)        // high parts, low parts: two steps of 32 channels each
              tc_mma_ts_e4m3(tmem + kProducts + h * 2 * NT, tmem + (g & 1) * 16 + (k & 1) * 8,
                             xdesc + (uint64_t)((((g >> 1) * 2 + (k >> 1)) * NT * 128 + (g & 1) * 64 + (k & 1) * 32) >> 4),
                             idesc, k != 0 ? 1u : 0u);
          }
          tc_commit(done);
        }
        if (ok) tc_commit(&empty[s]);
        if (++s == p.stages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  } else {
    const int quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lane_sel = static_cast<uint32_t>(quad * 32) << 16;
    const uint2* pairs = reinterpret_cast<const uint2*>(
        p.affine + static_cast<long long>(min(tile * 128 + row, p.N - 1)) * (p.width / 16)) + 2 * kb0;
    const int n_pairs = min(2 * n_kb, p.width / 128 - 2 * kb0);   // of 128 channels; the last stage may have one
    uint32_t r[32];
    // codes of half a stage: rows of 128 bytes, their 16-byte chunks exchanged by row % 8
    auto expand = [&](int s, int half) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint4 w = *reinterpret_cast<const uint4*>(smem + s * STAGE + sw128_offset(row, half * 4 + c));
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {          // word 4 c + k: channels 64 (k & 1) + 8 (2 c + k / 2) ..
          const int at = 16 * (k & 1) + 2 * (2 * c + (k >> 1));
          r[at] = v[k] & 0x0f0f0f0fu;
          r[at + 1] = (v[k] >> 4) & 0x0f0f0f0fu;
        }
      }
    };
    auto hand_over = [&] {                     // what this warp wrote and read of tensor memory is done with
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(go);
    };
    uint64_t y[NT / 2];                        // two rows of x each
#pragma unroll
    for (int c = 0; c < NT / 2; ++c) y[c] = f2_pack(0.f, 0.f);
    {
      uint32_t fours[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) fours[c] = 0x48484848u;
      tmem_st16(tmem + kFours + lane_sel, fours);
    }
    pdl_wait();
    if constexpr (!SPLIT) {
      // PER threads for a token, of which thread q has every PER-th chunk of 16 channels: four neighbours have a group
      constexpr int PER = 128 / NT, MOST = kOwnStages * 16 / PER;
      const int t = threadIdx.x - 64, token = t / PER, q = t % PER;
      float x[MOST][16];
      uint32_t most = 0;
#pragma unroll
      for (int it = 0; it < MOST; ++it) {
        const int c = it * PER + q;
        if (it * PER >= n_kb * 16) break;        // a stage less
        load16(p.x, p.ldx, p.rows, p.K, p.aligned, tokens0 * NT + token, kb0 * kStage + c * 16, x[it]);
#pragma unroll
        for (int k = 0; k < 16; ++k) most = max(most, __float_as_uint(x[it][k]) & 0x7f800000u);
      }
#pragma unroll
      for (int off = 1; off < PER; off <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, off));
      float up, back;
      row_scale(most, up, back);
      if (q == 0) s_back[token] = back;
#pragma unroll
      for (int it = 0; it < MOST; ++it) {
        const int c = it * PER + q, half = c >> 3 & 1;
        if (it * PER >= n_kb * 16) break;
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          x[it][k] *= up;
          sum += x[it][k];
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        uint8_t* to = smem + (c >> 4) * STAGE + kCodeBytes;
        uint4 high, low;
        split16(x[it], high, low);
        *reinterpret_cast<uint4*>(to + half * 2 * NT * 128 + sw128_offset(token, c & 7)) = high;
        *reinterpret_cast<uint4*>(to + half * 2 * NT * 128 + sw128_offset(NT + token, c & 7)) = low;
        if ((q & 3) == 0) {
          uint4 first, second;
          split_sum(sum, first, second);
          *reinterpret_cast<uint4*>(to + 4 * NT * 128 + sw128_offset(token, (c >> 2 & 3) * 2)) = first;
          *reinterpret_cast<uint4*>(to + 4 * NT * 128 + sw128_offset(token, (c >> 2 & 3) * 2 + 1)) = second;
        }
      }
      fence_proxy_async_smem();                  // the first hand-over lets the issuer read it
      asm volatile("bar.sync 1, 128;" ::: "memory");   // and s_back the workers
    }
    uint2 f[2] = {0 < n_pairs ? __ldg(pairs) : make_uint2(0, 0), 1 < n_pairs ? __ldg(pairs + 1) : make_uint2(0, 0)};
    bool ok = true;
    if (n_kb > 0) {
      ok = wait_warp(&full[0], 0, ab, ERR_WAIT_FULL);
      if (ok) {
        expand(0, 0);
        tmem_st_32x32b_x32(tmem + lane_sel, r);
        tmem_st_wait();
        hand_over();
      }
    }
    for (int i = 0, s = 0, ph = 0; i < n_kb && ok; ++i) {
      const int s1 = s + 1 == p.stages ? 0 : s + 1, ph1 = s + 1 == p.stages ? ph ^ 1 : ph;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int j = 2 * i + half;
        const bool more = half == 0 || i + 1 < n_kb;
        const uint2 pair = f[half];
        f[half] = j + 2 < n_pairs ? __ldg(pairs + j + 2) : make_uint2(0, 0);
        if (more) {                            // while the products of this half are made
          if (half == 1) ok = ok && wait_warp(&full[s1], ph1, ab, ERR_WAIT_FULL);
          if (!ok) break;
          expand(half == 0 ? s : s1, half ^ 1);
        }
        if (half == 0) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[s]);
        }
        constexpr int COLS = 16;
#pragma unroll
        for (int u = 0; u < 2 / UNIT; ++u) {
          ok = ok && wait_warp(done, (j * (2 / UNIT) + u) & 1, ab, ERR_Q4_D);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < UNIT; ++h) {
            const uint32_t of = u * UNIT + h ? pair.y : pair.x;
            const float w = 512.f * scale_of(of), z = least_of(of);
            const uint64_t w2 = f2_pack(w, w), z2 = f2_pack(z, z);
#pragma unroll
            for (int c = 0; c < NT; c += COLS) {
              uint32_t v[COLS], o[COLS];
              tmem_ld<COLS>(tmem + kProducts + h * 2 * NT + c + lane_sel, v);
              tmem_ld<COLS>(tmem + kProducts + (h * 2 + 1) * NT + c + lane_sel, o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < COLS; k += 2)
                y[(c + k) / 2] = f2_fma(z2, f2_pack(__uint_as_float(o[k]), __uint_as_float(o[k + 1])),
                                        f2_fma(w2, f2_pack(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), y[(c + k) / 2]));
            }
          }
          if (u + 1 < 2 / UNIT) hand_over();   // the half's second group
        }
        if (!ok) break;
        if (more) {
          tmem_st_32x32b_x32(tmem + lane_sel, r);
          tmem_st_wait();
          hand_over();
        }
      }
      s = s1;
      ph = ph1;
    }
    // every product has been made, so every copy has landed and every operand has been used: the ring is free
#pragma unroll
    for (int c = 0; c < NT; c += 2) {
      float u, v;
      f2_unpack(y[c / 2], u, v);
      red[c * 128 + row] = SPLIT ? u : u * s_back[c];
      red[(c + 1) * 128 + row] = SPLIT ? v : v * s_back[c + 1];
    }
  }
  __syncwarp();
  tc_fence_before();
  if (p.cluster > 1)
    cluster_sync();
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLUMNS);
  }

  finish<NT>(red, p, tile, tokens0, rank, kThreads);
}

// More than 16 rows of x: y = x W^T in bf16, tiles of 128 weight rows and 64 or 128 tokens, the weights expanded into tensor
// memory on their way.  The products of 128 x 128 x 128 take the tensor cores 512 clocks, expanding the codes for them
// takes each scheduler about 300 issue slots (a mask and a shift, 128 + n - 128, n s + z for two channels, rounded once), so that
// a matrix of bf16 weights need be neither written nor read.  (Taking the groups' products by themselves, as above, would
// need an FMA and a read of tensor memory for each of them and each group: 46 us for 777 rows of 5632 x 2048 channels.)
// Measured: 777 rows of 5632 x 2048 channels (112 tiles) 22.9 us, 0.46 of the measured bf16 rate, 32 rows of 11264 x 2048 9.7 us,
// 64 rows of 28672 x 4096 28.6 us.
//   warp 0      TMA: codes of 256 channels, x of 128 channels, in the order of use
//   warp 1      MMA issuer: one wait and one commit a step (each takes the thread a good 100 clocks in which it issues nothing:
//               with barriers of their own for weights and x, 777 rows of 5632 x 2048 channels took 28.0 us instead of 23.1)
//   warps 4-    for a quadrant's 32 weight rows: half of them has every second step's channels (each expanded by two warps where
//               the block has the SM for itself)
template <int NT, int BLOCKS>
struct Many {                                                    // BLOCKS an SM
  static constexpr int SIDES = BLOCKS == 1 ? 2 : 1;              // warps for a quadrant's step
  static constexpr int THREADS = 128 + 256 * SIDES;
  static constexpr int X = 2 * NT * 128;                         // bytes of a step's x
  static constexpr int STEPS = BLOCKS == 1 ? 4 : 3;              // whose operands are there at a time, one barrier for both
  static constexpr int CODE_STAGES = BLOCKS == 1 ? 5 : 3;
  static constexpr int SUMS = STEPS * 64, COLUMNS = SUMS + NT <= 256 ? 256 : 512;   // tensor memory: weights, sums
  static constexpr int BYTES = STEPS * X + CODE_STAGES * kCodeBytes + 1024;
  static_assert(BYTES - 1024 >= NT * 128 * 4 && BLOCKS * (BYTES + 1280) <= 228 * 1024 && BLOCKS * COLUMNS <= 512 &&
                NT <= 64 * SIDES, "an SM's room");
};

// Place in a ring of N, and the parity of its round.
template <int N>
struct Place {
  int at = 0;
  uint32_t round = 0;
  __device__ __forceinline__ void on() {
    if (++at == N) at = 0, round ^= 1;
  }
  __device__ __forceinline__ void on2() {
    at += 2;
    if (at >= N) at -= N, round ^= 1;
  }
};

// Values of a word as eight bf16 in channel order, n s + z rounded once; s2 and z2 hold s and z twice.
__device__ __forceinline__ void values(uint32_t word, uint32_t s2, uint32_t z2, uint32_t mask, uint32_t magic, uint32_t* to) {
  const uint32_t coded_pairs[4] = {coded<0>(word, mask, magic), coded<1>(word, mask, magic), coded<2>(word, mask, magic),
                                   coded<3>(word, mask, magic)};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t n;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(n) : "r"(coded_pairs[k]), "r"(magic));      // magic: 128, twice
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(to[k]) : "r"(n), "r"(s2), "r"(z2));
  }
}

template <int NT, int BLOCKS>
__global__ void __launch_bounds__(Many<NT, BLOCKS>::THREADS, BLOCKS)
linear_q4_many_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                      const __grid_constant__ LinearParams p) {
  using M = Many<NT, BLOCKS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* codes = smem + M::STEPS * M::X;
  __shared__ uint64_t full[M::STEPS], empty[M::STEPS], c_full[M::CODE_STAGES], c_empty[M::CODE_STAGES], done[1];
  __shared__ uint32_t tmem_slot[1];
  __shared__ int abort_word;
  pdl_launch_dependents();
  volatile int* abort_flag = &abort_word;
  const AbortCtx ab{abort_flag, p.status};
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = blockIdx.x % p.cluster;
  const int tokens0 = blockIdx.x / p.cluster % p.token_tiles, tile = blockIdx.x / p.cluster / p.token_tiles;
  const int blocks = (p.width + kStage - 1) / kStage, per = (blocks + p.cluster - 1) / p.cluster;
  const int step0 = 2 * rank * per;                                         // steps of 128 channels, two groups each
  const int steps = max(min(2 * per, p.width / 128 - step0), 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < M::STEPS; ++s) mbar_init(&full[s], 4 * M::SIDES + 1), mbar_init(&empty[s], 1);   // expanders' warps, x
    for (int s = 0; s < M::CODE_STAGES; ++s) mbar_init(&c_full[s], 1), mbar_init(&c_empty[s], 8 * M::SIDES);
    mbar_init(done, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, M::COLUMNS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  float* red = reinterpret_cast<float*>(smem);   // [token][128], over the ring of x once everything has been read

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&tmW);
      tma_prefetch_desc(&tmX);
      for (int i = 0; i < min((steps + 1) / 2, 4); ++i) tma_prefetch_l2_2d(&tmW, (step0 + 2 * i) * 64, tile * 128);
      pdl_wait();
      bool ok = true;
      Place<M::STEPS> x;
      Place<M::CODE_STAGES> c;
      for (int j = 0; j < steps; ++j) {
        if ((j & 1) == 0) {
          ok = wait(&c_empty[c.at], c.round ^ 1, ab, ERR_WAIT_EMPTY);
          if (!ok) break;
          mbar_expect_tx(&c_full[c.at], kCodeBytes);
          tma_load_2d(codes + c.at * kCodeBytes, &tmW, &c_full[c.at], (step0 + j) * 64, tile * 128);
          c.on();
        }
        ok = wait(&empty[x.at], x.round ^ 1, ab, ERR_WAIT_EMPTY);
        if (!ok) break;
        uint8_t* to = smem + x.at * M::X;
        mbar_expect_tx(&full[x.at], M::X);
        tma_load_2d(to, &tmX, &full[x.at], (step0 + j) * 128, tokens0 * NT);
        tma_load_2d(to + M::X / 2, &tmX, &full[x.at], (step0 + j) * 128 + 64, tokens0 * NT);
        x.on();
      }
      if (!ok) {
        // give copies already in flight time to land before the CTA's shared memory goes away
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc_bf16(128, NT, false, false);
      bool ok = true;
      Place<M::STEPS> x;
      for (int j = 0; j < steps; ++j) {
        ok = wait(&full[x.at], x.round, ab, ERR_WAIT_FULL);
        if (!ok) break;
        tc_fence_after();
        const uint64_t xdesc = make_smem_desc_sw128(smem_u32(smem + x.at * M::X), 16, 1024);
        const uint32_t weights = tmem + x.at * 64;
#pragma unroll
        for (int k = 0; k < 8; ++k)              // 16 channels each, 64 to a box of x
          tc_mma_ts(tmem + M::SUMS, weights + k * 8, xdesc + (uint64_t)(((k >> 2) * (M::X / 2) + (k & 3) * 32) >> 4), idesc,
                    (j | k) != 0 ? 1u : 0u);
        tc_commit(&empty[x.at]);
        x.on();
      }
      if (ok && steps > 0) tc_commit(done);
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, row = quad * 32 + lane, side = ((warp - 4) >> 2) % M::SIDES, half = (warp - 4) >> 2 >= M::SIDES;
    const uint32_t lane_sel = static_cast<uint32_t>(quad * 32) << 16;
    const uint2* pairs = reinterpret_cast<const uint2*>(
        p.affine + static_cast<long long>(min(tile * 128 + row, p.N - 1)) * (p.width / 16)) + step0;
    uint32_t mask, magic;
    opaque_masks(mask, magic);
    pdl_wait();
    bool ok = true;
    // a step takes a warp longer than it takes the tensor cores, mostly by waits: half of the warps have the odd steps
    Place<M::CODE_STAGES> c;
    Place<M::STEPS> w;
    if (half) w.on();
    uint2 pair = half < steps ? __ldg(pairs + half) : make_uint2(0, 0);
    for (int j = half; j < steps; j += 2) {
      ok = wait_warp(&c_full[c.at], c.round, ab, ERR_WAIT_FULL);
      if (!ok) break;
      const uint32_t s0 = __byte_perm(pair.x, pair.x, 0x1010), z0 = __byte_perm(pair.x, pair.x, 0x3232);
      const uint32_t s1 = __byte_perm(pair.y, pair.y, 0x1010), z1 = __byte_perm(pair.y, pair.y, 0x3232);
      pair = j + 2 < steps ? __ldg(pairs + j + 2) : make_uint2(0, 0);
#pragma unroll
      for (int part = side; part < 2; part += M::SIDES) {    // half of the channels each
        uint32_t r[2][16];
#pragma unroll
        for (int k = 0; k < 2; ++k) {            // word 4 c + k: channels 64 (k & 1) + 8 (2 c + k / 2) ..
          const uint4 v = *reinterpret_cast<const uint4*>(codes + c.at * kCodeBytes + sw128_offset(row, half * 4 + 2 * part + k));
          values(v.x, s0, z0, mask, magic, &r[0][8 * k]);
          values(v.y, s1, z1, mask, magic, &r[1][8 * k]);
          values(v.z, s0, z0, mask, magic, &r[0][8 * k + 4]);
          values(v.w, s1, z1, mask, magic, &r[1][8 * k + 4]);
        }
        if (part == side) {
          ok = wait_warp(&empty[w.at], w.round ^ 1, ab, ERR_Q4_D);
          if (!ok) break;
          tc_fence_after();
        }
        const uint32_t to = tmem + w.at * 64 + part * 16 + lane_sel;
        tmem_st16(to, r[0]);
        tmem_st16(to + 32, r[1]);
      }
      if (!ok) break;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&full[w.at]);
        mbar_arrive(&c_empty[c.at]);
      }
      w.on2();
      c.on();
    }
    if (steps > 0) ok = wait_warp(done, 0, ab, ERR_Q4_D) && ok;
    tc_fence_after();
    // every product has been made, so every copy has landed and every operand has been used: the ring is free
    const int token = (half * M::SIDES + side) * 32;
    if (token < NT) {
      uint32_t v[32];
      if (steps > 0 && ok) {
        tmem_ld_32x32b_x32(tmem + M::SUMS + token + lane_sel, v);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0;
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) red[(token + i) * 128 + row] = __uint_as_float(v[i]);
    }
  }
  __syncwarp();
  tc_fence_before();
  if (p.cluster > 1)
    cluster_sync();
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, M::COLUMNS);
  }
  finish<NT>(red, p, tile, tokens0, rank, M::THREADS);
}

// Rows of up to 64 channels (one group, words in channel order): one warp per weight row and eight rows of x, a lane per word.
__global__ void __launch_bounds__(128) linear_q4_narrow_kernel(const __nv_bfloat16* x, long long ldx, const uint32_t* codes,
                                                               const uint32_t* affine, __nv_bfloat16* out, long long ldo,
                                                               int rows, int N, int K) {
  const int n = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, m0 = blockIdx.y * 8;
  pdl_launch_dependents();
  pdl_wait();
  if (n >= N) return;
  const int m1 = min(rows - m0, 8), c = (lane & 7) * 8;
  const uint32_t a = affine[n];
  float acc[8] = {}, v[8];
  unpack(lane < 8 ? codes[static_cast<long long>(n) * 8 + lane] : 0u, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = fmaf(v[i], scale_of(a), least_of(a));
#pragma unroll
  for (int m = 0; m < 8; ++m) {
    if (m >= m1) break;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane < 8 && c + i < K) acc[m] = fmaf(__bfloat162float(x[(m0 + m) * ldx + c + i]), v[i], acc[m]);
  }
#pragma unroll
  for (int m = 0; m < 8; ++m) {
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], off);
    if (lane == 0 && m < m1) out[(m0 + m) * ldo + n] = __float2bfloat16(acc[m]);
  }
}

template <typename... Args>
int launch_cluster(void (*kern)(Args...), const LinearParams& p, int threads, int smem_bytes, cudaStream_t stream,
                   const std::common_type_t<Args>&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.N + 127) / 128 * p.token_tiles * p.cluster);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = b200host::pdl_enabled() ? 2 : 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, args...));
}

template <bool SPLIT>
int launch(const CUtensorMap& tmW, const CUtensorMap& tmX, const CUtensorMap& tmS, LinearParams p, cudaStream_t stream) {
  const int blocks = (p.width + kStage - 1) / kStage, slice = (blocks + p.cluster - 1) / p.cluster;
  constexpr int most = (222 * 1024 / kFewBlocks - 2048) / kStageBytes;
  static_assert(most >= kOwnStages && most <= kMaxStages && most * kStageBytes >= kFewRows * 128 * 4, "slots; the sums reuse them");
  p.stages = slice < most ? (slice < 2 ? 2 : slice) : most;
  const int smem_bytes = p.stages * kStageBytes + 1024;
  static bool configured[b200host::kMaxDevices] = {};
  if (int rc = b200host::ensure_dynamic_smem(linear_q4_kernel<SPLIT>, most * kStageBytes + 1024, configured)) return rc;
  return launch_cluster(linear_q4_kernel<SPLIT>, p, kThreads, smem_bytes, stream, tmW, tmX, tmS, p);
}

template <int NT, int BLOCKS>
int launch_many(const CUtensorMap& tmW, const CUtensorMap& tmX, const LinearParams& p, cudaStream_t stream) {
  using M = Many<NT, BLOCKS>;
  static bool configured[b200host::kMaxDevices] = {};
  if (int rc = b200host::ensure_dynamic_smem(linear_q4_many_kernel<NT, BLOCKS>, M::BYTES, configured)) return rc;
  return launch_cluster(linear_q4_many_kernel<NT, BLOCKS>, p, M::THREADS, M::BYTES, stream, tmW, tmX, p);
}

}  // namespace

// out [rows, N] (row stride ldo) = x [rows, K] (ldx) * W^T, W as codes [N, width / 8] words and affine [N, width / 64] pairs;
// `cluster` (1, 2, 4 or 8) slices of K.  `work` is the call's own: up to 16 rows, where a slice has more than
// 512 channels, 40 * width bytes and then 16 floats, width = K rounded up to 256.  With more than 16 rows of more than 64 channels
// rows of x start on 16 bytes.
extern "C" int b200_q4_linear(const void* x, long long ldx, const void* codes, const void* affine, void* out,
                              long long ldo, int rows, int N, int K, int cluster, void* work, void* status,
                              void* stream) {
  using namespace b200host;
  if (rows <= 0 || rows > (1 << 24) || N <= 0 || K <= 0 || K > (1 << 30) || !status) return RC_BAD_SHAPE;
  if (cluster != 1 && cluster != 2 && cluster != 4 && cluster != 8) return RC_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(affine)) & 15) return RC_BAD_ALIGNMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int width = row_width(K);
  const bool pdl = pdl_enabled() != 0;
  if (width == 64)
    return static_cast<int>(launch_kernel(linear_q4_narrow_kernel, dim3((N + 3) / 4, (rows + 7) / 8), dim3(128), 0, s, pdl,
                                          (const __nv_bfloat16*)x, ldx, (const uint32_t*)codes, (const uint32_t*)affine,
                                          (__nv_bfloat16*)out, ldo, rows, N, K));
  if (reinterpret_cast<uintptr_t>(out) & 7) return RC_BAD_ALIGNMENT;
  CUtensorMap tmW, tmX, tmS;
  int rc;
  if ((rc = make_map_2d(&tmW, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, width / 2, N, width / 2, 128, 128))) return rc;
  if (rows > kFewRows) {
    const int NT = rows <= 64 ? 64 : 128, tiles = (rows + NT - 1) / NT;
    if ((long long)tiles * ((N + 127) / 128) * cluster > 0x7fffffffll) return RC_BAD_SHAPE;
    if ((rc = make_map_2d(&tmX, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, K, rows, ldx * 2, 64, NT))) return rc;
    const LinearParams p{(const uint8_t*)affine, nullptr, (__nv_bfloat16*)out, ldo, rows, N, width, cluster, 0, tiles,
                         (int*)status};
    if (NT == 128) return launch_many<128, 1>(tmW, tmX, p, s);
    // two smaller blocks an SM where there are more than SMs: 64 rows, 224 blocks of 28672 x 4096 28.6 us instead of 35.5, 64 of
    // 4096 x 14336 in two slices 34 us instead of 27.7
    return (N + 127) / 128 * tiles * cluster > sm_count() ? launch_many<64, 2>(tmW, tmX, p, s) : launch_many<64, 1>(tmW, tmX, p, s);
  }
  const int aligned = ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const int xwidth = (K + kStage - 1) / kStage * kStage;
  LinearParams p{(const uint8_t*)affine, nullptr, (__nv_bfloat16*)out, ldo, rows, N, width, cluster, 0, 1,
                 (int*)status, (const __nv_bfloat16*)x, ldx, K, aligned};
  if ((xwidth / kStage + cluster - 1) / cluster <= kOwnStages) return launch<false>(tmW, tmW, tmW, p, s);
  if (!work || (reinterpret_cast<uintptr_t>(work) & 15)) return RC_BAD_ALIGNMENT;
  uint8_t* xq = static_cast<uint8_t*>(work);
  uint8_t* sums = xq + 2ll * kFewRows * xwidth;
  float* xs = reinterpret_cast<float*>(sums + kFewRows * (xwidth / 2ll));
  if ((rc = make_map_2d(&tmX, CU_TENSOR_MAP_DATA_TYPE_UINT8, xq, xwidth, 2 * kFewRows, xwidth, 128, 2 * kFewRows))) return rc;
  if ((rc = make_map_2d(&tmS, CU_TENSOR_MAP_DATA_TYPE_UINT8, sums, xwidth / 2, kFewRows, xwidth / 2, 128, kFewRows))) return rc;
  if (cudaError_t e = launch_kernel(linear_q4_split_kernel, dim3(kFewRows), dim3(512), 0, s, pdl, (const __nv_bfloat16*)x, ldx,
                                    rows, K, xwidth, aligned, xq, xs))
    return static_cast<int>(e);
  p.xs = xs;
  return launch<true>(tmW, tmX, tmS, p, s);
}

// y = x W^T with weights held in 4 bits (quant4.cuh): x [rows, K] bf16, W [N, K], y [rows, N] bf16 with fp32 sums.
//
// Up to 8 or 16 rows of x (the caller's choice) the time is that of streaming the codes once (0.56 bytes a weight), as long as
// expanding them keeps up: at the copy bandwidth an SM gets 46 codes a clock.  linear_q4_few_kernel expands nothing: the codes
// go from memory to registers to mma.sync m16n8k16 as the bf16 numbers that their bits are, n 2^-133 (subnormals and the first
// binade are one straight line), by a mask each and one shift for four of eight; x is the column operand, brought to about
// 2^120 by a power of two of the warp's share of its row, and divided by 16 where a code sits four bits up.  Products are
// exact, and scales and least values are applied to the groups' sums in fp32:  y = sum_g s_g (sum_k x_k n_k) + z_g sum_k x_k.
// Each warp keeps its channels of x in registers and has every tile of weight rows pass by, so that there is nothing to
// prepare per tile, nothing goes through shared memory but the partial sums of 16 x 8, and one load is always under way.
// Measured, 1 row: 2048 x 2048 3.5 us, 11264 x 2048 5.6, 28672 x 4096 16.0 (0.63 of the copy bandwidth), 50304 x 2048 13.9; 8
// rows take 3.8, 6.0, 16.6 and 14.4 us.  (With x from memory for each tile 28672 x 4096 took 31 us; on tcgen05, with the codes
// as e4m3 subnormals written to tensor memory, x in two e4m3 parts and each group's product read back, 22.4, and 2048 x 2048
// 5.7.)
//
// More rows: linear_q4_many_kernel below.
#include <type_traits>

#include "quant4.cuh"
#include "host_util.cuh"

namespace {

using namespace q4;
using namespace b200;

constexpr int kStage = 256;                    // channels of a stage of codes
constexpr int kCodeBytes = 128 * kStage / 2;
constexpr int ERR_Q4_D = 42;                   // status code: operands that were never used, or products that never came

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

__device__ __forceinline__ float ld_cluster(uint32_t saddr, uint32_t rank) {
  uint32_t peer;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer) : "memory");
  return v;
}

struct FewParams {
  const __nv_bfloat16* x;             // [rows, K], `aligned` where 16 bytes may be read at once
  long long ldx;
  const uint8_t *codes, *affine;
  __nv_bfloat16* out;
  long long ldo;
  int rows, N, K, width, aligned, cluster;
};
constexpr int kHeld = 8;              // rounds after which a cluster adds up its blocks' sums

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld_stream(const uint4* at) {   // read once: not to stay in L1
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at));
  return v;
}

// A warp has KB blocks of 128 channels of up to 8 * NC rows of x; a block has WARPS * KB of them, and a cluster the whole row.
// Tiles of 16 weight rows go round the clusters.
template <int KB, int WARPS, int NC>
__global__ void __launch_bounds__(WARPS * 32) linear_q4_few_kernel(const __grid_constant__ FewParams p) {
  __shared__ float red[2][WARPS][8 * NC][17];
  __shared__ float part[kHeld][128 * NC];      // sums of the cluster's last rounds
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % p.cluster, first = blockIdx.x / p.cluster, clusters = gridDim.x / p.cluster;
  const int blocks = p.width >> 7, tiles = (p.N + 15) >> 4;
  const int kb0 = (rank * WARPS + warp) * KB;
  const long long row_bytes = p.width >> 1;
  uint4 code[2][KB];
  uint2 pair[2][KB];
  auto at_row = [&](int tile, int m) { return static_cast<long long>(min(tile * 16 + 8 * m + g, p.N - 1)); };
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int b = 0; b < KB; ++b) code[m][b] = make_uint4(0, 0, 0, 0), pair[m][b] = make_uint2(0, 0);
  b200::pdl_launch_dependents();
  // what runs before may be what writes the weights: they are read after the wait, by loads that do not take them for
  // unchanging, and only brought into L2 ahead of it
#pragma unroll
  for (int m = 0; m < 2; ++m)
    if (kb0 < blocks)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.codes + at_row(first, m) * row_bytes + (4ll * kb0 + t) * 16));
  b200::pdl_wait();
  auto load_w = [&](int tile) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const long long n = at_row(tile, m);
      const uint4* c = reinterpret_cast<const uint4*>(p.codes + n * row_bytes + t * 16) + 4 * kb0;
      const uint2* f = reinterpret_cast<const uint2*>(p.affine + n * (p.width >> 4)) + kb0;
#pragma unroll
      for (int b = 0; b < KB; ++b)
        if (kb0 + b < blocks) {
          code[m][b] = ld_stream(c + 4 * b);
          pair[m][b] = f[b];
        }
    }
  };
  if (first < tiles) load_w(first);

  // x as the column operand: column g is row 8 c + g of x; channels of this lane's words
  uint32_t x[NC][KB][4][4];
  float back1[NC][2], back2[NC][2], sum[NC][KB][2][2];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    uint32_t most = 0;
    const int token = 8 * c + g;
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int ch = (kb0 + b) * 128 + 64 * (j & 1) + 16 * t + 8 * (j >> 1);
        uint4 u = make_uint4(0, 0, 0, 0);
        if (token < p.rows && ch < p.K) {
          const __nv_bfloat16* at = p.x + token * p.ldx + ch;
          if (p.aligned && ch + 8 <= p.K) {
            u = *reinterpret_cast<const uint4*>(at);
          } else {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t lo = ch + 2 * k < p.K ? __bfloat16_as_ushort(at[2 * k]) : 0;
              const uint32_t hi = ch + 2 * k + 1 < p.K ? __bfloat16_as_ushort(at[2 * k + 1]) : 0;
              w[k] = lo | hi << 16;
            }
            u = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        x[c][b][j][0] = u.x, x[c][b][j][1] = u.y, x[c][b][j][2] = u.z, x[c][b][j][3] = u.w;
#pragma unroll
        for (int k = 0; k < 4; ++k) most = max(most, max(x[c][b][j][k] & 0x7f80u, (x[c][b][j][k] >> 16) & 0x7f80u));
      }
    // a power of two brings the warp's share of a column to about 2^120, as far as one factor can
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int f = min(127, 247 - static_cast<int>(most >> 7));   // exponent of the factor: 120 - e
    const uint32_t up = static_cast<uint32_t>(f + 127) * 0x00800080u, up16 = static_cast<uint32_t>(f + 123) * 0x00800080u;
#pragma unroll
    for (int k = 0; k < 2; ++k) {              // what undoes it, of columns 2 t and 2 t + 1: 2^6 .. 2^141, in two factors
      const int e = 133 - __shfl_sync(0xffffffffu, f, 8 * t + 4 * k);
      back1[c][k] = __uint_as_float(static_cast<uint32_t>((e >> 1) + 127) << 23);
      back2[c][k] = __uint_as_float(static_cast<uint32_t>(e - (e >> 1) + 127) << 23);
    }
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      float acc[2][4] = {};                    // sums over the groups: the product with a row of ones
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(x[c][b][j][k]) : "r"(x[c][b][j][k]), "r"(k & 1 ? up16 : up));
        mma_bf16(acc[j & 1], 0x00010001u, 0x00010001u, 0x00100010u, 0x00100010u, x[c][b][j][0], x[c][b][j][1]);
        mma_bf16(acc[j & 1], 0x00010001u, 0x00010001u, 0x00100010u, 0x00100010u, x[c][b][j][2], x[c][b][j][3]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) sum[c][b][h][0] = acc[h][0], sum[c][b][h][1] = acc[h][1];
    }
  }

  int round = 0;
  for (int tile = first; tile < tiles; tile += clusters, ++round) {
    float y[NC][4] = {};
    uint4 w[2][KB];
    uint2 of[2][KB];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int b = 0; b < KB; ++b) w[m][b] = code[m][b], of[m][b] = pair[m][b];
    if (tile + clusters < tiles) load_w(tile + clusters);
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const uint32_t wa[4] = {w[0][b].x, w[0][b].y, w[0][b].z, w[0][b].w}, wb[4] = {w[1][b].x, w[1][b].y, w[1][b].z, w[1][b].w};
      float acc[NC][2][4] = {};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a = wa[j], b8 = wb[j], a2 = a >> 8, b2 = b8 >> 8;
        const uint32_t lo[2] = {a & 0x000f000fu, b8 & 0x000f000fu}, hi[2] = {a & 0x00f000f0u, b8 & 0x00f000f0u};
        const uint32_t lo2[2] = {a2 & 0x000f000fu, b2 & 0x000f000fu}, hi2[2] = {a2 & 0x00f000f0u, b2 & 0x00f000f0u};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          mma_bf16(acc[c][j & 1], lo[0], lo[1], hi[0], hi[1], x[c][b][j][0], x[c][b][j][1]);
          mma_bf16(acc[c][j & 1], lo2[0], lo2[1], hi2[0], hi2[1], x[c][b][j][2], x[c][b][j][3]);
        }
      }
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint2 q = of[i >> 1][b];
          float v = y[c][i];
          v = fmaf(scale_of(q.x), acc[c][0][i], v);
          v = fmaf(least_of(q.x), sum[c][b][0][i & 1], v);
          v = fmaf(scale_of(q.y), acc[c][1][i], v);
          y[c][i] = fmaf(least_of(q.y), sum[c][b][1][i & 1], v);
        }
    }
    float(*r)[8 * NC][17] = red[round & 1];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        r[warp][8 * c + 2 * t + (i & 1)][g + 8 * (i >> 1)] = y[c][i] * back1[c][i & 1] * back2[c][i & 1];
    __syncthreads();                           // who read this buffer two rounds ago is past the barrier before this one
    if (threadIdx.x < 128 * NC) {
      const int token = threadIdx.x >> 4, n = threadIdx.x & 15;
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) v += r[k][token][n];
      if (p.cluster > 1)
        part[round % kHeld][threadIdx.x] = v;
      else if (token < p.rows && tile * 16 + n < p.N)
        p.out[token * p.ldo + tile * 16 + n] = __float2bfloat16(v);
    }
    if (p.cluster > 1 && ((round + 1) % kHeld == 0 || tile + clusters >= tiles)) {   // the same for all blocks of the cluster
      __syncwarp();
      cluster_sync();
      const int held = round % kHeld + 1;
      for (int i = threadIdx.x + rank * WARPS * 32; i < held * 128 * NC; i += p.cluster * WARPS * 32) {
        const int back = held - 1 - i / (128 * NC), at = i % (128 * NC), token = at >> 4;
        const int n = (tile - back * clusters) * 16 + (at & 15);
        if (token >= p.rows || n >= p.N) continue;
        float v = 0.f;
        for (int k = 0; k < p.cluster; ++k) v += ld_cluster(smem_u32(&part[0][0] + i), k);
        p.out[token * p.ldo + n] = __float2bfloat16(v);
      }
      __syncwarp();
      cluster_sync();                          // peers may still read this block's sums
    }
  }
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
struct LinearParams {
  const uint8_t* affine;
  __nv_bfloat16* out;
  long long ldo;
  int rows, N, width, cluster, token_tiles;
  int* status;
};

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

// More than 16 rows of x: y = x W^T in bf16, tiles of 128 weight rows and 64 or 128 tokens, the weights expanded into tensor
// memory on their way.  The products of 128 x 128 x 128 take the tensor cores 512 clocks, expanding the codes for them
// takes each scheduler about 300 issue slots (a mask and a shift, 128 + n - 128, n s + z for two channels, rounded once), so that
// a matrix of bf16 weights need be neither written nor read.  (Taking the groups' products by themselves, codes as e4m3
// subnormals and x in two parts, would need an FMA and a read of tensor memory for each of them and each group: 46 us for 777
// rows of 5632 x 2048 channels.)  That a weight counts as a bf16 here, n s + z rounded once, is the price: 0.0023 of the result
// away from 64 bits where codes as they are have its own rounding, 0.0017, and a row's results depend on which kernel the
// number of rows beside it picks.
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
    uint2 pair = half < steps ? pairs[half] : make_uint2(0, 0);
    for (int j = half; j < steps; j += 2) {
      ok = wait_warp(&c_full[c.at], c.round, ab, ERR_WAIT_FULL);
      if (!ok) break;
      const uint32_t s0 = __byte_perm(pair.x, pair.x, 0x1010), z0 = __byte_perm(pair.x, pair.x, 0x3232);
      const uint32_t s1 = __byte_perm(pair.y, pair.y, 0x1010), z1 = __byte_perm(pair.y, pair.y, 0x3232);
      pair = j + 2 < steps ? pairs[j + 2] : make_uint2(0, 0);
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
int launch_cluster(void (*kern)(Args...), int cluster, long long blocks, int threads, int smem_bytes, cudaStream_t stream,
                   const std::common_type_t<Args>&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = b200host::pdl_enabled() ? 2 : 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, args...));
}

template <int KB, int WARPS, int NC>
int launch_few(FewParams p, int blocks_per_sm, cudaStream_t stream) {
  const int tiles = (p.N + 15) / 16;
  p.cluster = (p.width / 128 + WARPS * KB - 1) / (WARPS * KB);
  if (p.cluster > 8) return b200host::RC_BAD_SHAPE;   // more channels than a cluster's registers hold of x
  // clusters of more than 2 and 4 find no room on some of the SMs
  int clusters = blocks_per_sm * b200host::sm_count() * (p.cluster > 4 ? 75 : p.cluster > 2 ? 90 : 100) / 100 / p.cluster;
  if (clusters > tiles) clusters = tiles;
  if (clusters < 1) clusters = 1;
  return launch_cluster(linear_q4_few_kernel<KB, WARPS, NC>, p.cluster, (long long)clusters * p.cluster, WARPS * 32, 0, stream, p);
}

template <int NT, int BLOCKS>
int launch_many(const CUtensorMap& tmW, const CUtensorMap& tmX, const LinearParams& p, cudaStream_t stream) {
  using M = Many<NT, BLOCKS>;
  static bool configured[b200host::kMaxDevices] = {};
  if (int rc = b200host::ensure_dynamic_smem(linear_q4_many_kernel<NT, BLOCKS>, M::BYTES, configured)) return rc;
  return launch_cluster(linear_q4_many_kernel<NT, BLOCKS>, p.cluster, (long long)((p.N + 127) / 128) * p.token_tiles * p.cluster,
                        M::THREADS, M::BYTES, stream, tmW, tmX, p);
}

}  // namespace

// out [rows, N] (row stride ldo) = x [rows, K] (ldx) * W^T, W as codes [N, width / 8] words and affine [N, width / 64] pairs.  With
// more than 64 channels the caller says how: `cluster` 0 multiplies the codes as they are (up to 16 rows of 16384 channels or 8
// of 32768), 1, 2, 4 or 8 cuts K into as many slices of expanded weights, for which rows of x start on 16 bytes.
extern "C" int b200_q4_linear(const void* x, long long ldx, const void* codes, const void* affine, void* out,
                              long long ldo, int rows, int N, int K, int cluster, void* status, void* stream) {
  using namespace b200host;
  if (rows <= 0 || rows > (1 << 24) || N <= 0 || K <= 0 || K > (1 << 30) || !status) return RC_BAD_SHAPE;
  if (cluster < 0 || cluster > 8 || (cluster & (cluster - 1))) return RC_BAD_SHAPE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int width = row_width(K);
  if (!rows_aligned(codes, affine, width)) return RC_BAD_ALIGNMENT;
  if (width == 64)
    return static_cast<int>(launch_kernel(linear_q4_narrow_kernel, dim3((N + 3) / 4, (rows + 7) / 8), dim3(128), 0, s,
                                          pdl_enabled() != 0, (const __nv_bfloat16*)x, ldx, (const uint32_t*)codes,
                                          (const uint32_t*)affine, (__nv_bfloat16*)out, ldo, rows, N, K));
  if (cluster == 0) {
    if (rows > 16) return RC_BAD_SHAPE;
    const int aligned = ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0, blocks = width / 128;
    const FewParams p{(const __nv_bfloat16*)x, ldx, (const uint8_t*)codes, (const uint8_t*)affine, (__nv_bfloat16*)out, ldo, rows,
                      N, K, width, aligned, 1};
    // registers for x: two blocks of 128 channels a warp, or one of twice the rows; as many warps as that takes
    if (rows > 8) return blocks <= 8 ? launch_few<1, 8, 2>(p, 2, s) : launch_few<1, 16, 2>(p, 1, s);
    if (blocks <= 8) return launch_few<1, 8, 1>(p, 3, s);
    return blocks <= 16 ? launch_few<2, 8, 1>(p, 2, s) : launch_few<2, 16, 1>(p, 1, s);
  }
  if (reinterpret_cast<uintptr_t>(out) & 7) return RC_BAD_ALIGNMENT;
  const int NT = rows <= 64 ? 64 : 128, tiles = (rows + NT - 1) / NT;
  if ((long long)tiles * ((N + 127) / 128) * cluster > 0x7fffffffll) return RC_BAD_SHAPE;
  CUtensorMap tmW, tmX;
  int rc;
  if ((rc = make_map_2d(&tmW, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, width / 2, N, width / 2, 128, 128))) return rc;
  if ((rc = make_map_2d(&tmX, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, K, rows, ldx * 2, 64, NT))) return rc;
  const LinearParams p{(const uint8_t*)affine, (__nv_bfloat16*)out, ldo, rows, N, width, cluster, tiles, (int*)status};
  if (NT == 128) return launch_many<128, 1>(tmW, tmX, p, s);
  // two smaller blocks an SM where there are more than SMs: 64 rows, 224 blocks of 28672 x 4096 28.6 us instead of 35.5, 64 of
  // 4096 x 14336 in two slices 34 us instead of 27.7
  return (long long)((N + 127) / 128) * tiles * cluster > sm_count() ? launch_many<64, 2>(tmW, tmX, p, s)
                                                                     : launch_many<64, 1>(tmW, tmX, p, s);
}

// y = x W^T for a few rows of x and weights held in 4 bits (quant4.cuh): x [rows, K] bf16, W [N, K], y [rows, N] bf16 with
// fp32 sums.  The time is that of streaming the codes once (0.56 bytes a weight), as long as expanding them keeps up.
//
// Weights are the 16-row operand of m16n8k16, the rows of x its columns, eight to a tile.  A code becomes the bf16 128 + n by
// half a shift and one and-or per two codes, exact; a group's sum is scaled in fp32, and what the offset and the least values
// add is taken off at the end by a small product over the groups:
//   y = sum_g s_g (sum_k x_k (128 + n_k)) + sum_g (z_g - 128 s_g) X_g,   X_g = sum_k x_k,
// with X_g, itself a product with ones, as three bf16 parts (24 bits) against s and z, which are bf16.
//
// A block of eight warps has 16 WM weight rows and a slice of K; WM warps share the rows, 8 / WM the slice's blocks of 128
// channels, and the blocks of a cluster share K.  Codes go straight to the registers of the lane that expands them, four
// blocks ahead; x goes through shared memory, two stages, rows 16 bytes apart from a multiple of 128, so that no two lanes
// of a read meet in a bank.  Partial sums are added in the order of warps and ranks, the same bits every time.
#include "quant4.cuh"
#include "host_util.cuh"

namespace {

using namespace q4;

constexpr int kWarps = 8, kThreads = kWarps * 32, kAhead = 4;

struct LinearParams {
  const __nv_bfloat16* x;
  long long ldx, ldo;
  const uint8_t *codes, *affine;
  __nv_bfloat16* out;
  int rows, N, K, width, cluster;
  int aligned;                        // rows of x start on 16 bytes
};

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Codes P of both halves of w as bf16 128 + n: one shift and one three-input operation (a & b) | c, whose constants are kept
// in registers, since an instruction has room for one.
template <int P>
__device__ __forceinline__ uint32_t coded(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(P ? w >> (4 * P) : w), "r"(mask), "r"(magic));
  return r;
}
constexpr uint32_t kOnes = 0x3f803f80u;

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t saddr, uint32_t rank) {
  uint32_t peer;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer) : "memory");
  return v;
}

template <int NT, int WM>
struct Shape {
  static constexpr int WK = kWarps / WM;
  static constexpr int BPW = WK >= 4 ? 1 : 2;                 // blocks a warp has in a stage
  static constexpr int STAGE_BLOCKS = WK * BPW, STAGE_CHANNELS = STAGE_BLOCKS * 128;
  static constexpr int TOKENS = NT * 8, PITCH = STAGE_CHANNELS * 2 + 16;
  static constexpr int STAGE_BYTES = TOKENS * PITCH;
  static constexpr int SUM_BYTES = kWarps * 16 * TOKENS * 4;  // partial results, over the stages
  static constexpr int RING_BYTES = 2 * STAGE_BYTES > SUM_BYTES ? 2 * STAGE_BYTES : SUM_BYTES;
  // groups of the slice: a 16-multiple of them, X_g in fp32
  static int xs_bytes(int slice_blocks) { return ((2 * slice_blocks + 15) / 16 * 16) * TOKENS * 4; }
};

template <int NT, int WM>
__global__ void __launch_bounds__(kThreads, NT <= 4 ? 2 : 1) linear_q4_kernel(const __grid_constant__ LinearParams p) {
  using S = Shape<NT, WM>;
  constexpr int WK = S::WK, BPW = S::BPW, TOKENS = S::TOKENS;
  extern __shared__ __align__(16) uint8_t smem[];
  float* xs = reinterpret_cast<float*>(smem + S::RING_BYTES);   // [groups][TOKENS]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int wm = warp % WM, wk = warp / WM;
  const int rank = blockIdx.x % p.cluster, tile = blockIdx.x / p.cluster;
  const int blocks = p.width / 128;
  const int slice = (blocks + p.cluster - 1) / p.cluster;       // blocks of 128 channels of a rank
  const int kb0 = rank * slice, n_blocks = max(min(slice, blocks - kb0), 0);
  const int mine = (n_blocks - wk + WK - 1) / WK;               // of this warp: kb0 + wk + i WK (may be none)
  const int stages = (n_blocks + S::STAGE_BLOCKS - 1) / S::STAGE_BLOCKS;

  const int n0 = (tile * WM + wm) * 16 + g;
  const long long ra = min(n0, p.N - 1), rb = min(n0 + 8, p.N - 1);
  const uint8_t* ca = p.codes + ra * (p.width / 2) + (kb0 + wk) * 64 + t * 16;
  const uint8_t* cb = p.codes + rb * (p.width / 2) + (kb0 + wk) * 64 + t * 16;
  const uint8_t* sa = p.affine + ra * (p.width / 16) + (kb0 + wk) * 8;
  const uint8_t* sb = p.affine + rb * (p.width / 16) + (kb0 + wk) * 8;
  b200::pdl_launch_dependents();
#pragma unroll
  for (int i = 0; i < kAhead; ++i)      // what runs before may be what writes the weights: only into L2 ahead of the wait
    if (i < mine && t == 0) {
      asm volatile("prefetch.global.L2 [%0];" ::"l"(ca + i * WK * 64));
      asm volatile("prefetch.global.L2 [%0];" ::"l"(cb + i * WK * 64));
    }
  // columns behind the last row of x stay zero
  for (int i = threadIdx.x; i < 2 * (TOKENS - p.rows) * (S::PITCH / 16); i += kThreads) {
    const int c = i % (S::PITCH / 16), r = i / (S::PITCH / 16);
    *reinterpret_cast<uint4*>(smem + (r & 1) * S::STAGE_BYTES + (p.rows + (r >> 1)) * S::PITCH + c * 16) = make_uint4(0, 0, 0, 0);
  }
  b200::pdl_wait();

  uint4 wa[kAhead], wb[kAhead];
  uint2 fa[kAhead], fb[kAhead];
  auto load = [&](int i, int slot) {
    if (i < mine) {
      wa[slot] = __ldg(reinterpret_cast<const uint4*>(ca + static_cast<long long>(i) * (WK * 64)));
      wb[slot] = __ldg(reinterpret_cast<const uint4*>(cb + static_cast<long long>(i) * (WK * 64)));
      fa[slot] = __ldg(reinterpret_cast<const uint2*>(sa + static_cast<long long>(i) * (WK * 8)));
      fb[slot] = __ldg(reinterpret_cast<const uint2*>(sb + static_cast<long long>(i) * (WK * 8)));
    }
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(i, i);

  auto stage_in = [&](int s) {
    if (s < stages) {
      uint8_t* dst = smem + (s & 1) * S::STAGE_BYTES;
      const int c0 = kb0 * 128 + s * S::STAGE_CHANNELS;
      constexpr int CHUNKS = S::STAGE_CHANNELS / 8;
      for (int i = threadIdx.x; i < p.rows * CHUNKS; i += kThreads) {
        const int r = i / CHUNKS, cc = i - r * CHUNKS, c = c0 + cc * 8;
        uint8_t* to = dst + r * S::PITCH + cc * 16;
        const __nv_bfloat16* from = p.x + r * p.ldx + c;
        if (p.aligned) {
          const int bytes = max(min((p.K - c) * 2, 16), 0);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(b200::smem_u32(to)), "l"(bytes ? from : p.x), "r"(bytes)
                       : "memory");
        } else {
          const uint16_t* u = reinterpret_cast<const uint16_t*>(from);
          uint32_t v[4] = {};
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (c + k < p.K) v[k >> 1] |= static_cast<uint32_t>(u[k]) << (16 * (k & 1));
          *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  stage_in(0);

  uint32_t mask = 0x000f000fu, magic = 0x43004300u;
  asm volatile("" : "+r"(mask), "+r"(magic));
  float y[NT][4] = {};
  for (int i0 = 0; i0 < stages * BPW; i0 += kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u;
      if (i < stages * BPW) {             // the same for every thread of the block
        const int s = i / BPW;
        if (i % BPW == 0) {
          asm volatile("cp.async.wait_group 0;" ::: "memory");
          __syncthreads();                // stage s is there, and nobody reads stage s - 1 any more
          stage_in(s + 1);
        }
        if (i < mine) {
          const uint8_t* xb = smem + (s & 1) * S::STAGE_BYTES + g * S::PITCH + ((i % BPW) * WK + wk) * 256 + t * 32;
          const uint32_t ka[4] = {wa[u].x, wa[u].y, wa[u].z, wa[u].w}, kb[4] = {wb[u].x, wb[u].y, wb[u].z, wb[u].w};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float acc[NT][4], ones[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int c = 0; c < 4; ++c) acc[n][c] = ones[n][c] = 0.f;
#pragma unroll
            for (int j = h; j < 4; j += 2) {
              const uint32_t a0 = coded<0>(ka[j], mask, magic), a1 = coded<0>(kb[j], mask, magic);
              const uint32_t a2 = coded<1>(ka[j], mask, magic), a3 = coded<1>(kb[j], mask, magic);
              const uint32_t e0 = coded<2>(ka[j], mask, magic), e1 = coded<2>(kb[j], mask, magic);
              const uint32_t e2 = coded<3>(ka[j], mask, magic), e3 = coded<3>(kb[j], mask, magic);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const uint4 b = *reinterpret_cast<const uint4*>(xb + n * 8 * S::PITCH + h * 128 + (j >> 1) * 16);
                mma(acc[n], a0, a1, a2, a3, b.x, b.y);
                mma(acc[n], e0, e1, e2, e3, b.z, b.w);
                if ((h * NT + n) % WM == wm) {        // the warps of the rows share the sums of x
                  mma(ones[n], kOnes, kOnes, kOnes, kOnes, b.x, b.y);
                  mma(ones[n], kOnes, kOnes, kOnes, kOnes, b.z, b.w);
                }
              }
            }
            const float s0 = scale_of(h ? fa[u].y : fa[u].x), s1 = scale_of(h ? fb[u].y : fb[u].x);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              y[n][0] = fmaf(s0, acc[n][0], y[n][0]);
              y[n][1] = fmaf(s0, acc[n][1], y[n][1]);
              y[n][2] = fmaf(s1, acc[n][2], y[n][2]);
              y[n][3] = fmaf(s1, acc[n][3], y[n][3]);
              if ((h * NT + n) % WM == wm && g == 0)
                *reinterpret_cast<float2*>(xs + ((i * WK + wk) * 2 + h) * TOKENS + n * 8 + 2 * t) =
                    make_float2(ones[n][0], ones[n][1]);
            }
          }
        }
        load(i + kAhead, u);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  // groups up to a multiple of 16 count nothing
  for (int i = 2 * n_blocks * TOKENS + threadIdx.x; i < (2 * n_blocks + 15) / 16 * 16 * TOKENS; i += kThreads) xs[i] = 0.f;
  __syncthreads();

  // sum_g z_g X_g - 128 s_g X_g: 16 groups a step, dealt to the warps that share the slice
  for (int k0 = wk * 16; k0 < 2 * n_blocks; k0 += WK * 16) {
    uint32_t as[4], az[4];        // (row g, groups 2t, 2t + 1), (row g + 8, same), (row g, + 8), (row g + 8, + 8)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int group = k0 + 2 * t + (q >> 1) * 8;
      uint2 v = make_uint2(0, 0);
      if (group < 2 * n_blocks)
        v = __ldg(reinterpret_cast<const uint2*>(p.affine + ((q & 1) ? rb : ra) * (p.width / 16) + (kb0 * 2 + group) * 4));
      as[q] = __byte_perm(v.x, v.y, 0x5410);
      az[q] = __byte_perm(v.x, v.y, 0x7632);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t bz[3][2], bs[3][2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float* at = xs + (k0 + 2 * t + half * 8) * TOKENS + n * 8 + g;
        float u = at[0], v = at[TOKENS];
#pragma unroll
        for (int part = 0; part < 3; ++part) {
          const float hu = __uint_as_float(__float_as_uint(u) & 0xffff0000u), hv = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
          bz[part][half] = __byte_perm(__float_as_uint(hu), __float_as_uint(hv), 0x7632);
          bs[part][half] = b200::pack_bf16x2(-128.f * hu, -128.f * hv);
          u -= hu;
          v -= hv;
        }
      }
#pragma unroll
      for (int part = 0; part < 3; ++part) {
        mma(y[n], as[0], as[1], as[2], as[3], bs[part][0], bs[part][1]);
        mma(y[n], az[0], az[1], az[2], az[3], bz[part][0], bz[part][1]);
      }
    }
  }

  // partial sums [wk][token][16 WM rows] over the stages of x
  constexpr int ROWS = 16 * WM;
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      part[(wk * TOKENS + n * 8 + 2 * t + (c & 1)) * ROWS + wm * 16 + g + (c >> 1) * 8] = y[n][c];
  if (p.cluster > 1)
    cluster_sync();
  else
    __syncthreads();
  const int share = ROWS / p.cluster;             // weight rows that this rank finishes
  for (int it = threadIdx.x; it < p.rows * share; it += kThreads) {
    const int token = it / share, r = rank * share + (it - token * share), n = tile * ROWS + r;
    float v = 0.f;
    for (int c = 0; c < p.cluster; ++c)
#pragma unroll
      for (int k = 0; k < WK; ++k) {
        const float* at = part + (k * TOKENS + token) * ROWS + r;
        v += p.cluster == 1 ? *at : ld_cluster(b200::smem_u32(at), c);
      }
    if (n < p.N) p.out[token * p.ldo + n] = __float2bfloat16(v);
  }
  if (p.cluster > 1) cluster_sync();              // peers may still read this block's sums
}

// Rows of up to 64 channels (one group, words in channel order): one warp per weight row and eight rows of x, a lane per word.
__global__ void __launch_bounds__(128) linear_q4_narrow_kernel(const __grid_constant__ LinearParams p) {
  const int n = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, m0 = blockIdx.y * 8;
  b200::pdl_launch_dependents();
  b200::pdl_wait();
  if (n >= p.N) return;
  const int m1 = min(p.rows - m0, 8), c = (lane & 7) * 8;
  const uint32_t a = reinterpret_cast<const uint32_t*>(p.affine)[n];
  float acc[8] = {}, v[8];
  unpack(lane < 8 ? reinterpret_cast<const uint32_t*>(p.codes)[static_cast<long long>(n) * 8 + lane] : 0u, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = fmaf(v[i], scale_of(a), least_of(a));
#pragma unroll
  for (int m = 0; m < 8; ++m) {
    if (m >= m1) break;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane < 8 && c + i < p.K) acc[m] = fmaf(__bfloat162float(p.x[(m0 + m) * p.ldx + c + i]), v[i], acc[m]);
  }
#pragma unroll
  for (int m = 0; m < 8; ++m) {
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], off);
    if (lane == 0 && m < m1) p.out[(m0 + m) * p.ldo + n] = __float2bfloat16(acc[m]);
  }
}

template <int NT, int WM>
int launch(LinearParams p, int cluster, cudaStream_t stream) {
  using S = Shape<NT, WM>;
  auto* kern = linear_q4_kernel<NT, WM>;
  p.cluster = cluster;
  const int blocks = p.width / 128, slice = (blocks + cluster - 1) / cluster;
  const int bytes = S::RING_BYTES + S::xs_bytes(slice);
  if (bytes > 226 * 1024) return b200host::RC_TOO_LARGE;
  static bool configured[b200host::kMaxDevices] = {};
  if (int rc = b200host::ensure_dynamic_smem(kern, 226 * 1024, configured)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.N + 16 * WM - 1) / (16 * WM) * cluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = b200host::pdl_enabled() ? 2 : 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, p));
}

template <int NT>
int launch_rows(const LinearParams& p, int wm, int cluster, cudaStream_t s) {
  switch (wm) {
    case 1:
      if constexpr (NT <= 2) return launch<NT, 1>(p, cluster, s);
      return b200host::RC_BAD_SHAPE;
    case 2: return launch<NT, 2>(p, cluster, s);
    case 4: return launch<NT, 4>(p, cluster, s);
    case 8: return launch<NT, 8>(p, cluster, s);
    default: return b200host::RC_BAD_SHAPE;
  }
}

}  // namespace

// out [rows, N] (row stride ldo) = x [rows, K] (ldx) * W^T, W as codes [N, width / 8] words and affine [N, width / 64] pairs.
// Blocks of 16 wm weight rows (wm 1, 2, 4 or 8), `cluster` (1, 2, 4 or 8) slices of K.
extern "C" int b200_q4_linear(const void* x, long long ldx, const void* codes, const void* affine, void* out,
                              long long ldo, int rows, int N, int K, int wm, int cluster, void* stream) {
  if (rows <= 0 || rows > 64 || N <= 0 || K <= 0 || K > (1 << 30)) return b200host::RC_BAD_SHAPE;
  if (cluster != 1 && cluster != 2 && cluster != 4 && cluster != 8) return b200host::RC_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(affine)) & 15) return b200host::RC_BAD_ALIGNMENT;
  LinearParams p{(const __nv_bfloat16*)x, ldx, ldo, (const uint8_t*)codes, (const uint8_t*)affine, (__nv_bfloat16*)out,
                 rows, N, K, row_width(K), 1, (ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0) ? 1 : 0};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (p.width == 64)
    return static_cast<int>(b200host::launch_kernel(linear_q4_narrow_kernel, dim3((N + 3) / 4, (rows + 7) / 8), dim3(128), 0,
                                                    s, b200host::pdl_enabled() != 0, p));
  if (rows <= 8) return launch_rows<1>(p, wm, cluster, s);
  if (rows <= 16) return launch_rows<2>(p, wm, cluster, s);
  if (rows <= 32) return launch_rows<4>(p, wm, cluster, s);
  return launch_rows<8>(p, wm, cluster, s);
}

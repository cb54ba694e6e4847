// y = x W^T for a few rows of x and weights held in 4 bits (quant4.cuh): x [rows, K] bf16, W [N, K], y [rows, N] bf16 with
// fp32 sums.
#include "quant4.cuh"
#include "host_util.cuh"

namespace {

using namespace q4;

struct LinearParams {
  const __nv_bfloat16* x;
  long long ldx, ldo;
  const uint32_t *codes, *affine;
  __nv_bfloat16* out;
  int rows, N, K, width;
};

// One warp per weight row and eight rows of x: a lane per word.
__global__ void __launch_bounds__(128) linear_q4_kernel(const LinearParams p) {
  const int n = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, m0 = blockIdx.y * 8;
  b200::pdl_launch_dependents();
  b200::pdl_wait();
  if (n >= p.N) return;
  const int words = p.width / 8, m1 = min(p.rows - m0, 8);
  float acc[8] = {};
  for (int w = lane; w < words; w += 32) {
    const int c = word_channel(w, p.width);
    const uint32_t a = p.affine[static_cast<long long>(n) * (p.width / kGroup) + word_group(w, p.width)];
    float v[8];
    unpack(p.codes[static_cast<long long>(n) * words + w], v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(v[i], scale_of(a), least_of(a));
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      if (m >= m1) break;
      const __nv_bfloat16* x = p.x + (m0 + m) * p.ldx + c;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < p.K) acc[m] = fmaf(__bfloat162float(x[i]), v[i], acc[m]);
    }
  }
#pragma unroll
  for (int m = 0; m < 8; ++m) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], off);
    if (lane == m && m < m1) p.out[(m0 + m) * p.ldo + n] = __float2bfloat16(acc[m]);
  }
}

}  // namespace

// out [rows, N] (row stride ldo) = x [rows, K] (ldx) * W^T, W as codes [N, width / 8] words and affine [N, width / 64] pairs.
extern "C" int b200_q4_linear(const void* x, long long ldx, const void* codes, const void* affine, void* out,
                              long long ldo, int rows, int N, int K, void* stream) {
  if (rows <= 0 || rows > 64 || N <= 0 || K <= 0 || K > (1 << 30)) return b200host::RC_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(affine)) & 15) return b200host::RC_BAD_ALIGNMENT;
  LinearParams p{(const __nv_bfloat16*)x, ldx, ldo, (const uint32_t*)codes, (const uint32_t*)affine, (__nv_bfloat16*)out,
                 rows, N, K, row_width(K)};
  return static_cast<int>(b200host::launch_kernel(linear_q4_kernel, dim3((N + 3) / 4, (rows + 7) / 8), dim3(128), 0,
                                                  reinterpret_cast<cudaStream_t>(stream), b200host::pdl_enabled() != 0, p));
}

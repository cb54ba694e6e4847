// 4-bit rows (quant4.cuh): a K/V cache that is quantised as it is written and read back, and whole matrices.
#include <math_constants.h>

#include "quant4.cuh"
#include "host_util.cuh"

namespace {

using namespace q4;

struct KvParams {
  const __nv_bfloat16* src[2];        // K, V: [B, T, Hkv, D] by strides, heads D apart (write)
  __nv_bfloat16* dst[2];              // [B, T, Hkv, D] contiguous (read)
  uint32_t* codes[2];                 // [B, pages, Hkv, page_rows, D / 8] words
  uint32_t* affine[2];                // [B, pages, Hkv, page_rows, D / 64]
  const int* start;                   // [B] or null: first row of each sequence
  long long row[2], batch[2];         // element strides of src
  int B, T, Hkv, D, pages, page_rows;
};

// index of a cache row among the rows of the pool, or -1 outside the cache
__device__ __forceinline__ long long pool_row(const KvParams& p, int b, int h, int t) {
  const long long r = (p.start ? p.start[b] : 0) + static_cast<long long>(t);
  if (r < 0 || r >= static_cast<long long>(p.pages) * p.page_rows) return -1;
  const int pg = static_cast<int>(r) / p.page_rows, in = static_cast<int>(r) - pg * p.page_rows;
  return ((static_cast<long long>(b) * p.pages + pg) * p.Hkv + h) * p.page_rows + in;
}

// A lane per word: eight lanes share a group and find its least and largest value.
__global__ void __launch_bounds__(256) kv_write_q4_kernel(const __grid_constant__ KvParams p) {
  const int per = p.D / 8, which = blockIdx.y;
  const long long total = static_cast<long long>(p.B) * p.T * p.Hkv * per;
  b200::pdl_launch_dependents();
  b200::pdl_wait();
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i0 = static_cast<long long>(blockIdx.x) * blockDim.x; i0 < total; i0 += step) {
    const long long i = min(i0 + threadIdx.x, total - 1);      // whole groups of lanes stay together for the shuffles
    const int c = static_cast<int>(i % per);
    const long long token_head = i / per;
    const int h = static_cast<int>(token_head % p.Hkv);
    const long long token = token_head / p.Hkv;
    const int t = static_cast<int>(token % p.T), b = static_cast<int>(token / p.T);
    float x[8];
    unpack_bf16(*reinterpret_cast<const uint4*>(p.src[which] + b * p.batch[which] + t * p.row[which] + h * p.D + c * 8), x);
    float least = x[0], most = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) {
      least = min_nan(least, x[j]);
      most = max_nan(most, x[j]);
    }
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) {
      least = min_nan(least, __shfl_xor_sync(0xffffffffu, least, off));
      most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, off));
    }
    const uint32_t affine = (__float_as_uint(least) & 0xffff0000u) | scale_bits(least, most);
    const uint32_t word = pack(x, affine);
    const long long r = pool_row(p, b, h, t);
    if (r < 0 || i0 + threadIdx.x >= total) continue;
    const int g = c & 7, half = c >> 3;
    p.codes[which][r * per + (per == 8 ? g : 2 * g + half)] = word;
    if (g == 0) p.affine[which][r * (per >> 3) + half] = affine;
  }
}

__global__ void __launch_bounds__(256) kv_read_q4_kernel(const __grid_constant__ KvParams p) {
  const int per = p.D / 8, which = blockIdx.y;
  const long long total = static_cast<long long>(p.B) * p.T * p.Hkv * per;
  b200::pdl_launch_dependents();
  b200::pdl_wait();
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
    const int c = static_cast<int>(i % per);
    const long long token_head = i / per;
    const int h = static_cast<int>(token_head % p.Hkv);
    const long long token = token_head / p.Hkv;
    const int t = static_cast<int>(token % p.T), b = static_cast<int>(token / p.T);
    const long long r = pool_row(p, b, h, t);
    const int g = c & 7, half = c >> 3;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r >= 0)
      v = values_bf16(p.codes[which][r * per + (per == 8 ? g : 2 * g + half)], p.affine[which][r * (per >> 3) + half]);
    *reinterpret_cast<uint4*>(p.dst[which] + i * 8) = v;
  }
}

// Whole matrices (weights, once): eight lanes per group, any number of channels and any row stride.
__global__ void __launch_bounds__(256) quantize_rows_q4_kernel(const __nv_bfloat16* __restrict__ x, long long ldx,
                                                               uint32_t* __restrict__ codes,
                                                               uint32_t* __restrict__ affine, long long rows,
                                                               int channels, int width) {
  const int words = width / 8;
  const long long total = rows * words;
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i0 = static_cast<long long>(blockIdx.x) * blockDim.x; i0 < total; i0 += step) {
    const long long i = min(i0 + threadIdx.x, total - 1);
    const long long row = i / words;
    const int c = static_cast<int>(i - row * words) * 8;      // channels in their own order: a group is eight lanes
    float f[8], least = CUDART_INF_F, most = -CUDART_INF_F;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] = 0.f;
      if (c + j < channels) {
        f[j] = __bfloat162float(x[row * ldx + c + j]);
        least = min_nan(least, f[j]);
        most = max_nan(most, f[j]);
      }
    }
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) {
      least = min_nan(least, __shfl_xor_sync(0xffffffffu, least, off));
      most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, off));
    }
    const int group = c / kGroup;
    uint32_t pair = 0, word = 0;
    if (group * kGroup < channels) {
      pair = (__float_as_uint(least) & 0xffff0000u) | scale_bits(least, most);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j >= channels) f[j] = least;                  // padding has the code 0
      word = pack(f, pair);
    }
    if (i0 + threadIdx.x >= total) continue;
    const int block = c / 128, half = (c >> 6) & 1, g = (c >> 3) & 7;
    codes[row * words + (width == 64 ? g : block * 16 + 2 * g + half)] = word;
    if (g == 0) affine[row * (width / kGroup) + group] = pair;
  }
}

__global__ void __launch_bounds__(256) dequantize_rows_q4_kernel(const uint32_t* __restrict__ codes,
                                                                 const uint32_t* __restrict__ affine,
                                                                 __nv_bfloat16* __restrict__ out, long long rows,
                                                                 int width) {
  const int words = width / 8;
  const long long total = rows * words;
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  b200::pdl_launch_dependents();
  b200::pdl_wait();
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
    const long long row = i / words;
    const int w = static_cast<int>(i - row * words);
    *reinterpret_cast<uint4*>(out + row * width + word_channel(w, width)) =
        values_bf16(codes[i], affine[row * (width / kGroup) + word_group(w, width)]);
  }
}

int blocks_for(long long items) {
  const long long blocks = (items + 255) / 256, most = 148 * 8;
  return static_cast<int>(blocks < most ? blocks : most);
}

bool kv_shape_ok(int B, int T, int Hkv, int D, int pages, int page_rows) {
  return B > 0 && T > 0 && Hkv > 0 && (D == 64 || D == 128) && pages > 0 && page_rows > 0 &&
         static_cast<long long>(pages) * page_rows <= 0x7fffffffll;
}

}  // namespace

// Rows start[b] + t (start null: t) of both caches take the 4-bit form of k, v [B, T, Hkv, D] (heads D apart, element
// strides between rows and sequences).  Rows outside the cache are left out.
extern "C" int b200_q4_kv_write(const void* k, const void* v, long long k_row, long long k_batch, long long v_row,
                                long long v_batch, void* k_codes, void* k_affine, void* v_codes, void* v_affine,
                                const void* start, int B, int T, int Hkv, int D, int pages, int page_rows, void* stream) {
  if (!kv_shape_ok(B, T, Hkv, D, pages, page_rows)) return b200host::RC_BAD_SHAPE;
  if ((k_row | k_batch | v_row | v_batch) & 7) return b200host::RC_BAD_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) return b200host::RC_BAD_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes) |
       reinterpret_cast<uintptr_t>(k_affine) | reinterpret_cast<uintptr_t>(v_affine)) & 15)
    return b200host::RC_BAD_ALIGNMENT;
  KvParams p{{(const __nv_bfloat16*)k, (const __nv_bfloat16*)v}, {nullptr, nullptr},
             {(uint32_t*)k_codes, (uint32_t*)v_codes}, {(uint32_t*)k_affine, (uint32_t*)v_affine}, (const int*)start,
             {k_row, v_row}, {k_batch, v_batch}, B, T, Hkv, D, pages, page_rows};
  return static_cast<int>(b200host::launch_kernel(
      kv_write_q4_kernel, dim3(blocks_for((long long)B * T * Hkv * (D / 8)), 2), dim3(256), 0,
      reinterpret_cast<cudaStream_t>(stream), b200host::pdl_enabled() != 0, p));
}

// The same rows as bf16 into k, v [B, T, Hkv, D] contiguous; rows outside the cache read as zeros.
extern "C" int b200_q4_kv_read(void* k, void* v, const void* k_codes, const void* k_affine, const void* v_codes,
                               const void* v_affine, const void* start, int B, int T, int Hkv, int D, int pages,
                               int page_rows, void* stream) {
  if (!kv_shape_ok(B, T, Hkv, D, pages, page_rows)) return b200host::RC_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_codes) |
       reinterpret_cast<uintptr_t>(v_codes) | reinterpret_cast<uintptr_t>(k_affine) |
       reinterpret_cast<uintptr_t>(v_affine)) & 15)
    return b200host::RC_BAD_ALIGNMENT;
  KvParams p{{nullptr, nullptr}, {(__nv_bfloat16*)k, (__nv_bfloat16*)v}, {(uint32_t*)k_codes, (uint32_t*)v_codes},
             {(uint32_t*)k_affine, (uint32_t*)v_affine}, (const int*)start, {0, 0}, {0, 0}, B, T, Hkv, D, pages,
             page_rows};
  return static_cast<int>(b200host::launch_kernel(
      kv_read_q4_kernel, dim3(blocks_for((long long)B * T * Hkv * (D / 8)), 2), dim3(256), 0,
      reinterpret_cast<cudaStream_t>(stream), b200host::pdl_enabled() != 0, p));
}

// x [rows, channels] bf16 with row stride ldx -> codes [rows, width / 8] words, affine [rows, width / 64] pairs.
extern "C" int b200_q4_quantize_rows(const void* x, long long ldx, void* codes, void* affine, long long rows,
                                     int channels, void* stream) {
  if (rows <= 0 || channels <= 0 || channels > (1 << 30)) return b200host::RC_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(affine)) & 15) return b200host::RC_BAD_ALIGNMENT;
  const int width = row_width(channels);
  quantize_rows_q4_kernel<<<blocks_for(rows * (width / 8)), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      (const __nv_bfloat16*)x, ldx, (uint32_t*)codes, (uint32_t*)affine, rows, channels, width);
  return static_cast<int>(cudaGetLastError());
}

// codes, affine -> out [rows, width] bf16 contiguous (padding reads as zeros: its pair is zero).
extern "C" int b200_q4_dequantize_rows(const void* codes, const void* affine, void* out, long long rows, int width,
                                       void* stream) {
  if (rows <= 0 || width <= 0 || (width != 64 && width % 128)) return b200host::RC_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(affine) | reinterpret_cast<uintptr_t>(out)) & 15)
    return b200host::RC_BAD_ALIGNMENT;
  return static_cast<int>(b200host::launch_kernel(
      dequantize_rows_q4_kernel, dim3(blocks_for(rows * (width / 8))), dim3(256), 0,
      reinterpret_cast<cudaStream_t>(stream), b200host::pdl_enabled() != 0, (const uint32_t*)codes,
      (const uint32_t*)affine, (__nv_bfloat16*)out, rows, width));
}

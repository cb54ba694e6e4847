// 4-bit rows (quant4.cuh): a K/V cache that is quantised as it is written and read back, and whole matrices.
#include <math_constants.h>
#include <string.h>

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
  long long batch[2];                 // element strides of src
  int row[2];
  int T, Hkv, pages, page_rows, blocks;   // blocks of a sequence
  Divisor per_block, per_token, per_page;
};

constexpr uint32_t kThreads = 256;
// A lane has eight channels of every group of its row (words 2 g and 2 g + 1 of a row of 128), so that placing it, which costs
// as much as a word's codes, is done once for both.  Lanes of a thread, their loads all under way at once:
template <int D>
constexpr int items() { return D == 128 ? 2 : 4; }

// A thread's items among those of a sequence's new rows, counted over (token, head, g): this one, and 256 further on.
struct Walk {
  uint32_t token, e;                  // e: item of the token's row over all heads
  __device__ __forceinline__ Walk(const KvParams& p, uint32_t j) : token(p.per_token.of(j)), e(j - token * p.per_token.d) {}
  __device__ __forceinline__ void next(const KvParams& p, uint32_t tokens, uint32_t rest) {
    token += tokens;
    e += rest;
    if (e >= p.per_token.d) {
      e -= p.per_token.d;
      ++token;
    }
  }
};

// Row of a sequence in its cache as 32 bits without sign: whatever start + token is, it is below the capacity only if it is a
// row of the cache (both are below 2^31).
__device__ __forceinline__ uint32_t row_of(int first, const Walk& at) { return static_cast<uint32_t>(first) + at.token; }
// Pool row of a token's head.
__device__ __forceinline__ uint64_t pool_row(const KvParams& p, uint64_t seq_row, uint32_t r, const Walk& at) {
  const uint32_t pg = p.per_page.of(r), in = r - pg * p.per_page.d;
  return seq_row + in + static_cast<uint64_t>(pg * p.Hkv + at.e / 8) * p.per_page.d;
}

// Quantise as it is written: eight lanes have a row's head and find the least and largest value of its groups in bf16 (which
// they are).  Bound by the arithmetic, 20 instructions a channel: eight prompts of 4096 rows of 8 heads of 128 (172 MB read
// and written, 26 us at the copy bandwidth) take 47 us, and 26 us to read back.
template <int D>
__global__ void __launch_bounds__(kThreads) kv_write_q4_kernel(const __grid_constant__ KvParams p) {
  constexpr int ITEMS = items<D>(), GROUPS = D / 64;
  const int which = blockIdx.y, b = static_cast<int>(p.per_block.of(blockIdx.x)), block = blockIdx.x - b * p.blocks;
  b200::pdl_launch_dependents();
  b200::pdl_wait();
  const int first = p.start ? p.start[b] : 0;
  const uint32_t total = static_cast<uint32_t>(p.T) * p.per_token.d, j0 = block * (kThreads * ITEMS) + threadIdx.x;
  const uint32_t tokens = p.per_token.of(kThreads), rest = kThreads - tokens * p.per_token.d;
  const __nv_bfloat16* src = p.src[which] + b * p.batch[which];
  uint4 v[ITEMS][GROUPS];
  {
    Walk at(p, j0);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k, at.next(p, tokens, rest)) {  // beyond the rows: the last one's, whose groups are whole too
      const __nv_bfloat16* row = src + static_cast<long long>(min(at.token, p.T - 1u)) * p.row[which] + (at.e / 8) * D +
                                 (at.e & 7) * 8;
#pragma unroll
      for (int h = 0; h < GROUPS; ++h) v[k][h] = *reinterpret_cast<const uint4*>(row + 64 * h);
    }
  }
  const uint64_t seq_row = static_cast<uint64_t>(b) * p.pages * p.Hkv * p.page_rows;
  const uint32_t capacity = static_cast<uint32_t>(p.pages) * p.page_rows;
  Walk at(p, j0);
#pragma unroll
  for (int k = 0; k < ITEMS; ++k, at.next(p, tokens, rest)) {
    const uint32_t j = j0 + k * kThreads;
    if (j - (threadIdx.x & 31) >= total) break;           // the whole warp is beyond
    uint32_t word[GROUPS], affine[GROUPS];
#pragma unroll
    for (int h = 0; h < GROUPS; ++h) {
      __nv_bfloat162 w[4];
      memcpy(w, &v[k][h], 16);
      const __nv_bfloat162 lo = __hmin2_nan(__hmin2_nan(w[0], w[1]), __hmin2_nan(w[2], w[3]));
      const __nv_bfloat162 hi = __hmax2_nan(__hmax2_nan(w[0], w[1]), __hmax2_nan(w[2], w[3]));
      // (least, -largest), so that one minimum serves both
      __nv_bfloat162 m = __halves2bfloat162(__hmin_nan(lo.x, lo.y), __hneg(__hmax_nan(hi.x, hi.y)));
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) m = __hmin2_nan(m, __shfl_xor_sync(0xffffffffu, m, off));
      const float least = __low2float(m), most = -__high2float(m);
      affine[h] = (__float_as_uint(least) & 0xffff0000u) | scale_bits(least, most);
      float x[8];
      unpack_bf16(v[k][h], x);
      word[h] = pack(x, affine[h]);
    }
    const uint32_t r = row_of(first, at), g = at.e & 7;
    if (j >= total || r >= capacity) continue;
    const uint64_t row = pool_row(p, seq_row, r, at);
    if constexpr (GROUPS == 2) {
      reinterpret_cast<uint2*>(p.codes[which])[row * 8 + g] = make_uint2(word[0], word[1]);
      if (g == 0) reinterpret_cast<uint2*>(p.affine[which])[row] = make_uint2(affine[0], affine[1]);
    } else {
      p.codes[which][row * 8 + g] = word[0];
      if (g == 0) p.affine[which][row] = affine[0];
    }
  }
}

// Read back.
template <int D>
__global__ void __launch_bounds__(kThreads) kv_read_q4_kernel(const __grid_constant__ KvParams p) {
  constexpr int ITEMS = items<D>(), GROUPS = D / 64;
  const int which = blockIdx.y, b = static_cast<int>(p.per_block.of(blockIdx.x)), block = blockIdx.x - b * p.blocks;
  b200::pdl_launch_dependents();
  b200::pdl_wait();
  const int first = p.start ? p.start[b] : 0;
  const uint32_t total = static_cast<uint32_t>(p.T) * p.per_token.d, j0 = block * (kThreads * ITEMS) + threadIdx.x;
  const uint32_t tokens = p.per_token.of(kThreads), rest = kThreads - tokens * p.per_token.d;
  const uint64_t seq_row = static_cast<uint64_t>(b) * p.pages * p.Hkv * p.page_rows;
  const uint32_t capacity = static_cast<uint32_t>(p.pages) * p.page_rows;
  uint32_t word[ITEMS][GROUPS], affine[ITEMS][GROUPS];
  Walk at(p, j0);
#pragma unroll
  for (int k = 0; k < ITEMS; ++k, at.next(p, tokens, rest)) {
    const uint32_t r = row_of(first, at), g = at.e & 7;
    const bool there = j0 + k * kThreads < total && r < capacity;   // a row that the cache does not have reads as zeros
    const uint64_t row = there ? pool_row(p, seq_row, r, at) : 0;
    if constexpr (GROUPS == 2) {
      const uint2 w = there ? reinterpret_cast<const uint2*>(p.codes[which])[row * 8 + g] : make_uint2(0, 0);
      const uint2 a = there ? reinterpret_cast<const uint2*>(p.affine[which])[row] : make_uint2(0, 0);
      word[k][0] = w.x, word[k][1] = w.y, affine[k][0] = a.x, affine[k][1] = a.y;
    } else {
      word[k][0] = there ? p.codes[which][row * 8 + g] : 0u;
      affine[k][0] = there ? p.affine[which][row] : 0u;
    }
  }
  uint32_t mask, magic;
  opaque_masks(mask, magic);
  // an item's first chunk of eight channels among the sequence's: the item with the groups' chunks counted in
  uint4* to = reinterpret_cast<uint4*>(p.dst[which]) + static_cast<long long>(b) * total * GROUPS;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const uint32_t j = j0 + k * kThreads;
    if (j >= total) break;
#pragma unroll
    for (int h = 0; h < GROUPS; ++h)
      to[static_cast<uint64_t>(j / 8) * (8 * GROUPS) + 8 * h + (j & 7)] = values_bf16(word[k][h], affine[k][h], mask, magic);
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

// Codes and pairs may be the predecessor's work: only the output is said to be alone.
__global__ void __launch_bounds__(256) dequantize_rows_q4_kernel(const uint32_t* codes, const uint32_t* affine,
                                                                 __nv_bfloat16* __restrict__ out, long long rows,
                                                                 int width) {
  const int words = width / 8;
  const long long total = rows * words;
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  uint32_t mask, magic;
  opaque_masks(mask, magic);
  b200::pdl_launch_dependents();
  b200::pdl_wait();
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
    const long long row = i / words;
    const int w = static_cast<int>(i - row * words);
    *reinterpret_cast<uint4*>(out + row * width + word_channel(w, width)) =
        values_bf16(codes[i], affine[row * (width / kGroup) + word_group(w, width)], mask, magic);
  }
}

int blocks_for(long long items) {
  const long long blocks = (items + 255) / 256, most = 148 * 8;
  return static_cast<int>(blocks < most ? blocks : most);
}

bool kv_shape_ok(int B, int T, int Hkv, int D, int pages, int page_rows) {
  return B > 0 && T > 0 && Hkv > 0 && (D == 64 || D == 128) && pages > 0 && page_rows > 0 &&
         static_cast<long long>(pages) * page_rows <= 0x7fffffffll &&
         static_cast<long long>(pages) * Hkv <= 0x7fffffffll && static_cast<long long>(T) * Hkv * (D / 8) <= 0x7ffff000ll &&
         static_cast<long long>(B) * (static_cast<long long>(T) * Hkv * 8 / (kThreads * 2) + 1) <= 0x7fffffffll;
}

template <typename Kern>
int launch_kv(Kern* kern64, Kern* kern128, KvParams p, int B, int D, void* stream) {
  const uint32_t per = static_cast<uint32_t>(p.Hkv) * 8, block = kThreads * (D == 64 ? items<64>() : items<128>());
  p.blocks = static_cast<int>((static_cast<uint32_t>(p.T) * per + block - 1) / block);
  p.per_block = Divisor(p.blocks);
  p.per_token = Divisor(per);
  p.per_page = Divisor(p.page_rows);
  return static_cast<int>(b200host::launch_kernel(D == 64 ? kern64 : kern128, dim3(B * p.blocks, 2), dim3(kThreads), 0,
                                                  reinterpret_cast<cudaStream_t>(stream), b200host::pdl_enabled() != 0, p));
}

}  // namespace

// Rows start[b] + t (start null: t) of both caches take the 4-bit form of k, v [B, T, Hkv, D] (heads D apart, element
// strides between rows and sequences).  Rows outside the cache are left out.
extern "C" int b200_q4_kv_write(const void* k, const void* v, long long k_row, long long k_batch, long long v_row,
                                long long v_batch, void* k_codes, void* k_affine, void* v_codes, void* v_affine,
                                const void* start, int B, int T, int Hkv, int D, int pages, int page_rows, void* stream) {
  if (!kv_shape_ok(B, T, Hkv, D, pages, page_rows)) return b200host::RC_BAD_SHAPE;
  if ((k_row | k_batch | v_row | v_batch) & 7) return b200host::RC_BAD_ALIGNMENT;
  if (k_row < 0 || v_row < 0 || k_row > 0x7fffffff || v_row > 0x7fffffff) return b200host::RC_TOO_LARGE;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) return b200host::RC_BAD_ALIGNMENT;
  if (!rows_aligned(k_codes, k_affine, D) || !rows_aligned(v_codes, v_affine, D)) return b200host::RC_BAD_ALIGNMENT;
  KvParams p{{(const __nv_bfloat16*)k, (const __nv_bfloat16*)v}, {nullptr, nullptr},
             {(uint32_t*)k_codes, (uint32_t*)v_codes}, {(uint32_t*)k_affine, (uint32_t*)v_affine}, (const int*)start,
             {k_batch, v_batch}, {(int)k_row, (int)v_row}, T, Hkv, pages, page_rows, 0, {}, {}, {}};
  return launch_kv(kv_write_q4_kernel<64>, kv_write_q4_kernel<128>, p, B, D, stream);
}

// The same rows as bf16 into k, v [B, T, Hkv, D] contiguous; rows outside the cache read as zeros.
extern "C" int b200_q4_kv_read(void* k, void* v, const void* k_codes, const void* k_affine, const void* v_codes,
                               const void* v_affine, const void* start, int B, int T, int Hkv, int D, int pages,
                               int page_rows, void* stream) {
  if (!kv_shape_ok(B, T, Hkv, D, pages, page_rows)) return b200host::RC_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) return b200host::RC_BAD_ALIGNMENT;
  if (!rows_aligned(k_codes, k_affine, D) || !rows_aligned(v_codes, v_affine, D)) return b200host::RC_BAD_ALIGNMENT;
  KvParams p{{nullptr, nullptr}, {(__nv_bfloat16*)k, (__nv_bfloat16*)v}, {(uint32_t*)k_codes, (uint32_t*)v_codes},
             {(uint32_t*)k_affine, (uint32_t*)v_affine}, (const int*)start, {0, 0}, {0, 0}, T, Hkv, pages,
             page_rows, 0, {}, {}, {}};
  return launch_kv(kv_read_q4_kernel<64>, kv_read_q4_kernel<128>, p, B, D, stream);
}

// x [rows, channels] bf16 with row stride ldx -> codes [rows, width / 8] words, affine [rows, width / 64] pairs.
extern "C" int b200_q4_quantize_rows(const void* x, long long ldx, void* codes, void* affine, long long rows,
                                     int channels, void* stream) {
  if (rows <= 0 || channels <= 0 || channels > (1 << 30)) return b200host::RC_BAD_SHAPE;
  const int width = row_width(channels);
  if (!rows_aligned(codes, affine, width)) return b200host::RC_BAD_ALIGNMENT;
  quantize_rows_q4_kernel<<<blocks_for(rows * (width / 8)), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      (const __nv_bfloat16*)x, ldx, (uint32_t*)codes, (uint32_t*)affine, rows, channels, width);
  return static_cast<int>(cudaGetLastError());
}

// codes, affine -> out [rows, width] bf16 contiguous (padding reads as zeros: its pair is zero).
extern "C" int b200_q4_dequantize_rows(const void* codes, const void* affine, void* out, long long rows, int width,
                                       void* stream) {
  if (rows <= 0 || width <= 0 || (width != 64 && width % 128)) return b200host::RC_BAD_SHAPE;
  if (!rows_aligned(codes, affine, width) || (reinterpret_cast<uintptr_t>(out) & 15)) return b200host::RC_BAD_ALIGNMENT;
  return static_cast<int>(b200host::launch_kernel(
      dequantize_rows_q4_kernel, dim3(blocks_for(rows * (width / 8))), dim3(256), 0,
      reinterpret_cast<cudaStream_t>(stream), b200host::pdl_enabled() != 0, (const uint32_t*)codes,
      (const uint32_t*)affine, (__nv_bfloat16*)out, rows, width));
}

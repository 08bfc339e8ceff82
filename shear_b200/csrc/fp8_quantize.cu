// FP8 codes (E4M3) with a power-of-two scale (E8M0) for each block of 128
// values, along rows, along columns, or both from one read.
//
// The scale of a block is the least s = 2^e with max|x| / s <= 448.  With
// max|x| = f * 2^p, 1 <= f < 2, and 448 = 1.75 * 2^8: e = p - 8 if f <= 1.75,
// else p - 7, read off the maximum's bits.  x / s is exact (a power of two),
// so each value is rounded once, by the conversion.  Powers of two lose
// nothing against a free scale but up to a binade of the smallest codes'
// range, and they are what the tensor cores apply by themselves.
#include "train_common.cuh"

namespace tessa {
namespace train {

// Bits of |x|, 0 where x is NaN or infinite (it takes no part in the maximum).
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// Scale byte of a block whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  if (amax == 0u) return 0u;
  int e;
  uint32_t frac;
  if (amax >= 0x00800000u) {
    e = (int)(amax >> 23) - 127;
    frac = amax & 0x007fffffu;
  } else {  // subnormal: normalise
    const int lead = __clz(amax) - 8;
    e = -126 - lead;
    frac = (amax << lead) & 0x007fffffu;
  }
  const int p = e - (frac <= 0x00600000u ? 8 : 7) + 127;
  return p < 0 ? 0u : (uint32_t)p;
}

// 2^-(byte - 127), exactly (byte 254, the largest that occurs, would need
// 2^-127: scale bytes stop at 127 + 127 - 7 = 247).
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Two values as E4M3 codes, lo in the low byte; NaN and infinities as NaN.
__device__ __forceinline__ uint32_t codes2(float lo, float hi) {
  lo = fabsf(lo) < INFINITY ? lo : NAN;
  hi = fabsf(hi) < INFINITY ? hi : NAN;
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t codes4(const float (&x)[4]) { return codes2(x[0], x[1]) | codes2(x[2], x[3]) << 16; }

// Four consecutive values of a row, zeros past `cols`.
template <class T, int VE>
__device__ __forceinline__ void load4(const T* row, uint64_t col, uint64_t cols, float (&x)[4]) {
  if constexpr (VE == 4) {
    if (col < cols) {  // cols is a multiple of 4 here
      const Vec<T, 4> v = *reinterpret_cast<const Vec<T, 4>*>(row + col);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = to_f32(v.v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = col + i < cols ? to_f32(row[col + i]) : 0.0f;
  }
}

// Codes along rows: a warp takes a block of 128 of a row, four values a lane.
template <class T, int VE>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const tessa_fp8_quantize_args a, uint32_t blocks,
                                                            uint32_t code_cols, uint32_t scale_cols) {
  const uint32_t lane = threadIdx.x % 32u;
  const uint64_t total = a.rows * scale_cols, step = (uint64_t)gridDim.x * 8u;
  for (uint64_t w = (uint64_t)blockIdx.x * 8u + threadIdx.x / 32u; w < total; w += step) {
    const uint64_t row = w / scale_cols;
    const uint32_t b = (uint32_t)(w % scale_cols);
    uint32_t byte = 0;
    if (b < blocks) {
      const uint64_t col = (uint64_t)b * 128u + lane * 4u;
      float x[4];
      load4<T, VE>(static_cast<const T*>(a.x) + row * a.stride, col, a.cols, x);
      const uint32_t m = max(max(finite_bits(x[0]), finite_bits(x[1])), max(finite_bits(x[2]), finite_bits(x[3])));
      byte = scale_byte(__reduce_max_sync(0xffffffffu, m));
      const float inv = inverse_scale(byte);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] *= inv;
      if (col < code_cols) *reinterpret_cast<uint32_t*>(a.codes + row * code_cols + col) = codes4(x);
    }
    if (lane == 0) a.scales[row * scale_cols + b] = (uint8_t)byte;
  }
}

// Codes along columns, and along rows too where asked: a block takes a tile of
// 128 x 128 through shared memory, one thread a column half (64 rows).
template <class T, int VE, bool ROWS>
__global__ void __launch_bounds__(256) quantize_tiles_kernel(const tessa_fp8_quantize_args a, uint32_t col_tiles,
                                                             uint32_t row_tiles, uint32_t code_cols,
                                                             uint32_t scale_cols, uint32_t code_rows,
                                                             uint32_t scale_rows) {
  extern __shared__ __align__(16) uint8_t tile_bytes[];
  T* tile = reinterpret_cast<T*>(tile_bytes);  // 128 x 128
  __shared__ uint32_t half_max[2][128];
  const uint32_t bx = blockIdx.x % col_tiles, by = blockIdx.x / col_tiles;
  const uint64_t r0 = (uint64_t)by * 128u, c0 = (uint64_t)bx * 128u;
  const uint32_t tid = threadIdx.x, warp = tid / 32u, lane = tid % 32u;
  const uint64_t col = c0 + lane * 4u;
#pragma unroll 4
  for (uint32_t i = 0; i < 16; ++i) {
    const uint32_t r = i * 8u + warp;
    const uint64_t row = r0 + r;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (row < a.rows) load4<T, VE>(static_cast<const T*>(a.x) + row * a.stride, col, a.cols, x);
    Vec<T, 4> v;
#pragma unroll
    for (int q = 0; q < 4; ++q) v.v[q] = from_f32<T>(x[q]);
    *reinterpret_cast<Vec<T, 4>*>(tile + r * 128u + lane * 4u) = v;
    if constexpr (ROWS) {
      const uint32_t m = max(max(finite_bits(x[0]), finite_bits(x[1])), max(finite_bits(x[2]), finite_bits(x[3])));
      const uint32_t byte = scale_byte(__reduce_max_sync(0xffffffffu, m));
      const float inv = inverse_scale(byte);
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] *= inv;
      if (row < a.rows) {
        if (col < code_cols) *reinterpret_cast<uint32_t*>(a.codes + row * code_cols + col) = codes4(x);
        // the last tile of a row also clears the bytes past the last block
        const uint32_t last = bx == col_tiles - 1u ? scale_cols : bx + 1u;
        if (bx + lane < last) a.scales[row * scale_cols + bx + lane] = lane == 0 ? (uint8_t)byte : 0;
      }
    }
  }
  __syncthreads();
  const uint32_t c = tid % 128u, half = tid / 128u;
  const T* mine = tile + half * 64u * 128u + c;
  uint32_t m = 0;
#pragma unroll 16
  for (uint32_t r = 0; r < 64; ++r) m = max(m, finite_bits(to_f32(mine[r * 128u])));
  half_max[half][c] = m;
  __syncthreads();
  if (c0 + c >= a.cols) return;
  const uint32_t byte = scale_byte(max(half_max[0][c], half_max[1][c]));
  const float inv = inverse_scale(byte);
  uint8_t* out = a.codes_t + (c0 + c) * code_rows + r0 + half * 64u;
#pragma unroll
  for (uint32_t q = 0; q < 4; ++q) {
    if (r0 + half * 64u + q * 16u >= code_rows) break;
    uint32_t w[4];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      float x[4];
#pragma unroll
      for (uint32_t v = 0; v < 4; ++v) x[v] = to_f32(mine[(q * 16u + u * 4u + v) * 128u]) * inv;
      w[u] = codes4(x);
    }
    *reinterpret_cast<uint4*>(out + q * 16u) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (half == 0) {
    const uint32_t last = by == row_tiles - 1u ? scale_rows : by + 1u;
    for (uint32_t b = by; b < last; ++b) a.scales_t[(c0 + c) * scale_rows + b] = b == by ? (uint8_t)byte : 0;
  }
}

template <class T, int VE, bool ROWS>
cudaError_t launch_tiles(const tessa_fp8_quantize_args& a, int device, uint32_t cc, uint32_t sc, uint32_t cr, uint32_t sr,
                         cudaStream_t stream) {
  const uint32_t smem = 128u * 128u * sizeof(T);
  static SmemRaised raised;
  cudaError_t e = raise_smem(quantize_tiles_kernel<T, VE, ROWS>, device, (int)smem, raised);
  if (e != cudaSuccess) return e;
  const uint32_t ct = (uint32_t)div_up(a.cols, 128), rt = (uint32_t)div_up(a.rows, 128);
  quantize_tiles_kernel<T, VE, ROWS><<<ct * rt, 256, smem, stream>>>(a, ct, rt, cc, sc, cr, sr);
  return cudaGetLastError();
}

}  // namespace train

cudaError_t launch_quantize_fp8(const tessa_fp8_quantize_args& a, const AsyncCtx& c, cudaStream_t stream) {
  using namespace train;
  const uint32_t code_cols = (uint32_t)div_up(a.cols, 16) * 16u, scale_cols = (uint32_t)div_up(a.cols, 512) * 4u;
  const uint32_t code_rows = (uint32_t)div_up(a.rows, 16) * 16u, scale_rows = (uint32_t)div_up(a.rows, 512) * 4u;
  const bool vec = vector_elems(a.x, a.rows, a.cols, a.stride, type_bytes(a.dtype), 4) == 4;
  return with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    if (a.codes_t) {
      if (a.codes)
        return vec ? launch_tiles<T, 4, true>(a, c.device, code_cols, scale_cols, code_rows, scale_rows, stream)
                   : launch_tiles<T, 1, true>(a, c.device, code_cols, scale_cols, code_rows, scale_rows, stream);
      return vec ? launch_tiles<T, 4, false>(a, c.device, code_cols, scale_cols, code_rows, scale_rows, stream)
                 : launch_tiles<T, 1, false>(a, c.device, code_cols, scale_cols, code_rows, scale_rows, stream);
    }
    const uint32_t blocks = (uint32_t)div_up(a.cols, 128);
    const uint64_t want = div_up(a.rows * scale_cols, 8), most = (uint64_t)c.sm_count * 32;
    const uint32_t grid = (uint32_t)(want < most ? want : most);
    if (vec)
      quantize_rows_kernel<T, 4><<<grid, 256, 0, stream>>>(a, blocks, code_cols, scale_cols);
    else
      quantize_rows_kernel<T, 1><<<grid, 256, 0, stream>>>(a, blocks, code_cols, scale_cols);
    return cudaGetLastError();
  });
}

}  // namespace tessa

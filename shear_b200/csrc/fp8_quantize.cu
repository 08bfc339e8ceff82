// FP8 codes (E4M3) with a power-of-two scale (E8M0) for each block of 128
// values, along rows, along columns, or both from one read.
//
// The scale of a block is the least s = 2^e with max|x| / s <= 448.  With
// max|x| = f * 2^p, 1 <= f < 2, and 448 = 1.75 * 2^8: e = p - 8 if f <= 1.75,
// else p - 7, read off the maximum's bits.  x / s is exact (a power of two),
// so each value is rounded once, by the conversion.  Powers of two lose
// nothing against a free scale but up to a binade of the smallest codes'
// range, and they are what the tensor cores apply by themselves.
#include <cstring>

#include "train_common.cuh"

namespace tessa {
namespace train {

// 32 bits of a row: two values of 16 bits, or one of 32.  Magnitudes are
// compared as integers, both halves at once.
template <class T>
struct Words {
  static constexpr uint32_t kValues = 2, kAbs = 0x7fff7fffu;
  static constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
  // NaN in place of infinities and NaN, so that neither is clamped to 448.
  static __device__ __forceinline__ uint32_t only_nan(uint32_t w) {
    return ((w & 0x7fffu) >= kInf ? 0x7fffu : w & 0xffffu) | ((w >> 16 & 0x7fffu) >= kInf ? 0x7fff0000u : w & 0xffff0000u);
  }
  // Magnitudes of the finite values.
  static __device__ __forceinline__ uint32_t finite(uint32_t w) {
    return ((w & 0x7fffu) >= kInf ? 0u : w & 0x7fffu) | ((w & 0x7fff0000u) >= kInf << 16 ? 0u : w & 0x7fff0000u);
  }
  static __device__ __forceinline__ uint32_t value(uint32_t w, uint32_t i) { return i ? w >> 16 : w & 0xffffu; }
  static __device__ __forceinline__ uint32_t largest(uint32_t w) { return max(w & 0xffffu, w >> 16); }
  static __device__ __forceinline__ float f32(uint32_t w, uint32_t i) {
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)value(w, i)));
    else return __uint_as_float(i ? w & 0xffff0000u : w << 16);
  }
};
template <>
struct Words<float> {
  static constexpr uint32_t kValues = 1, kAbs = 0x7fffffffu, kInf = 0x7f800000u;
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
  static __device__ __forceinline__ uint32_t only_nan(uint32_t w) { return (w & kAbs) >= kInf ? kAbs : w; }
  static __device__ __forceinline__ uint32_t finite(uint32_t w) { return (w & kAbs) >= kInf ? 0u : w & kAbs; }
  static __device__ __forceinline__ uint32_t value(uint32_t w, uint32_t) { return w; }
  static __device__ __forceinline__ uint32_t largest(uint32_t w) { return w; }
  static __device__ __forceinline__ float f32(uint32_t w, uint32_t) { return __uint_as_float(w); }
};

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

// Two values as E4M3 codes, lo in the low byte; NaN as NaN.
__device__ __forceinline__ uint32_t codes2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// 16 values of a block of 128: eight lanes hold the block, lane j its pieces
// j, j + 8, ... of 16 bytes, so that all maths is a lane's own but for three
// exchanges.
template <class T>
struct Share {
  using W = Words<T>;
  static constexpr uint32_t kPiece = 16 / sizeof(T), kPieces = 16 / kPiece, kWords = 16 / W::kValues;
  uint32_t w[kWords];

  // `left`: values from the block's first to the row's end, zeros beyond (VE of
  // them can be read at a time, and `left` is a multiple of VE).
  template <int VE>
  __device__ __forceinline__ void load(const T* block, uint32_t j, uint32_t left) {
#pragma unroll
    for (uint32_t p = 0; p < kPieces; ++p) {
      Vec<T, kPiece> v;
      const uint32_t at = (p * 8u + j) * kPiece;
#pragma unroll
      for (uint32_t i = 0; i < kPiece; i += VE) {
        Vec<T, VE> x;
        if (at + i < left) {
          x = *reinterpret_cast<const Vec<T, VE>*>(block + at + i);
        } else {
#pragma unroll
          for (int u = 0; u < VE; ++u) x.v[u] = from_f32<T>(0.0f);
        }
#pragma unroll
        for (int u = 0; u < VE; ++u) v.v[i + u] = x.v[u];
      }
      memcpy(w + p * 4u, &v, 16);
    }
  }
  // Bits of the block's largest finite magnitude; infinities become NaN.
  __device__ __forceinline__ uint32_t block_magnitude() {
    uint32_t m = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWords; ++i) m = W::larger(m, w[i] & W::kAbs);
    m = over_lanes(W::largest(m));
    if (__any_sync(0xffffffffu, m >= W::kInf)) {
      m = 0;
#pragma unroll
      for (uint32_t i = 0; i < kWords; ++i) {
        m = W::larger(m, W::finite(w[i]));
        w[i] = W::only_nan(w[i]);
      }
      m = over_lanes(W::largest(m));
    }
    return m;
  }
  // Codes of piece p, four a word.
  __device__ __forceinline__ void store(uint8_t* block, uint32_t j, uint32_t left, float inv) const {
#pragma unroll
    for (uint32_t p = 0; p < kPieces; ++p) {
      Vec<uint32_t, kPiece / 4> c;
#pragma unroll
      for (uint32_t i = 0; i < kPiece; i += 4) {
        float x[4];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) x[u] = W::f32(w[(p * kPiece + i + u) / W::kValues], u % W::kValues) * inv;
        c.v[i / 4] = codes2(x[0], x[1]) | codes2(x[2], x[3]) << 16;
      }
      const uint32_t at = (p * 8u + j) * kPiece;
      if (at < left) *reinterpret_cast<Vec<uint32_t, kPiece / 4>*>(block + at) = c;
    }
  }

 private:
  static __device__ __forceinline__ uint32_t over_lanes(uint32_t m) {
#pragma unroll
    for (uint32_t o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
  }
};

// The magnitude's bits as a f32's.
template <class T>
__device__ __forceinline__ uint32_t f32_bits(uint32_t m) {
  return __float_as_uint(Words<T>::f32(m, 0));
}

// Codes along rows: eight lanes a block of 128, four blocks (of one row or of
// several) a warp.  Bound by memory, with 70 % of the issue slots taken: 200000 x
// 768 bf16 79 us (5.8 TB/s; a warp to a block, four values a lane, took 115), 777
// x 5003, which only single values can read, 5.0.
template <class T, int VE>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const tessa_fp8_quantize_args a, uint32_t total,
                                                            uint32_t blocks, uint32_t code_cols, uint32_t scale_cols) {
  const uint32_t item = blockIdx.x * 32u + threadIdx.x / 8u, j = threadIdx.x % 8u;
  const uint32_t row = item / blocks, block = item - row * blocks;
  const bool in = item < total;
  Share<T> x;
  x.template load<VE>(static_cast<const T*>(a.x) + (in ? row * a.stride + block * 128u : 0u), j,
                      in ? (uint32_t)a.cols - block * 128u : 0u);
  const uint32_t byte = scale_byte(f32_bits<T>(x.block_magnitude()));
  if (!in) return;
  x.store(a.codes + (uint64_t)row * code_cols + block * 128u, j, code_cols - block * 128u, inverse_scale(byte));
  // and behind a row's last block the zeros that end its scales
  const uint32_t end = block == blocks - 1u ? scale_cols - block : 1u;
  if (j < end) a.scales[(uint64_t)row * scale_cols + block + j] = j == 0u ? (uint8_t)byte : 0;
}

// Codes along columns, and along rows too where asked: a block brings a tile of
// 128 x 128 to shared memory, all of it under way at once where rows can be
// read some values at a time.  Rows are a warp's, four side by side as above.
// Down the columns a thread holds a word's columns (two of 16 bits) over a
// quarter of the rows (a half for f32) in registers, so that shared memory is
// read once and both columns' maxima are one maximum; the quarters meet in
// shared memory.  200000 x 768 bf16: columns 73 us (6.3 TB/s), both 111 (5.5
// TB/s); with 16-byte stores straight to the columns, a line each, 113 and 155.
template <class T, int VE, bool ROWS>
__global__ void __launch_bounds__(256) quantize_tiles_kernel(const tessa_fp8_quantize_args a, uint32_t col_tiles,
                                                             uint32_t row_tiles, uint32_t code_cols,
                                                             uint32_t scale_cols, uint32_t code_rows,
                                                             uint32_t scale_rows) {
  using W = Words<T>;
  constexpr uint32_t kRowWords = 128u / W::kValues;  // words of a tile's row
  constexpr uint32_t kParts = 256u / kRowWords, kHeld = 128u / kParts;
  extern __shared__ __align__(16) uint32_t tile[];   // 128 x kRowWords
  __shared__ uint32_t part_max[kParts][kRowWords];
  const uint32_t bx = blockIdx.x % col_tiles, by = blockIdx.x / col_tiles;
  const uint64_t r0 = (uint64_t)by * 128u, c0 = (uint64_t)bx * 128u;
  const uint32_t tid = threadIdx.x, warp = tid / 32u, lane = tid % 32u;
  constexpr uint32_t kPiece = Share<T>::kPiece;
  // a warp brings and quantizes 16 rows
  if constexpr (VE > 1) {
#pragma unroll
    for (uint32_t i = 0; i < 16u * 128u / (32u * VE); ++i) {
      const uint32_t at = i * 32u + lane, r = warp * 16u + at / (128u / VE), q = at % (128u / VE) * VE;
      const bool in = r0 + r < a.rows && c0 + q < a.cols;
      const T* src = static_cast<const T*>(a.x) + (in ? (r0 + r) * a.stride + c0 + q : 0u);
      constexpr uint32_t kBytes = VE * sizeof(T);
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(
                       smem_u32(reinterpret_cast<T*>(tile) + r * 128u + q)),
                   "l"(src), "n"(kBytes), "r"(in ? kBytes : 0u)
                   : "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
#pragma unroll 16
    for (uint32_t i = 0; i < 64; ++i) {
      const uint32_t r = warp * 16u + i / 4u, q = i % 4u * 32u + lane;
      reinterpret_cast<T*>(tile)[r * 128u + q] = r0 + r < a.rows && c0 + q < a.cols
                                                     ? static_cast<const T*>(a.x)[(r0 + r) * a.stride + c0 + q]
                                                     : from_f32<T>(0.0f);
    }
  }
  if constexpr (ROWS) {
    __syncwarp();  // a warp's rows are its own
    const uint32_t j = lane % 8u;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t r = warp * 16u + i * 4u + lane / 8u;
      const uint64_t row = r0 + r;
      Share<T> x;
      x.template load<(int)kPiece>(reinterpret_cast<const T*>(tile) + r * 128u, j, 128u);
      const uint32_t byte = scale_byte(f32_bits<T>(x.block_magnitude()));
      if (row < a.rows) {
        x.store(a.codes + row * code_cols + c0, j, code_cols - (uint32_t)c0, inverse_scale(byte));
        const uint32_t end = bx == col_tiles - 1u ? scale_cols - bx : 1u;
        if (j < end) a.scales[row * scale_cols + bx + j] = j == 0u ? (uint8_t)byte : 0;
      }
    }
  }
  __syncthreads();
  const uint32_t cw = tid % kRowWords, part = tid / kRowWords;
  uint32_t held[kHeld];
#pragma unroll
  for (uint32_t r = 0; r < kHeld; ++r) held[r] = tile[(part * kHeld + r) * kRowWords + cw];
  uint32_t m = 0;
#pragma unroll
  for (uint32_t r = 0; r < kHeld; ++r) m = W::larger(m, held[r] & W::kAbs);
  if (W::largest(m) >= W::kInf) {
    m = 0;
#pragma unroll
    for (uint32_t r = 0; r < kHeld; ++r) {
      m = W::larger(m, W::finite(held[r]));
      held[r] = W::only_nan(held[r]);
    }
  }
  part_max[part][cw] = m;
  __syncthreads();
#pragma unroll
  for (uint32_t p = 0; p < kParts; ++p) m = W::larger(m, part_max[p][cw]);
  // Codes go through the tile's memory (every value is in registers by now), so
  // that a column leaves 128 bytes at a time; 16-byte pieces are swizzled.
  uint8_t* turned = reinterpret_cast<uint8_t*>(tile);
#pragma unroll
  for (uint32_t v = 0; v < W::kValues; ++v) {
    const uint32_t c = cw * W::kValues + v;
    const uint32_t byte = scale_byte(f32_bits<T>(W::value(m, v)));
    const float inv = inverse_scale(byte);
#pragma unroll
    for (uint32_t q = 0; q < kHeld; q += 16u) {
      uint32_t w[4];
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        float x[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) x[i] = W::f32(held[q + u * 4u + i], v) * inv;
        w[u] = codes2(x[0], x[1]) | codes2(x[2], x[3]) << 16;
      }
      *reinterpret_cast<uint4*>(turned + c * 128u + (((part * kHeld + q) / 16u ^ cw % 8u) * 16u)) =
          make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (part == 0 && c0 + c < a.cols) {
      const uint32_t last = by == row_tiles - 1u ? scale_rows : by + 1u;
      for (uint32_t b = by; b < last; ++b) a.scales_t[(c0 + c) * scale_rows + b] = b == by ? (uint8_t)byte : 0;
    }
  }
  __syncthreads();
  const uint32_t piece = tid % 8u;
  if (r0 + piece * 16u >= code_rows) return;
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const uint32_t c = i * 32u + tid / 8u;
    if (c0 + c < a.cols)
      *reinterpret_cast<uint4*>(a.codes_t + (c0 + c) * code_rows + r0 + piece * 16u) =
          *reinterpret_cast<const uint4*>(turned + c * 128u + ((piece ^ c / W::kValues % 8u) * 16u));
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
  const uint32_t ve = vector_elems(a.x, a.rows, a.cols, a.stride, type_bytes(a.dtype), 16u / type_bytes(a.dtype));
  return with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto width) {
      constexpr int VE = decltype(width)::value;
      if (a.codes_t)
        return a.codes ? launch_tiles<T, VE, true>(a, c.device, code_cols, scale_cols, code_rows, scale_rows, stream)
                       : launch_tiles<T, VE, false>(a, c.device, code_cols, scale_cols, code_rows, scale_rows, stream);
      const uint32_t blocks = (uint32_t)div_up(a.cols, 128), total = (uint32_t)a.rows * blocks;
      quantize_rows_kernel<T, VE><<<(uint32_t)div_up(total, 32), 256, 0, stream>>>(a, total, blocks, code_cols, scale_cols);
      return cudaGetLastError();
    };
    // 16 bytes at a time, 8, or a value
    if (ve * sizeof(T) == 16) return launch(std::integral_constant<int, 16 / sizeof(T)>());
    if (ve * sizeof(T) == 8) return launch(std::integral_constant<int, 8 / sizeof(T)>());
    return launch(std::integral_constant<int, 1>());
  });
}

}  // namespace tessa

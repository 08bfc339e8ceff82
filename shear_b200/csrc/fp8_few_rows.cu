// The FP8 product where one operand has a handful of rows (a query against a
// table): out = sum over blocks of 128 of sp[b] sq[b] (p . q)_b.
//
// Every code of the long operand is used for eight products at most, so this
// is a read: bound by the long operand's bytes.  The form for large products
// (fp8_matmul.cu) spends about 1.2 us a tile on its chain of barriers however
// short the other operand.  Here a warp takes 32 rows and eight lanes' worth of
// the short operand without any shared memory: codes go from global memory to
// registers, m16n8k32 sums a block's 128 products in f32, and the two scales
// multiply that sum as it is added up.  Each lane reads 16 bytes at a time: the
// order of K within a block is free as long as both operands keep to it.
// One row against 200000 x 128: 6.2 us (4.2 TB/s; the other form 17), x 768 35 us
// (4.4 TB/s; 32), 1M x 768 135 us (5.7 TB/s; 140), 5000 x 768 3.1 us (6.9).  What
// bounds it is the latency of the reads: 28 warps an SM with 4 KB each.
#include "train_common.cuh"

namespace tessa {
namespace train {
namespace few {

constexpr uint32_t kRows = 32;       // of the long operand a warp
constexpr uint32_t kPlainWarps = 2;  // a block, where warps do not share rows: small blocks even the SMs' load out

struct Params {
  const uint8_t *p, *p_scales;  // the long operand
  const uint8_t *q, *q_scales;  // the short one
  uint32_t rows_p, rows_q, k, kblocks, scale_cols;
  uint64_t out_p, out_q;        // elements from row to row of p, of q in out
  void* out;
};

// c += a . b over 32 of K: 16 rows of a, 8 of b
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A scale's byte; 255, which stands for NaN, moved out of reach of any sum of two others.
__device__ __forceinline__ uint32_t scale_code(uint32_t byte) { return byte == 255u ? 4096u : byte; }

// s * 2^(a - 127) * 2^(b - 127)
__device__ __forceinline__ float scaled(float s, uint32_t a, uint32_t b) {
  const uint32_t t = a + b - 127u;  // the exponent of their product where it is a normal number
  if (t - 1u < 254u) return s * __uint_as_float(t << 23);
  return a + b >= 4096u ? NAN : scalbnf(s, (int)t - 127);
}

// SPLIT: the eight warps of a block share 32 rows and take blocks of K in turn;
// their sums are added in order.
template <class O, bool SPLIT, bool AHEAD>
__global__ void __launch_bounds__(256, AHEAD ? 1 : SPLIT ? 3 : 4) few_rows_kernel(const Params a) {
  const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u, g = lane / 4u, t = lane % 4u;
  const uint32_t row0 = (SPLIT ? blockIdx.x : blockIdx.x * kPlainWarps + warp) * kRows;
  if (!SPLIT && row0 >= a.rows_p) return;
  // rows g, g + 8, g + 16, g + 24 of the long operand, row g of the short one
  const uint8_t *p[4], *ps[4];
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const uint64_t row = min(row0 + i * 8u + g, a.rows_p - 1u);
    p[i] = a.p + row * a.k + t * 16u;
    ps[i] = a.p_scales + row * a.scale_cols;
  }
  const uint64_t q_row = min(g, a.rows_q - 1u);
  const uint8_t* q = a.q + q_row * a.k + t * 16u;
  const uint8_t* qs[2];  // of the two columns that the accumulator gives this lane
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) qs[i] = a.q_scales + (uint64_t)min(2u * t + i, a.rows_q - 1u) * a.scale_cols;
  float acc[4][2] = {};  // row g + 8i, column 2t + j
  struct Block {
    uint4 x[4][2], y[2];
    uint32_t sp[4], sq[2];
  };
  auto load = [&](Block& d, uint32_t b) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t at = b * 128u + h * 64u;
      const bool in = at + t * 16u < a.k;
      const uint4 none = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) d.x[i][h] = in ? __ldg(reinterpret_cast<const uint4*>(p[i] + at)) : none;
      d.y[h] = in ? __ldg(reinterpret_cast<const uint4*>(q + at)) : none;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) d.sp[i] = scale_code(__ldg(ps[i] + b));
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) d.sq[i] = scale_code(__ldg(qs[i] + b));
  };
  auto sum = [&](const Block& d) {
    float c[2][4] = {};
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        mma(c[i], d.x[2 * i][h].x, d.x[2 * i + 1][h].x, d.x[2 * i][h].y, d.x[2 * i + 1][h].y, d.y[h].x, d.y[h].y);
        mma(c[i], d.x[2 * i][h].z, d.x[2 * i + 1][h].z, d.x[2 * i][h].w, d.x[2 * i + 1][h].w, d.y[h].z, d.y[h].w);
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
      for (uint32_t j = 0; j < 2; ++j) acc[i][j] += scaled(c[i / 2][i % 2 * 2 + j], d.sp[i], d.sq[j]);
  };
  constexpr uint32_t kStep = SPLIT ? 8u : 1u;
  if constexpr (AHEAD) {  // the next block is under way while one is summed
    Block one, other;
    uint32_t b = SPLIT ? warp : 0u;
    if (b < a.kblocks) load(one, b);
#pragma unroll 1
    for (; b < a.kblocks; b += 2u * kStep) {
      if (b + kStep < a.kblocks) load(other, b + kStep);
      sum(one);
      if (b + kStep >= a.kblocks) break;
      if (b + 2u * kStep < a.kblocks) load(one, b + 2u * kStep);
      sum(other);
    }
  } else {  // the other warps' are: registers for more of them pay better
#pragma unroll 1
    for (uint32_t b = SPLIT ? warp : 0u; b < a.kblocks; b += kStep) {
      Block one;
      load(one, b);
      sum(one);
    }
  }
  if constexpr (SPLIT) {
    __shared__ float part[8][kRows][8];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
      for (uint32_t j = 0; j < 2; ++j) part[warp][i * 8u + g][2u * t + j] = acc[i][j];
    __syncthreads();
    const uint32_t row = threadIdx.x % kRows, r = threadIdx.x / kRows;
    if (r < a.rows_q && row0 + row < a.rows_p) {
      float s = part[0][row][r];
#pragma unroll
      for (int w = 1; w < 8; ++w) s += part[w][row][r];
      static_cast<O*>(a.out)[(row0 + row) * a.out_p + r * a.out_q] = from_f32<O>(s);
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t row = row0 + i * 8u + g;
#pragma unroll
      for (uint32_t j = 0; j < 2; ++j) {
        const uint32_t r = 2u * t + j;
        if (row < a.rows_p && r < a.rows_q) static_cast<O*>(a.out)[row * a.out_p + r * a.out_q] = from_f32<O>(acc[i][j]);
      }
    }
  }
}

}  // namespace few
}  // namespace train

cudaError_t launch_fp8_few_rows(const tessa_fp8_matmul_args& a, const AsyncCtx& c, cudaStream_t stream) {
  using namespace train;
  const bool swap = a.m <= a.n;  // a is the short operand
  few::Params p = {};
  p.p = swap ? a.b_codes : a.a_codes;
  p.p_scales = swap ? a.b_scales : a.a_scales;
  p.q = swap ? a.a_codes : a.b_codes;
  p.q_scales = swap ? a.a_scales : a.b_scales;
  p.rows_p = (uint32_t)(swap ? a.n : a.m);
  p.rows_q = (uint32_t)(swap ? a.m : a.n);
  p.k = (uint32_t)a.k;
  p.kblocks = (uint32_t)div_up(a.k, 128);
  p.scale_cols = (uint32_t)div_up(a.k, 512) * 4u;
  p.out_p = swap ? 1 : a.out_stride;
  p.out_q = swap ? a.out_stride : 1;
  p.out = a.out;
  // Where the rows do not fill the SMs' warps twice, K is shared out as well (40000
  // x 768: 6.9 us, 9.6 otherwise; 100000 x 768: 14.3 and 14.0); where blocks have
  // an SM each, a warp looks ahead (64 x 16384: 14 us, 21 otherwise; 20000 x 4096:
  // 23 and 16).
  const bool split = p.kblocks >= 4 && p.rows_p < 512ull * c.sm_count;
  const uint32_t grid = (uint32_t)div_up(p.rows_p, (split ? 1 : few::kPlainWarps) * few::kRows);
  const bool ahead = split && grid <= (uint32_t)c.sm_count;
  return with_type(a.out_dtype, [&](auto o) {
    if (ahead) few::few_rows_kernel<decltype(o), true, true><<<grid, 256, 0, stream>>>(p);
    else if (split) few::few_rows_kernel<decltype(o), true, false><<<grid, 256, 0, stream>>>(p);
    else few::few_rows_kernel<decltype(o), false, false><<<grid, 32 * few::kPlainWarps, 0, stream>>>(p);
    return cudaGetLastError();
  });
}

}  // namespace tessa

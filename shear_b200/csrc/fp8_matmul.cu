// out[m][n] = sum over blocks of 128 of sa[m][b] sb[n][b] (a[m] . b[n])_b on
// E4M3 codes with power-of-two block scales.
//
// tcgen05.mma kind::mxf8f6f4 applies a scale byte per row and 32 values of K
// by itself, so a block's byte is named by its four K steps of 32 (the byte of
// a 32-bit word of scales that the instruction descriptor selects), and the
// sum over K never leaves the f32 accumulator in tensor memory: no pass over
// the accumulator per block, as a free f32 scale would need.
//
// One persistent CTA per SM; the roles run concurrently:
//   warp 0    TMA: stages of 128 bytes of K: 128 rows of b, BN rows of a
//   warp 1    tensor memory, scales' copies into it (tcgen05.cp), MMAs
//   warp 2    scales: 32-bit words (four blocks of K) from global to shared
//             memory, in the order tcgen05.cp wants
//   warps 4-7 epilogue: accumulators to global memory
// b's rows are the accumulator's 128 lanes and a's rows its columns, so a warp
// holds 32 consecutive n of one m and stores them straight to out, and a batch
// of few rows makes a narrow MMA (BN from 16) instead of a mostly empty one.
// Two accumulators: one is emptied while the next is summed.
//
// K may be split over units (few tiles, long K): each unit writes f32 parts to
// the workspace and a second kernel adds them in order of K, so the result
// does not depend on timing.
#include "train_common.cuh"

namespace tessa {
namespace train {
namespace mm {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kBP = 128;             // rows of b a tile (accumulator lanes)
constexpr uint32_t kMaxBN = 240;          // rows of a a tile: two accumulators and the scales fit 512 columns
constexpr uint32_t kBK = 128;             // bytes of K a stage
constexpr uint32_t kScaleBufs = 4;        // shared memory buffers of scale words
constexpr uint32_t kScaleBytes = 512 + 1024;  // 128 words of b, up to 256 of a
constexpr uint32_t kScaleCol = 480;       // tensor memory columns of the scales: two sets of 16
constexpr uint32_t kMaxStages = 10;
constexpr uint32_t kSmemLimit = 227u * 1024u;

struct Params {
  const uint8_t* p_scales;  // b's
  const uint8_t* q_scales;  // a's
  uint64_t scale_cols;
  uint64_t m, n;
  uint32_t kblocks;         // blocks of 128
  uint32_t ksteps;          // steps of 32 that hold data
  uint32_t bn;
  uint32_t tiles_p, tiles_q;
  uint32_t splits, split_groups;  // groups of four blocks a split
  uint32_t stages;
  void* out;
  uint64_t out_stride;
  float* parts;             // splits x m x n, splits > 1
  uint32_t* err;
  uint64_t timeout_ns;
};

// kind::mxf8f6f4, E4M3 x E4M3, both K-major, E8M0 scales, f32 accumulators;
// scale_id selects the byte of the scale words.
__device__ __forceinline__ uint32_t idesc_mx(uint32_t bn, uint32_t scale_id) {
  return (scale_id << 4) | ((bn >> 3) << 17) | (1u << 23) | ((kBP >> 4) << 24) | (scale_id << 29);
}

__device__ __forceinline__ void mma_mx(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                       uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate));
}

// 32 rows x 16 bytes of shared memory (unswizzled, rows 16 bytes apart) to
// four tensor memory columns, repeated in the four lane quadrants.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t smem_addr) {
  const uint64_t desc = (uint64_t)((smem_addr >> 4) & 0x3FFFu) | (uint64_t)(128u >> 4) << 32 | (uint64_t)1u << 46;
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

struct Unit {
  uint32_t p, q;       // tile
  uint32_t kb0, kb1;   // blocks of K
  uint32_t split;
};

// Tiles in blocks of up to 16 along a: the tiles in flight at a time then
// share few rows of b and of a in L2.
__device__ __forceinline__ Unit unit_of(const Params& p, uint32_t u) {
  Unit r;
  r.split = u % p.splits;
  const uint32_t t = u / p.splits;
  constexpr uint32_t kGroup = 16;
  const uint32_t block = t / (kGroup * p.tiles_p), in = t % (kGroup * p.tiles_p);
  const uint32_t wide = min(kGroup, p.tiles_q - block * kGroup);
  r.q = block * kGroup + in % wide;
  r.p = in / wide;
  r.kb0 = r.split * p.split_groups * 4u;
  r.kb1 = min(p.kblocks, r.kb0 + p.split_groups * 4u);
  return r;
}

template <class O, bool PARTS>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_matmul_kernel(const __grid_constant__ CUtensorMap pmap, const __grid_constant__ CUtensorMap qmap,
                      const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~(uintptr_t)1023u);
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], sf_full[kScaleBufs], sf_empty[kScaleBufs],
      acc_full[2], acc_empty[2], group_done[2], drained;
  __shared__ uint32_t tmem_slot, abort_word;
  volatile uint32_t* abort_flag = &abort_word;
  const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
  const uint32_t stage_bytes = (kBP + p.bn) * kBK;
  uint8_t* scales = smem + p.stages * stage_bytes;
  const uint32_t units = p.tiles_p * p.tiles_q * p.splits;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < kMaxStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (uint32_t i = 0; i < kScaleBufs; ++i) {
      mbar_init(&sf_full[i], 1);
      mbar_init(&sf_empty[i], 1);
    }
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4);
      mbar_init(&group_done[i], 1);
    }
    mbar_init(&drained, 1);
    abort_word = 0u;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&pmap);
    tma_prefetch_desc(&qmap);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait(bar, parity, abort_flag, p.err, p.timeout_ns);
  };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;  // stages filled so far
      bool ok = true;
      for (uint32_t u = blockIdx.x; u < units && ok; u += gridDim.x) {
        const Unit t = unit_of(p, u);
        for (uint32_t kb = t.kb0; kb < t.kb1; ++kb, ++it) {
          const uint32_t s = it % p.stages;
          if (!wait(&empty[s], ((it / p.stages) & 1u) ^ 1u)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], stage_bytes);
          uint8_t* dst = smem + s * stage_bytes;
          tma_load_2d(&pmap, dst, &full[s], (int32_t)(kb * kBK), (int32_t)(t.p * kBP));
          tma_load_2d(&qmap, dst + kBP * kBK, &full[s], (int32_t)(kb * kBK), (int32_t)(t.q * p.bn));
        }
      }
      // The block may not end before its copies have landed.
      uint32_t dummy = 0u;
      for (uint32_t i = it > p.stages ? it - p.stages : 0u; i < it; ++i)
        mbar_wait(&full[i % p.stages], (i / p.stages) & 1u, &dummy, p.err, p.timeout_ns);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t base = smem_u32(smem), scale_base = smem_u32(scales);
      uint32_t it = 0, group = 0, acc = 0;
      bool ok = true;
      for (uint32_t u = blockIdx.x; u < units && ok; u += gridDim.x, ++acc) {
        const Unit t = unit_of(p, u);
        const uint32_t buf = acc & 1u;
        if (!wait(&acc_empty[buf], ((acc >> 1) & 1u) ^ 1u)) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * kMaxBN;
        for (uint32_t kb = t.kb0; kb < t.kb1 && ok; kb += 4u, ++group) {
          // The group's scales: into the tensor memory set that the group
          // before the last has finished reading.
          const uint32_t sb = group % kScaleBufs, set = group & 1u;
          const uint32_t sfp = tmem + kScaleCol + set * 16u, sfq = sfp + 4u;
          if (!wait(&sf_full[sb], (group / kScaleBufs) & 1u) ||
              (group >= 2u && !wait(&group_done[set], ((group >> 1) - 1u) & 1u))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = scale_base + sb * kScaleBytes;
          copy_scales(sfp, sa);
          copy_scales(sfq, sa + 512u);
          if (p.bn > 128u) copy_scales(sfq + 4u, sa + 1024u);
          mma_commit(&sf_empty[sb]);
          const uint32_t end = min(kb + 4u, t.kb1);
          for (uint32_t b = kb; b < end; ++b, ++it) {
            const uint32_t s = it % p.stages;
            if (!wait(&full[s], (it / p.stages) & 1u)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t pa = base + s * stage_bytes, qa = pa + kBP * kBK;
            const uint32_t idesc = idesc_mx(p.bn, b - kb);
            const uint32_t steps = min(4u, p.ksteps - b * 4u);
            for (uint32_t k = 0; k < steps; ++k)
              mma_mx(d, smem_desc_sw128(pa + k * 32u), smem_desc_sw128(qa + k * 32u), idesc, sfp, sfq,
                     b > t.kb0 || k > 0u ? 1u : 0u);
            mma_commit(&empty[s]);
          }
          if (ok) mma_commit(&group_done[set]);
        }
        if (ok) mma_commit(&acc_full[buf]);
      }
      // Everything issued has completed before tensor memory is released.
      mma_commit(&drained);
      uint32_t dummy = 0u;
      mbar_wait(&drained, 0u, &dummy, p.err, p.timeout_ns);
    }
  } else if (warp == 2) {
    uint32_t group = 0;
    bool ok = true;
    for (uint32_t u = blockIdx.x; u < units && ok; u += gridDim.x) {
      const Unit t = unit_of(p, u);
      for (uint32_t kb = t.kb0; kb < t.kb1; kb += 4u, ++group) {
        uint32_t w[12];
#pragma unroll
        for (uint32_t i = 0; i < 12; ++i) {
          const bool of_p = i < 4;
          const uint32_t r = (of_p ? i : i - 4u) * 32u + lane;
          const uint64_t row = of_p ? (uint64_t)t.p * kBP + r : (uint64_t)t.q * p.bn + r;
          const bool in = of_p ? row < p.n : row < p.m && r < p.bn;
          w[i] = in ? *reinterpret_cast<const uint32_t*>((of_p ? p.p_scales : p.q_scales) + row * p.scale_cols + kb) : 0u;
        }
        const uint32_t sb = group % kScaleBufs;
        const bool freed = lane != 0 || wait(&sf_empty[sb], ((group / kScaleBufs) & 1u) ^ 1u);
        if (!__shfl_sync(0xffffffffu, freed ? 1u : 0u, 0)) {
          ok = false;
          break;
        }
        uint4* dst = reinterpret_cast<uint4*>(scales + sb * kScaleBytes) + lane;
        dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
        dst[32] = make_uint4(w[4], w[5], w[6], w[7]);
        dst[64] = make_uint4(w[8], w[9], w[10], w[11]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sf_full[sb]);
      }
    }
  } else if (warp >= 4) {
    const uint32_t quad = warp - 4u;
    uint32_t acc = 0;
    for (uint32_t u = blockIdx.x; u < units; u += gridDim.x, ++acc) {
      const Unit t = unit_of(p, u);
      const uint32_t buf = acc & 1u;
      const bool full_ok = lane != 0 || wait(&acc_full[buf], (acc >> 1) & 1u);
      if (!__shfl_sync(0xffffffffu, full_ok ? 1u : 0u, 0)) break;
      tc_fence_after();
      const uint64_t n = (uint64_t)t.p * kBP + quad * 32u + lane;
      const uint64_t m0 = (uint64_t)t.q * p.bn;
      const uint32_t rows = (uint32_t)min((uint64_t)p.bn, p.m - m0);
      O* out;
      uint64_t stride;
      if constexpr (PARTS) {
        out = reinterpret_cast<O*>(p.parts) + ((uint64_t)t.split * p.m + m0) * p.n + n;
        stride = p.n;
      } else {
        out = static_cast<O*>(p.out) + m0 * p.out_stride + n;
        stride = p.out_stride;
      }
      const uint32_t ta = tmem + buf * kMaxBN + (quad << 21);  // lane quad * 32
#pragma unroll 2
      for (uint32_t c = 0; c < p.bn; c += 16u) {
        uint32_t v[16];
        tmem_ld_x16(ta + c, v);
        tmem_ld_wait();
        if (n < p.n) {
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i)
            if (c + i < rows) out[(c + i) * stride] = from_f32<O>(__uint_as_float(v[i]));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[buf]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// out = the parts' sum in order of K.
template <class O>
__global__ void __launch_bounds__(256) add_parts_kernel(const float* parts, uint32_t splits, uint64_t m, uint64_t n,
                                                        O* out, uint64_t out_stride) {
  const uint64_t total = m * n, step = (uint64_t)gridDim.x * 256u;
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < total; i += step) {
    float s = parts[i];
#pragma unroll 4
    for (uint32_t k = 1; k < splits; ++k) s += parts[(uint64_t)k * total + i];
    out[i / n * out_stride + i % n] = from_f32<O>(s);
  }
}

struct Plan {
  uint32_t bn, tiles_p, tiles_q, splits, split_groups;
};

// Rows of a a tile and splits of K by the estimated cycles of the busiest SM:
// a block of K takes 2 BN cycles of the tensor core (not less than the 64 or
// so that its stage's bytes take to arrive), a tile about 1000 + 4 BN beside
// its MMAs, a split its parts' traffic and a second launch.
inline Plan plan(uint64_t m, uint64_t n, uint64_t k, int sm_count) {
  Plan best = {};
  double best_cost = 0.0;
  const uint32_t groups = (uint32_t)div_up(k, 512), tp = (uint32_t)div_up(n, kBP);
  const uint64_t least = div_up(m, kMaxBN);
  for (uint64_t tq = least; tq <= least + 8 && tq <= div_up(m, 16); ++tq) {
    const uint32_t bn = (uint32_t)(div_up(div_up(m, tq), 16) * 16);
    if (div_up(m, bn) != tq) continue;
    // splitting pays only while whole tiles leave SMs without work
    const uint32_t most = (uint64_t)tp * tq >= (uint64_t)sm_count ? 1u : 32u;
    for (uint32_t want = 1; want <= groups && want <= most; ++want) {
      const uint32_t sg = (uint32_t)div_up(groups, want), splits = (uint32_t)div_up(groups, sg);
      if (splits != want) continue;
      const double units = (double)tp * (double)tq * splits;
      if (splits > 1 && units > 2.0 * sm_count) break;
      const double blocks = sg * 4.0 < (double)div_up(k, 128) ? sg * 4.0 : (double)div_up(k, 128);
      const double waves = (double)(uint64_t)((units + sm_count - 1) / sm_count);
      double cost = waves * (blocks * (2.0 * bn > 64.0 ? 2.0 * bn : 64.0) + 1000.0 + 4.0 * bn);
      if (splits > 1) cost += 5000.0 + 8.0 * splits * (double)m * (double)n / 3500.0;
      if (best.bn == 0 || cost < best_cost) {
        best = {bn, tp, (uint32_t)tq, splits, sg};
        best_cost = cost;
      }
    }
  }
  return best;
}

template <class O, bool PARTS>
cudaError_t launch(const CUtensorMap& pm, const CUtensorMap& qm, const Params& p, uint32_t smem, uint32_t grid,
                   cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute(fp8_matmul_kernel<O, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)smem);
  if (e != cudaSuccess) return e;
  fp8_matmul_kernel<O, PARTS><<<grid, kThreads, smem, stream>>>(pm, qm, p);
  return cudaGetLastError();
}

}  // namespace mm
}  // namespace train

uint64_t fp8_matmul_workspace(uint64_t m, uint64_t n, uint64_t k, int sm_count) {
  if (m == 0 || n == 0 || k == 0) return 0;
  const train::mm::Plan pl = train::mm::plan(m, n, k, sm_count);
  return pl.splits > 1 ? (uint64_t)pl.splits * m * n * 4 : 0;
}

cudaError_t launch_matmul_fp8(const tessa_fp8_matmul_args& a, void* workspace, const AsyncCtx& c,
                              cudaStream_t stream) {
  using namespace train;
  if (a.k == 0)
    return cudaMemset2DAsync(a.out, (a.m > 1 ? a.out_stride : a.n) * type_bytes(a.out_dtype), 0,
                             a.n * type_bytes(a.out_dtype), a.m, stream);
  const mm::Plan pl = mm::plan(a.m, a.n, a.k, c.sm_count);
  CUtensorMap pm, qm;
  if (make_code_tmap(&pm, a.b_codes, a.n, (uint32_t)a.k, mm::kBP) != 0 ||
      make_code_tmap(&qm, a.a_codes, a.m, (uint32_t)a.k, pl.bn) != 0)
    return cudaErrorInvalidValue;
  mm::Params p = {};
  p.p_scales = a.b_scales;
  p.q_scales = a.a_scales;
  p.scale_cols = div_up(a.k, 512) * 4;
  p.m = a.m;
  p.n = a.n;
  p.kblocks = (uint32_t)div_up(a.k, 128);
  p.ksteps = (uint32_t)div_up(a.k, 32);
  p.bn = pl.bn;
  p.tiles_p = pl.tiles_p;
  p.tiles_q = pl.tiles_q;
  p.splits = pl.splits;
  p.split_groups = pl.split_groups;
  const uint32_t stage = (mm::kBP + pl.bn) * mm::kBK, fixed = 1024u + mm::kScaleBufs * mm::kScaleBytes + 1024u;
  p.stages = (mm::kSmemLimit - fixed) / stage;
  if (p.stages > mm::kMaxStages) p.stages = mm::kMaxStages;
  p.out = a.out;
  p.out_stride = a.out_stride;
  p.parts = static_cast<float*>(workspace);
  p.err = c.err;
  p.timeout_ns = c.timeout_ns;
  const uint32_t smem = p.stages * stage + mm::kScaleBufs * mm::kScaleBytes + 1024u;
  const uint64_t units = (uint64_t)pl.tiles_p * pl.tiles_q * pl.splits;
  const uint32_t grid = (uint32_t)(units < (uint64_t)c.sm_count ? units : (uint64_t)c.sm_count);
  if (pl.splits > 1) {
    cudaError_t e = mm::launch<float, true>(pm, qm, p, smem, grid, stream);
    if (e != cudaSuccess) return e;
    const uint64_t want = div_up(a.m * a.n, 256), most = (uint64_t)c.sm_count * 16;
    return with_type(a.out_dtype, [&](auto o) {
      using O = decltype(o);
      mm::add_parts_kernel<O><<<(uint32_t)(want < most ? want : most), 256, 0, stream>>>(
          p.parts, pl.splits, a.m, a.n, static_cast<O*>(a.out), a.out_stride);
      return cudaGetLastError();
    });
  }
  return with_type(a.out_dtype,
                   [&](auto o) { return mm::launch<decltype(o), false>(pm, qm, p, smem, grid, stream); });
}

}  // namespace tessa

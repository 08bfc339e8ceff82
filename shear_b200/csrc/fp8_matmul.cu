// out[m][n] = sum over blocks of 128 of sa[m][b] sb[n][b] (a[m] . b[n])_b on
// E4M3 codes with power-of-two block scales.
//
// tcgen05.mma kind::mxf8f6f4 applies a scale byte per row and 32 values of K
// by itself, so a block's byte is named by its four K steps of 32 (the byte of
// a 32-bit word of scales that the instruction descriptor selects), and the
// sum over K never leaves the f32 accumulator in tensor memory: no pass over
// the accumulator per block, as a free f32 scale would need.
//
// Persistent pairs of CTAs (two SMs) share a tile of 256 rows of b and BN rows
// of a: each CTA holds 128 rows of b and half of a's in shared memory, and one
// MMA (cta_group::2) reads both halves, so a stage brings 31 KB into an SM
// where a CTA alone would need 47 KB for the same work.  Roles, concurrently:
//   warp 0      TMA: stages of 128 bytes of K
//   warp 1      tensor memory; in the first CTA the pair's MMAs
//   warps 4-7   scales: 32-bit words (four blocks of K) from global memory to
//               the four lane quadrants of tensor memory
//   warps 8-15  epilogue: accumulators to global memory
// b's rows are the accumulator's lanes and a's rows its columns, so a warp
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

constexpr uint32_t kThreads = 512;
constexpr uint32_t kBP = 128;             // rows of b a CTA (accumulator lanes)
constexpr uint32_t kMaxBN = 224;          // rows of a a tile: two accumulators leave 64 of 512 columns to the scales
constexpr uint32_t kBK = 128;             // bytes of K a stage
constexpr uint32_t kScaleCol = 448;       // tensor memory columns of the scales
constexpr uint32_t kSets = 4;             // sets of 16: the scale warps run up to three groups ahead
constexpr uint32_t kMaxStages = 10;
constexpr uint32_t kSmemLimit = 227u * 1024u;
constexpr uint32_t kScaleWarp = 4, kEpiWarp = 8;

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
  return (scale_id << 4) | ((bn >> 3) << 17) | (1u << 23) | ((2u * kBP >> 4) << 24) | (scale_id << 29);
}

__device__ __forceinline__ void mma_mx(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                       uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate));
}

__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_st_x4(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0u;
}

// Arrives on the barrier at this offset in both CTAs once the MMAs issued so far have completed.
__device__ __forceinline__ void commit_both(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}

// Arrives on a barrier of either CTA.  What the pair's barriers guard is
// tensor memory, ordered by tcgen05.fence, and shared memory that TMA writes:
// no ordinary memory, so a release at cluster scope, which waits for the
// thread's loads and stores in flight (2000 cycles here), is not needed.
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ void expect_at(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// TMA tile load into this CTA whose bytes complete on a barrier of the pair (no multicast).
__device__ __forceinline__ void load_at(const CUtensorMap* map, uint32_t dst, uint32_t bar, int32_t x, int32_t y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ bool try_at(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0u;
}
// mbar_wait by shared-memory address; the first look costs a few instructions.
__device__ __forceinline__ bool wait_at(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* err,
                                        uint64_t timeout_ns) {
  return try_at(bar, parity) || mbar_wait(reinterpret_cast<uint64_t*>(__cvta_shared_to_generic(bar)), parity,
                                          abort_flag, err, timeout_ns);
}

// Barrier of the four scale warps; whether any thread said so.
__device__ __forceinline__ bool meet_any(bool said) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(said ? 1u : 0u)
      : "memory");
  return r != 0u;
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
// The blocks of K alone: all that the MMA warp needs, without the divisions
// that would leave the tensor core idle between tiles.
__device__ __forceinline__ void span_of(const Params& p, uint32_t u, uint32_t& kb0, uint32_t& kb1) {
  kb0 = 0;
  kb1 = p.kblocks;
  if (p.splits > 1u) {
    kb0 = u % p.splits * p.split_groups * 4u;
    kb1 = min(p.kblocks, kb0 + p.split_groups * 4u);
  }
}

// Sixteen accumulator columns of the lane's row: out[i * stride], i < rows.
template <class O>
__device__ __forceinline__ void store16(O* out, uint64_t stride, const uint32_t (&v)[16], uint32_t rows) {
  if (rows >= 16u) {
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      *out = from_f32<O>(__uint_as_float(v[i]));
      out += stride;
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      if (i < rows) *out = from_f32<O>(__uint_as_float(v[i]));
      out += stride;
    }
  }
}

template <class O, bool PARTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    fp8_matmul_kernel(const __grid_constant__ CUtensorMap pmap, const __grid_constant__ CUtensorMap qmap,
                      const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~(uintptr_t)1023u);
  // In the first CTA: full, scale_full and acc_empty count both CTAs' work.
  // The other barriers are signalled in both CTAs.
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], scale_full[kSets], group_done[kSets],
      acc_full[2], acc_empty[2], drained;
  __shared__ uint32_t scale_words[2][kBP + 256];  // a group's words: b's rows, a's rows
  __shared__ uint32_t tmem_slot, abort_word;
  volatile uint32_t* abort_flag = &abort_word;
  const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
  const uint32_t rank = cluster_ctarank();
  const uint32_t half_bn = p.bn / 2u;
  const uint32_t stage_bytes = (kBP + half_bn) * kBK;  // of one CTA
  const uint32_t units = p.tiles_p * p.tiles_q * p.splits;
  const uint32_t unit0 = blockIdx.x / 2u, ustep = gridDim.x / 2u;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < kMaxStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (uint32_t i = 0; i < kSets; ++i) {
      mbar_init(&scale_full[i], 8);
      mbar_init(&group_done[i], 1);
    }
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 16);
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
    tmem_alloc_pair(&tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the peer's barriers are initialised before any arrival on them
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait(bar, parity, abort_flag, p.err, p.timeout_ns);
  };

  if (warp == 0) {
    const bool one = elect_one();
    const uint32_t ring = smem_u32(smem), empty_base = smem_u32(empty), full_base = smem_u32(full);
    const uint32_t full_first = mapa_shared(full, 0);  // both CTAs' bytes complete on the first CTA's barrier
    uint32_t s = 0, phase = 0, filled = 0;
    bool ok = true;
    for (uint32_t u = unit0; u < units && ok; u += ustep) {
      const Unit t = unit_of(p, u);
      const int32_t py = (int32_t)((t.p * 2u + rank) * kBP), qy = (int32_t)(t.q * p.bn + rank * half_bn);
      for (uint32_t kb = t.kb0; kb < t.kb1; ++kb) {
        ok &= wait_at(empty_base + s * 8u, phase ^ 1u, abort_flag, p.err, p.timeout_ns);
        if (one && ok) {
          if (rank == 0) expect_at(full_base + s * 8u, 2u * stage_bytes);
          const uint32_t dst = ring + s * stage_bytes, bar = full_first + s * 8u;
          load_at(&pmap, dst, bar, (int32_t)(kb * kBK), py);
          load_at(&qmap, dst + kBP * kBK, bar, (int32_t)(kb * kBK), qy);
        }
        __syncwarp();
        filled += ok ? 1u : 0u;
        if (++s == p.stages) {
          s = 0;
          phase ^= 1u;
        }
      }
      ok = __all_sync(0xffffffffu, ok);
    }
    // The block may not end before its copies have landed.  The first CTA sees
    // both CTAs' bytes; after a wait gave up somewhere the other, whose copies
    // may lack their counterpart, leaves them ample time instead.
    if (lane == 0 && rank == 0) {
      uint32_t dummy = 0u;
      for (uint32_t i = filled > p.stages ? filled - p.stages : 0u; i < filled; ++i)
        mbar_wait(&full[i % p.stages], (i / p.stages) & 1u, &dummy, p.err, p.timeout_ns);
    } else if (lane == 0 && !ok) {
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 1000000ull) __nanosleep(1000);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 1) {
      // The pair's MMAs read this CTA's memory until they have all completed.
      uint32_t dummy = 0u;
      if (lane == 0) mbar_wait(&drained, 0u, &dummy, p.err, p.timeout_ns);
    } else {
      // The warp stays together, every operand of an MMA is the same in all
      // lanes and no branch depends on a wait's answer, so that the compiler
      // keeps the operands in uniform registers: an issue from one diverged
      // lane costs over 100 cycles, as much as an MMA.  After a wait that gave
      // up the tile's remaining MMAs therefore still run, on whatever the
      // stages hold, and the loop ends with the tile.
      const bool one = elect_one();
      const uint64_t base = smem_desc_sw128(smem_u32(smem));
      const uint32_t full_base = smem_u32(full), empty_base = smem_u32(empty);
      const uint32_t desc_step = stage_bytes >> 4;
      const uint32_t whole = p.ksteps / 4u;  // blocks before the one that K may end inside
      uint32_t s = 0, phase = 0, group = 0, acc = 0;
      bool ok = true;
      for (uint32_t u = unit0; u < units && ok; u += ustep, ++acc) {
        uint32_t kb0, kb1;
        span_of(p, u, kb0, kb1);
        const uint32_t buf = acc & 1u;
        ok &= wait_at(smem_u32(&acc_empty[buf]), ((acc >> 1) & 1u) ^ 1u, abort_flag, p.err, p.timeout_ns);
        const uint32_t d = tmem + buf * kMaxBN;
        uint32_t accumulate = 0;
        for (uint32_t kb = kb0; kb < kb1; kb += 4u, ++group) {
          const uint32_t set = group % kSets;
          const uint32_t sfp = tmem + kScaleCol + set * 16u, sfq = sfp + 4u;
          ok &= wait_at(smem_u32(&scale_full[set]), (group / kSets) & 1u, abort_flag, p.err, p.timeout_ns);
          const uint32_t end = min(kb + 4u, kb1), full_end = min(end, whole);
          uint32_t idesc = idesc_mx(p.bn, 0), b = kb;
          for (; b < full_end; ++b, idesc += idesc_mx(0, 1) - idesc_mx(0, 0)) {
            ok &= wait_at(full_base + s * 8u, phase, abort_flag, p.err, p.timeout_ns);
            tc_fence_after();
            const uint64_t pd = base + s * desc_step, qd = pd + (kBP * kBK >> 4);
            if (one) {
              mma_mx(d, pd, qd, idesc, sfp, sfq, accumulate);
              mma_mx(d, pd + 2u, qd + 2u, idesc, sfp, sfq, 1u);
              mma_mx(d, pd + 4u, qd + 4u, idesc, sfp, sfq, 1u);
              mma_mx(d, pd + 6u, qd + 6u, idesc, sfp, sfq, 1u);
              commit_both(empty_base + s * 8u);
            }
            __syncwarp();
            accumulate = 1u;
            if (++s == p.stages) {
              s = 0;
              phase ^= 1u;
            }
          }
          if (b < end) {
            ok &= wait_at(full_base + s * 8u, phase, abort_flag, p.err, p.timeout_ns);
            tc_fence_after();
            const uint64_t pd = base + s * desc_step, qd = pd + (kBP * kBK >> 4);
            const uint32_t steps = p.ksteps - b * 4u;  // 1 to 3
            if (one) {
              mma_mx(d, pd, qd, idesc, sfp, sfq, accumulate);
              if (steps > 1u) mma_mx(d, pd + 2u, qd + 2u, idesc, sfp, sfq, 1u);
              if (steps > 2u) mma_mx(d, pd + 4u, qd + 4u, idesc, sfp, sfq, 1u);
              commit_both(empty_base + s * 8u);
            }
            __syncwarp();
            if (++s == p.stages) {
              s = 0;
              phase ^= 1u;
            }
          }
          if (one) commit_both(smem_u32(&group_done[set]));
          __syncwarp();
        }
        if (one) commit_both(smem_u32(&acc_full[buf]));
        ok = __all_sync(0xffffffffu, ok);
      }
      // Everything issued has completed before tensor memory is released.
      if (one) commit_both(smem_u32(&drained));
      __syncwarp();
      uint32_t dummy = 0u;
      if (lane == 0) mbar_wait(&drained, 0u, &dummy, p.err, p.timeout_ns);
    }
  } else if (warp >= kScaleWarp && warp < kScaleWarp + 4u) {
    // Row r of a tile has its word in lane r % 32, column r / 32, the same in
    // every quadrant: this CTA's 128 rows of b, all BN rows of a.  Thread i
    // fetches the words of row i of b and of rows i and i + 128 of a, a group
    // ahead; shared memory hands them to all four warps.
    const uint32_t quad = warp - kScaleWarp, i = threadIdx.x - kScaleWarp * 32u;
    const uint32_t words_q = (p.bn + 31u) / 32u;
    uint32_t u = unit0, group = 0, next[3] = {0u, 0u, 0u};
    Unit t = {};
    uint32_t kb = 0;
    bool gave_up = false;
    auto fetch = [&]() {  // the words of (t, kb)
      const uint64_t pr = (uint64_t)(t.p * 2u + rank) * kBP + i, qr = (uint64_t)t.q * p.bn + i;
      auto word = [&](const uint8_t* scales, uint64_t row) {
        return __ldg(reinterpret_cast<const uint32_t*>(scales + row * p.scale_cols + kb));
      };
      next[0] = pr < p.n ? word(p.p_scales, pr) : 0u;
      next[1] = i < p.bn && qr < p.m ? word(p.q_scales, qr) : 0u;
      next[2] = i + 128u < p.bn && qr + 128u < p.m ? word(p.q_scales, qr + 128u) : 0u;
    };
    if (u < units) {
      t = unit_of(p, u);
      kb = t.kb0;
      fetch();
    }
    while (u < units) {
      uint32_t* words = scale_words[group & 1u];
      words[i] = next[0];
      words[kBP + i] = next[1];
      words[kBP + 128u + i] = next[2];
      // The four warps meet, and end together if one of them gave up waiting.
      if (meet_any(gave_up)) break;
      const uint32_t set = group % kSets, use = group / kSets;
      kb += 4u;
      if (kb >= t.kb1) {
        u += ustep;
        if (u < units) {
          t = unit_of(p, u);
          kb = t.kb0;
        }
      }
      if (u < units) fetch();
      uint32_t w[12];
#pragma unroll
      for (uint32_t q = 0; q < 12; ++q) w[q] = words[q * 32u + lane];
      // the set's last group has been read
      const bool freed = lane != 0 || use == 0u || wait(&group_done[set], (use - 1u) & 1u);
      gave_up = !__shfl_sync(0xffffffffu, freed ? 1u : 0u, 0);
      if (!gave_up) {
        tc_fence_after();
        const uint32_t ta = tmem + kScaleCol + set * 16u + (quad << 21);
        tmem_st_x4(ta, w);
        tmem_st_x4(ta + 4u, w + 4);
        if (words_q > 4u) tmem_st_x4(ta + 8u, w + 8);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_at(mapa_shared(&scale_full[set], 0));
      }
      ++group;
    }
  } else if (warp >= kEpiWarp) {
    // Two warps a lane quadrant, taking turns at sixteen columns.
    const uint32_t quad = warp % 4u, turn = (warp - kEpiWarp) / 4u;
    uint32_t acc = 0;
    for (uint32_t u = unit0; u < units; u += ustep, ++acc) {
      const Unit t = unit_of(p, u);
      const uint32_t buf = acc & 1u;
      const bool full_ok = lane != 0 || wait(&acc_full[buf], (acc >> 1) & 1u);
      if (!__shfl_sync(0xffffffffu, full_ok ? 1u : 0u, 0)) break;
      tc_fence_after();
      const uint64_t n = (uint64_t)(t.p * 2u + rank) * kBP + quad * 32u + lane;
      const uint64_t m0 = (uint64_t)t.q * p.bn;
      const uint32_t rows = n < p.n ? (uint32_t)min((uint64_t)p.bn, p.m - m0) : 0u;
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
      uint32_t v[2][16];
      uint32_t c = turn * 16u;
      if (c < p.bn) tmem_ld_x16(ta + c, v[0]);
      tmem_ld_wait();
      while (c < p.bn) {  // the next columns load while these are stored
        if (c + 32u < p.bn) tmem_ld_x16(ta + c + 32u, v[1]);
        store16(out + c * stride, stride, v[0], rows > c ? rows - c : 0u);
        tmem_ld_wait();
        c += 32u;
        if (c >= p.bn) break;
        if (c + 32u < p.bn) tmem_ld_x16(ta + c + 32u, v[0]);
        store16(out + c * stride, stride, v[1], rows > c ? rows - c : 0u);
        tmem_ld_wait();
        c += 32u;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_at(mapa_shared(&acc_empty[buf], 0));
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no arrival, copy or MMA of the peer is under way on this CTA's memory
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
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

// Rows of a a tile and splits of K by the estimated cycles of the busiest
// pair: a block of K takes 2 BN cycles of the tensor cores (not less than the
// 128 or so that its 16 KB of b alone take to arrive), a tile about 1000 + 4 BN
// beside its MMAs, a split its parts' traffic and a second launch.
inline Plan plan(uint64_t m, uint64_t n, uint64_t k, int sm_count) {
  Plan best = {};
  double best_cost = 0.0;
  const uint32_t pairs = (uint32_t)sm_count / 2u;
  const uint32_t groups = (uint32_t)div_up(k, 512), tp = (uint32_t)div_up(n, 2 * kBP);
  const uint64_t least = div_up(m, kMaxBN);
  for (uint64_t tq = least; tq <= least + 8 && tq <= div_up(m, 16); ++tq) {
    const uint32_t bn = (uint32_t)(div_up(div_up(m, tq), 16) * 16);
    if (div_up(m, bn) != tq) continue;
    // splitting pays only while whole tiles leave SMs without work
    const uint32_t most = (uint64_t)tp * tq >= (uint64_t)pairs ? 1u : 32u;
    for (uint32_t want = 1; want <= groups && want <= most; ++want) {
      const uint32_t sg = (uint32_t)div_up(groups, want), splits = (uint32_t)div_up(groups, sg);
      if (splits != want) continue;
      const double units = (double)tp * (double)tq * splits;
      if (splits > 1 && units > 2.0 * pairs) break;
      const double blocks = sg * 4.0 < (double)div_up(k, 128) ? sg * 4.0 : (double)div_up(k, 128);
      const double waves = (double)(uint64_t)((units + pairs - 1) / pairs);
      double cost = waves * (blocks * (2.0 * bn > 128.0 ? 2.0 * bn : 128.0) + 1000.0 + 4.0 * bn);
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
      make_code_tmap(&qm, a.a_codes, a.m, (uint32_t)a.k, pl.bn / 2) != 0)
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
  const uint32_t stage = (mm::kBP + pl.bn / 2) * mm::kBK;
  p.stages = (mm::kSmemLimit - 5120u) / stage;  // beside the stages: alignment, barriers and scale words
  if (p.stages > mm::kMaxStages) p.stages = mm::kMaxStages;
  p.out = a.out;
  p.out_stride = a.out_stride;
  p.parts = static_cast<float*>(workspace);
  p.err = c.err;
  p.timeout_ns = c.timeout_ns;
  const uint32_t smem = p.stages * stage + 1024u;
  const uint64_t units = (uint64_t)pl.tiles_p * pl.tiles_q * pl.splits, pairs = (uint64_t)c.sm_count / 2;
  const uint32_t grid = 2u * (uint32_t)(units < pairs ? units : pairs);
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

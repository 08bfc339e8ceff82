// out[m][n] = sum over blocks of 128 of sa[m][b] sb[n][b] (a[m] . b[n])_b on
// E4M3 codes with power-of-two block scales.
//
// tcgen05.mma kind::mxf8f6f4 applies a scale byte per row and 32 values of K
// by itself, so a block's byte is named by its four K steps of 32 (the byte of
// a 32-bit word of scales that the instruction descriptor selects), and the
// sum over K never leaves the f32 accumulator in tensor memory: no pass over
// the accumulator per block, as a free f32 scale would need.
//
// Persistent pairs of CTAs (two SMs) share a tile of 256 rows of a and BN rows
// of b: each CTA holds 128 rows of a and half of b's in shared memory, and one
// MMA (cta_group::2) reads both halves, so a stage brings 30 KB into an SM
// where a CTA alone would need 44 KB for the same work.  Roles, concurrently:
//   warp 0      TMA: stages of 128 bytes of K
//   warp 1      tensor memory; in the first CTA the pair's MMAs
//   warps 4-7   scales: 32-bit words (four blocks of K) from global memory to
//               the four lane quadrants of tensor memory
//   warps 8-15  epilogue: accumulators to global memory
// A thread of the epilogue holds one row of out, so it packs neighbouring
// columns into 16-byte pieces of a swizzled box that TMA stores: about one
// instruction a column.  (With b's rows in the lanes, a warp stores 32 columns
// of one row at a time, five instructions a column.)
// Two accumulators: one is emptied while the next is summed.
//
// Measured (bf16 out): 8192 x 8192 x 8192 0.355 ms from a cool GPU (3.1 PFLOP/s),
// 0.40 in a row, where the power cap sets the clock; the tensor pipe is active 89 %
// of the cycles, which bounds it.  4096 x 200000 x 768 0.55 and 0.60 ms (2.7 TB/s
// of stores, where a plain fill writes 7.3): the tensor pipe is active 61 %, a tile
// takes 4700 cycles of which its six stages' MMAs are 2700.  The rest is the time
// of a tile that does not grow with K (its start, its accumulator's way out through
// two boxes a warp); which part of it counts has not been measured.  2048 x 16384 x
// 768 26 us, 2048 x 768 x 16384 30 us.
//
// K may be split over units (few tiles, long K): each unit writes f32 parts to
// the workspace and a second kernel adds them in order of K, so the result
// does not depend on timing.
#include "train_common.cuh"

namespace tessa {
namespace train {
namespace mm {

constexpr uint32_t kThreads = 512;
constexpr uint32_t kBP = 128;             // rows of a a CTA (accumulator lanes)
constexpr uint32_t kMaxBN = 224;          // rows of b a tile: two accumulators leave 64 of 512 columns to the scales
constexpr uint32_t kBK = 128;             // bytes of K a stage
constexpr uint32_t kScaleCol = 448;       // tensor memory columns of the scales
constexpr uint32_t kSets = 4;             // sets of 16: the scale warps run up to three groups ahead
constexpr uint32_t kRing = 6, kAhead = 4;  // groups of scale words in shared memory, and under way of them
constexpr uint32_t kMaxStages = 10;
constexpr uint32_t kBoxBytes = 2048;      // one TMA store of a warp: 32 rows of 64 bytes
constexpr uint32_t kBoxes = 2;            // a warp of the epilogue
constexpr uint32_t kSmemLimit = 227u * 1024u;
constexpr uint32_t kStatic = 10u * 1024u;  // barriers and scale words, and a little
constexpr uint64_t kGivenUpNs = 1000000ull;  // for what is still under way after a wait gave up
constexpr uint32_t kScaleWarp = 4, kEpiWarp = 8;

struct Params {
  const uint8_t* p_scales;  // of the operand in the accumulator's lanes: a, or b where swapped
  const uint8_t* q_scales;  // of the other
  uint64_t scale_cols;
  uint64_t rows_p, rows_q;  // m and n, or n and m where the operands are swapped
  uint64_t m;
  uint32_t kblocks;         // blocks of 128
  uint32_t ksteps;          // steps of 32 that hold data
  uint32_t bn;
  uint32_t tiles_p, tiles_q;
  uint32_t splits, split_groups;  // groups of four blocks a split
  uint32_t raster;          // tiles along b that go together
  uint32_t stages;
  void* out;
  uint64_t out_stride;
  float* parts;             // splits x m x parts_stride, splits > 1
  uint64_t parts_stride;    // n rounded up to 4
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

// Four bytes to shared memory, asynchronously; zero where there is no such row.
__device__ __forceinline__ void copy_word(uint32_t* dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 4u : 0u)
               : "memory");
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

template <class O>
__device__ __forceinline__ uint4 pack8(const uint32_t* v) {
  Vec<O, 8> o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o.v[i] = from_f32<O>(__uint_as_float(v[i]));
  return *reinterpret_cast<const uint4*>(&o);
}

__device__ __forceinline__ void store_box(const CUtensorMap* map, uint32_t box, int32_t x, int32_t y, int32_t z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(box), "r"(x), "r"(y), "r"(z)
               : "memory");
}

struct Unit {
  uint32_t p, q;       // tile
  uint32_t kb0, kb1;   // blocks of K
  uint32_t split;
};

// Tiles in blocks of `raster` along b, a's tiles one after the other within a
// block: the tiles in flight write neighbouring pieces of the same rows of out,
// and find the block's rows of b in L2.
__device__ __forceinline__ Unit unit_of(const Params& p, uint32_t u) {
  Unit r;
  r.split = u % p.splits;
  const uint32_t t = u / p.splits;
  const uint32_t block = t / (p.raster * p.tiles_p), in = t % (p.raster * p.tiles_p);
  const uint32_t wide = min(p.raster, p.tiles_q - block * p.raster);
  r.q = block * p.raster + in % wide;
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

// Accumulator columns of the lane's place: out[i * stride], i < rows.  Four
// pointers, so that a store does not wait for the address of the one before.
template <class O>
__device__ __forceinline__ void store32(O* out, uint64_t stride, const uint32_t (&v)[32], uint32_t rows) {
  O *p0 = out, *p1 = out + stride, *p2 = p1 + stride, *p3 = p2 + stride;
  const uint64_t step = 4u * stride;
#pragma unroll
  for (uint32_t i = 0; i < 32; i += 4) {
    if (i < rows) *p0 = from_f32<O>(__uint_as_float(v[i]));
    if (i + 1u < rows) *p1 = from_f32<O>(__uint_as_float(v[i + 1]));
    if (i + 2u < rows) *p2 = from_f32<O>(__uint_as_float(v[i + 2]));
    if (i + 3u < rows) *p3 = from_f32<O>(__uint_as_float(v[i + 3]));
    p0 += step;
    p1 += step;
    p2 += step;
    p3 += step;
  }
}

// 128 bytes of a row (32 f32 or 64 16-bit columns) of the accumulator as eight
// 16-byte pieces.
template <class O>
__device__ __forceinline__ void load_row(uint32_t taddr, uint4 (&piece)[8]) {
  uint32_t v[32];
  if constexpr (sizeof(O) == 4) {
    tmem_ld_32x32b_x32(taddr, v);
    tmem_ld_wait();
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) piece[j] = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  } else {
    uint32_t w[32];
    tmem_ld_32x32b_x32(taddr, v);
    tmem_ld_32x32b_x32(taddr + 32u, w);
    tmem_ld_wait();
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      piece[j] = pack8<O>(v + 8 * j);
      piece[4 + j] = pack8<O>(w + 8 * j);
    }
  }
}

template <class O, bool PARTS, bool SWAP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    fp8_matmul_kernel(const __grid_constant__ CUtensorMap pmap, const __grid_constant__ CUtensorMap qmap,
                      const __grid_constant__ CUtensorMap omap, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~(uintptr_t)1023u);
  // In the first CTA: full, scale_full and acc_empty count both CTAs' work.
  // The other barriers are signalled in both CTAs.
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], scale_full[kSets], group_done[kSets],
      acc_full[2], acc_empty[2], drained;
  __shared__ uint32_t scale_words[kRing][kBP + 256];  // a group's words: a's rows, b's rows
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
    // The block may not end before its copies have landed and before the MMAs
    // that read them have signalled both CTAs: a signal that came later would
    // find no barrier.  Each stage's last use says both.
    if (lane == 0) {
      uint32_t dummy = 0u;
      const uint64_t limit = ok ? p.timeout_ns : kGivenUpNs;
      for (uint32_t i = filled > p.stages ? filled - p.stages : 0u; i < filled; ++i)
        mbar_wait(&empty[i % p.stages], (i / p.stages) & 1u, &dummy, p.err, limit);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
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
            const uint64_t pd = base + s * desc_step, qd = pd + (kBP * kBK >> 4);
            ok &= wait_at(full_base + s * 8u, phase, abort_flag, p.err, p.timeout_ns);
            tc_fence_after();
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
            const uint64_t pd = base + s * desc_step, qd = pd + (kBP * kBK >> 4);
            const uint32_t steps = p.ksteps - b * 4u;  // 1 to 3
            ok &= wait_at(full_base + s * 8u, phase, abort_flag, p.err, p.timeout_ns);
            tc_fence_after();
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
    // every quadrant: this CTA's 128 rows of a, all BN rows of b.  Thread i
    // fetches the words of row i of a and of rows i and i + 128 of b into a
    // ring in shared memory, kAhead groups before they are used (a group may
    // be a whole tile, shorter than a load from HBM), and all four warps read
    // them there.
    const uint32_t quad = warp - kScaleWarp, i = threadIdx.x - kScaleWarp * 32u;
    const uint32_t words_q = (p.bn + 31u) / 32u;
    uint32_t u = unit0, kb = 0, kb1 = 0, fetched = 0;  // the next group to fetch
    const uint8_t *src_p = nullptr, *src_q = nullptr, *src_r = nullptr;
    bool has_p = false, has_q = false, has_r = false;
    auto open_unit = [&]() {
      if (u >= units) return;
      const Unit t = unit_of(p, u);
      const uint64_t pr = (uint64_t)(t.p * 2u + rank) * kBP + i, qr = (uint64_t)t.q * p.bn + i;
      kb = t.kb0;
      kb1 = t.kb1;
      has_p = pr < p.rows_p;
      has_q = i < p.bn && qr < p.rows_q;
      has_r = i + 128u < p.bn && qr + 128u < p.rows_q;
      src_p = p.p_scales + (has_p ? pr : 0u) * p.scale_cols;
      src_q = p.q_scales + (has_q ? qr : 0u) * p.scale_cols;
      src_r = p.q_scales + (has_r ? qr + 128u : 0u) * p.scale_cols;
    };
    auto fetch = [&]() {
      if (u < units) {
        uint32_t* words = scale_words[fetched % kRing];
        copy_word(words + i, src_p + kb, has_p);
        copy_word(words + kBP + i, src_q + kb, has_q);
        copy_word(words + kBP + 128u + i, src_r + kb, has_r);
        ++fetched;
        kb += 4u;
        if (kb >= kb1) {
          u += ustep;
          open_unit();
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    open_unit();
    for (uint32_t g = 0; g < kAhead; ++g) fetch();
    bool gave_up = false;
    uint32_t done = 0;  // groups handed to the MMAs
    for (uint32_t group = 0; group < fetched; ++group) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
      // The four warps meet, and end together if one of them gave up waiting.
      if (meet_any(gave_up)) break;
      const uint32_t* words = scale_words[group % kRing];
      uint32_t w[12];
#pragma unroll
      for (uint32_t q = 0; q < 12; ++q) w[q] = words[q * 32u + lane];
      fetch();  // into the place of a group that all four have read (they have met since)
      const uint32_t set = group % kSets, use = group / kSets;
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
        ++done;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // The last groups' signals, too, come while this CTA is there.
    if (quad == 0 && lane == 0) {
      uint32_t dummy = 0u;
      const uint64_t limit = *abort_flag ? kGivenUpNs : p.timeout_ns;
      for (uint32_t g = done > kSets ? done - kSets : 0u; g < done; ++g)
        mbar_wait(&group_done[g % kSets], (g / kSets) & 1u, &dummy, p.err, limit);
    }
    __syncwarp();
  } else if (warp >= kEpiWarp) {
    // Two warps a lane quadrant take turns at 128 bytes of its rows.
    const uint32_t quad = warp % 4u, turn = (warp - kEpiWarp) / 4u;
    [[maybe_unused]] uint8_t* boxes = smem + p.stages * stage_bytes + (warp - kEpiWarp) * kBoxes * kBoxBytes;
    uint32_t acc = 0;
    for (uint32_t u = unit0; u < units; u += ustep, ++acc) {
      const Unit t = unit_of(p, u);
      const uint32_t buf = acc & 1u;
      const bool full_ok = lane != 0 || wait(&acc_full[buf], (acc >> 1) & 1u);
      if (!__shfl_sync(0xffffffffu, full_ok ? 1u : 0u, 0)) break;
      tc_fence_after();
      const uint64_t p0 = (uint64_t)(t.p * 2u + rank) * kBP + quad * 32u, q0 = (uint64_t)t.q * p.bn;
      const uint32_t rows = p0 < p.rows_p ? (uint32_t)min((uint64_t)32u, p.rows_p - p0) : 0u;
      const uint32_t cols = rows ? (uint32_t)min((uint64_t)p.bn, p.rows_q - q0) : 0u;
      const uint32_t ta = tmem + buf * kMaxBN + (quad << 21);  // lane quad * 32
      O* out = PARTS ? reinterpret_cast<O*>(p.parts) + (uint64_t)t.split * p.m * p.parts_stride : static_cast<O*>(p.out);
      const uint64_t stride = PARTS ? p.parts_stride : p.out_stride;
      if constexpr (SWAP) {
        // A column of the accumulator is 32 neighbours of one row of out.
        out += q0 * stride + p0 + lane;
        for (uint32_t c = turn * 32u; c < cols; c += 64u) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(ta + c, v);  // BN is a multiple of 32
          tmem_ld_wait();
          if (lane < rows) store32(out + c * stride, stride, v, cols - c);
          __syncwarp();  // the next load is the whole warp's
        }
      } else {
        constexpr uint32_t kCols = 64u / sizeof(O);  // of a box, two boxes a turn
        for (uint32_t c = turn * 2u * kCols; c < cols; c += 4u * kCols) {
          uint4 piece[8];
          load_row<O>(ta + c, piece);  // may read past BN into other columns of the allocation
          // the last stores out of the boxes have read them
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(boxes + j / 4u * kBoxBytes + lane * 64u + ((j ^ (lane >> 1)) & 3u) * 16u) =
                piece[j];
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {  // out's right and lower edges TMA cuts
            store_box(&omap, smem_u32(boxes), (int32_t)(q0 + c), (int32_t)p0, (int32_t)t.split);
            if (cols - c > kCols)
              store_box(&omap, smem_u32(boxes) + kBoxBytes, (int32_t)(q0 + c + kCols), (int32_t)p0, (int32_t)t.split);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_at(mapa_shared(&acc_empty[buf], 0));
    }
    // the boxes may not go before the stores have read them
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
    // The pair's MMAs read the second CTA's memory until they have all completed,
    // too.  This warp has seen the last tile by now, so the wait is as short as any
    // other: from the kernel's start it would be the whole product's time, which
    // the limit of one wait says nothing about.  (Behind the block's barrier it made
    // the compiler's MMA loop slower: 8192 x 8192 x 8192 361 us instead of 355.)
    if (rank == 1 && warp == kEpiWarp && lane == 0) {
      uint32_t dummy = 0u;
      mbar_wait(&drained, 0u, &dummy, p.err, p.timeout_ns);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no arrival, copy or MMA of the peer is under way on this CTA's memory
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// out = the parts' sum in order of K; a row of blocks to a row of out, four
// columns a thread.
template <class O>
__global__ void __launch_bounds__(128) add_parts_kernel(const float* parts, uint64_t parts_stride, uint32_t splits,
                                                        uint64_t m, uint64_t n, O* out, uint64_t out_stride, bool vec) {
  const uint64_t n0 = ((uint64_t)blockIdx.x * 128u + threadIdx.x) * 4u, total = m * parts_stride;
  if (n0 >= n) return;
  for (uint64_t r = blockIdx.y; r < m; r += gridDim.y) {
    const float* src = parts + r * parts_stride + n0;
    O* dst = out + r * out_stride + n0;
    float4 s = __ldcs(reinterpret_cast<const float4*>(src));
#pragma unroll 4
    for (uint32_t k = 1; k < splits; ++k) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(src + k * total));
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    Vec<O, 4> o;
    o.v[0] = from_f32<O>(s.x);
    o.v[1] = from_f32<O>(s.y);
    o.v[2] = from_f32<O>(s.z);
    o.v[3] = from_f32<O>(s.w);
    if (vec) {  // rows of out aligned to four elements, n a multiple of 4
      *reinterpret_cast<Vec<O, 4>*>(dst) = o;
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        if (n0 + i < n) dst[i] = o.v[i];
    }
  }
}

struct Plan {
  uint32_t bn, tiles_p, tiles_q, splits, split_groups;
};

// Rows of b a tile and splits of K by the estimated cycles of the busiest
// pair: a block of K takes 2 BN cycles of the tensor cores (156 at least: the
// four MMAs' issue), a tile about 1500 beside its MMAs, a split its parts'
// traffic and a second launch.
inline Plan plan(uint64_t rows_p, uint64_t rows_q, uint64_t k, int sm_count) {
  Plan best = {};
  double best_cost = 0.0;
  const uint32_t pairs = (uint32_t)sm_count / 2u;
  const uint32_t groups = (uint32_t)div_up(k, 512), tp = (uint32_t)div_up(rows_p, 2 * kBP);
  const uint64_t least = div_up(rows_q, kMaxBN);
  // The tensor core cuts each sum's low bits, always towards zero: 4096 terms
  // of one sign end up 1.4e-6 off, and it grows with their number.  Parts of at
  // most 8192 terms are added with full rounding.
  const uint32_t fewest = (uint32_t)div_up(groups, 16);
  // tile counts that fill whole rounds of the SM pairs, and the fewest
  const uint64_t wave = pairs / tp ? pairs / tp : 1;
  for (uint64_t i = 0; i < 12; ++i) {
    const uint64_t tq = i < 8 ? least + i : div_up(least, wave) * wave + (i - 8) * wave;
    if (tq > div_up(rows_q, 32)) continue;
    const uint32_t bn = (uint32_t)(div_up(div_up(rows_q, tq), 32) * 32);
    if (div_up(rows_q, bn) != tq) continue;
    // splitting pays only while whole tiles leave SMs without work
    const uint32_t most = (uint64_t)tp * tq >= (uint64_t)pairs ? 1u : 32u;
    for (uint32_t want = fewest; want <= groups && (want <= most || want == fewest); ++want) {
      const uint32_t sg = (uint32_t)div_up(groups, want), splits = (uint32_t)div_up(groups, sg);
      if (splits != want) continue;
      const uint64_t units = (uint64_t)tp * tq * splits;
      if (want > fewest && units > 2 * pairs) break;
      const double blocks = sg * 4.0 < (double)div_up(k, 128) ? sg * 4.0 : (double)div_up(k, 128);
      double cost = (double)div_up(units, pairs) * (blocks * (2.0 * bn > 156.0 ? 2.0 * bn : 156.0) + 1500.0);
      if (splits > 1) cost += 5000.0 + 8.0 * splits * (double)rows_p * (double)rows_q / 3500.0;
      if (best.bn == 0 || cost < best_cost) {
        best = {bn, tp, (uint32_t)tq, splits, sg};
        best_cost = cost;
      }
    }
  }
  return best;
}

// The plan of the calling thread's last few shapes (the search takes longer
// than a launch).
inline Plan plan_of(uint64_t rows_p, uint64_t rows_q, uint64_t k, int sm_count) {
  struct Entry {
    uint64_t p = 0, q = 0, k = 0;
    int sms = 0;
    Plan plan;
  };
  thread_local Entry kept[16];
  Entry& e = kept[(rows_p * 31 + rows_q * 7 + k / 16) % 16];
  if (e.p != rows_p || e.q != rows_q || e.k != k || e.sms != sm_count) {
    e.plan = plan(rows_p, rows_q, k, sm_count);
    e.p = rows_p;
    e.q = rows_q;
    e.k = k;
    e.sms = sm_count;
  }
  return e.plan;
}

template <class O, bool PARTS, bool SWAP>
cudaError_t launch(const CUtensorMap& pm, const CUtensorMap& qm, const CUtensorMap& om, const Params& p, int device, uint32_t smem,
                   uint32_t grid, cudaStream_t stream) {
  static SmemRaised raised;
  cudaError_t e = raise_smem(fp8_matmul_kernel<O, PARTS, SWAP>, device, (int)(kSmemLimit - kStatic), raised);
  if (e != cudaSuccess) return e;
  fp8_matmul_kernel<O, PARTS, SWAP><<<grid, kThreads, smem, stream>>>(pm, qm, om, p);
  return cudaGetLastError();
}

}  // namespace mm

constexpr uint64_t kFewRows = 8;

}  // namespace train

// Products that fp8_few_rows.cu takes.
static bool few_rows(uint64_t m, uint64_t n) { return m <= train::kFewRows || n <= train::kFewRows; }

uint64_t fp8_matmul_workspace(uint64_t m, uint64_t n, uint64_t k, int sm_count) {
  using namespace train;
  if (m == 0 || n == 0 || k == 0 || few_rows(m, n)) return 0;
  const uint32_t one = mm::plan_of(m, n, k, sm_count).splits, other = mm::plan_of(n, m, k, sm_count).splits;
  const uint32_t splits = one > other ? one : other;  // which of the two depends on out's alignment
  return splits > 1 ? (uint64_t)splits * m * div_up(n, 4) * 16 : 0;
}

uint64_t fp8_matmul_units(uint64_t m, uint64_t n, uint64_t k, int sm_count) {
  using namespace train;
  if (m == 0 || n == 0 || k == 0 || few_rows(m, n)) return 0;
  auto units = [&](uint64_t rows_p, uint64_t rows_q) {
    const mm::Plan p = mm::plan_of(rows_p, rows_q, k, sm_count);
    return (uint64_t)p.tiles_p * p.tiles_q * p.splits;
  };
  const uint64_t one = units(m, n), other = units(n, m);  // which of the two depends on out's alignment
  return one > other ? one : other;
}

cudaError_t launch_matmul_fp8(const tessa_fp8_matmul_args& a, void* workspace, const AsyncCtx& c,
                              cudaStream_t stream) {
  using namespace train;
  const uint32_t ob = type_bytes(a.out_dtype);
  if (a.k == 0)
    return cudaMemset2DAsync(a.out, (a.m > 1 ? a.out_stride : a.n) * ob, 0, a.n * ob, a.m, stream);
  if (few_rows(a.m, a.n)) return launch_fp8_few_rows(a, c, stream);
  // b's rows take the accumulator's lanes (then out is stored straight, 32
  // neighbours at a time) where a has few rows, which would leave the lanes
  // empty (against 200000 x 768, f32 scores: m = 16 takes 39 us so and 47
  // otherwise, m = 128 54 and 55, m = 192 65 and 59), and where out's rows do
  // not suit TMA.
  CUtensorMap pm, qm, om = {};
  bool swap = a.m <= mm::kBP;
  mm::Plan pl = mm::plan_of(a.m, a.n, a.k, c.sm_count);
  if (!swap && pl.splits == 1) {
    const uint64_t stride = a.m > 1 ? a.out_stride : div_up(a.n, 8) * 8;
    swap = reinterpret_cast<uintptr_t>(a.out) % 16 != 0 || stride * ob % 16 != 0 ||
           make_store_tmap(&om, a.out, a.out_dtype, a.m, a.n, stride, 1) != 0;
  }
  if (swap) pl = mm::plan_of(a.n, a.m, a.k, c.sm_count);
  mm::Params p = {};
  p.parts = static_cast<float*>(workspace);
  p.parts_stride = div_up(a.n, 4) * 4;
  if (!swap && pl.splits > 1 &&
      make_store_tmap(&om, p.parts, TESSA_F32, a.m, a.n, p.parts_stride, pl.splits) != 0)
    return cudaErrorInvalidValue;
  p.rows_p = swap ? a.n : a.m;
  p.rows_q = swap ? a.m : a.n;
  if (make_code_tmap(&pm, swap ? a.b_codes : a.a_codes, p.rows_p, (uint32_t)a.k, mm::kBP) != 0 ||
      make_code_tmap(&qm, swap ? a.a_codes : a.b_codes, p.rows_q, (uint32_t)a.k, pl.bn / 2) != 0)
    return cudaErrorInvalidValue;
  p.p_scales = swap ? a.b_scales : a.a_scales;
  p.q_scales = swap ? a.a_scales : a.b_scales;
  p.scale_cols = div_up(a.k, 512) * 4;
  p.m = a.m;
  p.kblocks = (uint32_t)div_up(a.k, 128);
  p.ksteps = (uint32_t)div_up(a.k, 32);
  p.bn = pl.bn;
  p.tiles_p = pl.tiles_p;
  p.tiles_q = pl.tiles_q;
  p.splits = pl.splits;
  p.split_groups = pl.split_groups;
  // one tile an SM pair, as far as 32 MB of the columns' operand go
  const uint64_t fit = (32ull << 20) / (a.k * pl.bn), pairs = (uint64_t)c.sm_count / 2;
  p.raster = (uint32_t)(fit > pairs ? pairs : fit < 8 ? 8 : fit);
  const uint32_t stage = (mm::kBP + pl.bn / 2) * mm::kBK, boxes = swap ? 0u : 8u * mm::kBoxes * mm::kBoxBytes;
  p.stages = (mm::kSmemLimit - mm::kStatic - 1024u - boxes) / stage;
  if (p.stages > mm::kMaxStages) p.stages = mm::kMaxStages;
  p.out = a.out;
  p.out_stride = a.out_stride;
  p.err = c.err;
  p.timeout_ns = c.timeout_ns;
  const uint32_t smem = p.stages * stage + boxes + 1024u;
  const uint64_t units = (uint64_t)pl.tiles_p * pl.tiles_q * pl.splits;
  const uint32_t grid = 2u * (uint32_t)(units < pairs ? units : pairs);
  if (pl.splits == 1)
    return with_type(a.out_dtype, [&](auto o) {
      using O = decltype(o);
      return swap ? mm::launch<O, false, true>(pm, qm, om, p, c.device, smem, grid, stream)
                  : mm::launch<O, false, false>(pm, qm, om, p, c.device, smem, grid, stream);
    });
  cudaError_t e = swap ? mm::launch<float, true, true>(pm, qm, om, p, c.device, smem, grid, stream)
                       : mm::launch<float, true, false>(pm, qm, om, p, c.device, smem, grid, stream);
  if (e != cudaSuccess) return e;
  const bool vec = vector_elems(a.out, a.m, a.n, a.out_stride, ob, 4) == 4;
  const dim3 blocks((uint32_t)div_up(a.n, 512), (uint32_t)(a.m < 32768 ? a.m : 32768));
  return with_type(a.out_dtype, [&](auto o) {
    using O = decltype(o);
    mm::add_parts_kernel<O><<<blocks, 128, 0, stream>>>(p.parts, p.parts_stride, pl.splits, a.m, a.n,
                                                        static_cast<O*>(a.out), a.out_stride, vec);
    return cudaGetLastError();
  });
}

}  // namespace tessa

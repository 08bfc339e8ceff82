// Rows out of a table by id, scaled, and the gradient of that lookup.
//
// Lookup: out[t] = s * table[id_t].  A copy: bound by the bytes of the rows
// read and written.
//
// Gradient: grad[v] = s * sum_{t: id_t = v} dout[t].  Atomic adds would give
// another order, and other bits, every time, and a popular row would serialise
// them.  Some thousand entries are compared with one another, in one launch.
// More are sorted as (id, t) (stable radix sort, digits of at most 10 bits) and
// cut into tiles of 32 sorted entries (8 of fewer entries), and one warp sums a
// tile's rows run by run in f32: a run inside the tile is written at once, a run
// that crosses a tile border leaves its part in the workspace, and a last kernel
// adds each such run's parts.  Every tile holds as many entries however popular
// one id is, so skew costs nothing but the parts.  131072 rows of 128 f32 into
// 200000, skewed ids: 65 us in a graph.  Under the profiler, whose cold launches
// come to 82, the sort's four take 51 (39 without the clearing of other rows
// beside it), the tiles 16 (4 TB/s), the parts 15; adding to the gradient
// instead takes 49.
#include "train_common.cuh"

namespace tessa {
namespace train {

template <class T, class O, int VE>
__global__ void __launch_bounds__(256) lookup_kernel(const tessa_lookup_args a, uint32_t lanes, uint32_t* err) {
  const uint32_t per_block = 256u / lanes;  // rows a block
  const uint64_t t = (uint64_t)blockIdx.x * per_block + threadIdx.x / lanes;
  if (t >= a.count) return;
  int64_t id = a.id_bits == 32 ? (int64_t)static_cast<const int32_t*>(a.ids)[t] : static_cast<const int64_t*>(a.ids)[t];
  const bool ok = id >= 0 && (uint64_t)id < a.table_rows;
  if (!ok && id != -1) report(err, TESSA_DEVERR_BAD_ROW);
  const T* src = static_cast<const T*>(a.table) + (ok ? (uint64_t)id * a.table_stride : 0ull);
  O* dst = static_cast<O*>(a.out) + t * a.out_stride;
  const uint32_t step = lanes * VE;
#pragma unroll 4
  for (uint32_t c = threadIdx.x % lanes * VE; c < a.dim; c += step) {
    Vec<O, VE> o;
    if (ok) {
      const Vec<T, VE> x = *reinterpret_cast<const Vec<T, VE>*>(src + c);
#pragma unroll
      for (int i = 0; i < VE; ++i) o.v[i] = from_f32<O>(a.scale * to_f32(x.v[i]));
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) o.v[i] = from_f32<O>(0.0f);
    }
    *reinterpret_cast<Vec<O, VE>*>(dst + c) = o;
  }
}

// ------------------------------------------------------------------- sort

// After the one-launch sort the sums are launched ahead of its end (programmatic
// dependent launch): a kernel lets the next one start at once, and waits for all
// of the one before to be done before it touches memory.  10000 ids over 20000 x
// 64: 22.5 us a call instead of 25; after the longer sort, 262144 ids, 126 instead
// of 120.
__device__ __forceinline__ void after_the_last() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <class... Args, class... Given>
cudaError_t launch_after(bool ahead, void (*kernel)(Args...), uint32_t grid, uint32_t threads, cudaStream_t stream,
                         Given... given) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = ahead ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, Args(given)...);
}

constexpr uint32_t kSortThreads = 512;
constexpr uint32_t kSortWarps = kSortThreads / 32;
constexpr uint32_t kMaxDigitBits = 10;
constexpr uint32_t kBatch = 8;         // keys a thread has under way

// Entries that are compared instead of sorted: 4096, and fewer or none of wide
// rows, because one block has all rows of an id and one warp all columns (skewed
// ids; 1024 over 20000 x 128 f32 7 us, 15 sorted; 4096 17 either way; 1024 x 768
// bf16 13 and 17; 2048 x 768 19 and 18; 256 x 2048 f32 55 and 36).
inline bool unsorted(uint64_t count, uint32_t dim) { return count <= 4096 && dim <= 768 && count * dim <= 1u << 20; }

constexpr uint32_t kTile = 32;         // sorted entries a warp sums,
constexpr uint32_t kShortTile = 8;     // and where there are few: a warp's chain of reads is what they wait for
constexpr uint64_t kFewIds = 8192;      // (4096 of 128 f32 17 us, 19 with long tiles; 16384 x 768 bf16 31 and 27)
constexpr uint32_t kLongRun = 64;      // tiles that a run goes on for, from which a block adds its parts

struct SortPlan {
  uint32_t passes, digit_bits, chunk, blocks;
};

inline SortPlan sort_plan(uint64_t count, uint64_t table_rows) {
  uint32_t bits = 1;
  while (bits < 32 && (table_rows >> bits)) ++bits;  // keys 0 .. table_rows
  SortPlan p;
  p.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digit_bits = (bits + p.passes - 1) / p.passes;
  // At most 128 blocks, of a multiple of 1024 entries: every block reads all
  // blocks' digit counts.  65536 entries, gradient of 128 f32 columns: 56 us with
  // 1024 a block, 58 with 2048; 131072: 70 with 1024 or 2048, 77 with 4096.
  p.chunk = 1024u * (uint32_t)div_up(count, 1024ull * 128ull);
  p.blocks = (uint32_t)div_up(count, p.chunk ? p.chunk : 1);
  return p;
}

// Key of entry i of the first pass: its id, or table_rows for padding and bad ids.
__device__ __forceinline__ uint32_t id_key(const void* ids, uint32_t id_bits, uint64_t i, uint64_t table_rows,
                                           uint32_t* err) {
  const int64_t id = id_bits == 32 ? (int64_t)static_cast<const int32_t*>(ids)[i] : static_cast<const int64_t*>(ids)[i];
  if (id >= 0 && (uint64_t)id < table_rows) return (uint32_t)id;
  if (id != -1) report(err, TESSA_DEVERR_BAD_ROW);
  return (uint32_t)table_rows;
}

struct SortArgs {
  const void* ids;        // first pass: the ids themselves
  uint32_t id_bits;
  const uint32_t* keys;   // later passes
  const uint32_t* pos;
  uint32_t* out_keys;
  uint32_t* out_pos;
  uint32_t* counts;       // blocks x bins
  uint32_t* runs;         // two counters, cleared for the sums
  uint64_t table_rows;
  uint32_t count, chunk, shift, bins;
  uint32_t blocks;        // that sort; those behind them clear
  uint4* clear;
  uint64_t clear_count;
  uint32_t* err;
};

// A block behind the sort's: its share of the gradient's memory becomes zero.
__device__ __forceinline__ void clear_share(const SortArgs& a) {
  const uint64_t step = (uint64_t)(gridDim.x - a.blocks) * blockDim.x;
#pragma unroll 8
  for (uint64_t i = (uint64_t)(blockIdx.x - a.blocks) * blockDim.x + threadIdx.x; i < a.clear_count; i += step)
    a.clear[i] = make_uint4(0u, 0u, 0u, 0u);
}

template <bool FIRST>
__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, uint32_t i, uint32_t* err) {
  return FIRST ? id_key(a.ids, a.id_bits, i, a.table_rows, err) : a.keys[i];
}

template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortArgs a) {
  __shared__ uint32_t bin[1u << kMaxDigitBits];
  if (blockIdx.x >= a.blocks) return clear_share(a);
  for (uint32_t b = threadIdx.x; b < a.bins; b += kSortThreads) bin[b] = 0;
  __syncthreads();
  const uint32_t lo = blockIdx.x * a.chunk, hi = min(a.count, lo + a.chunk);
  if (FIRST && blockIdx.x == 0 && threadIdx.x < 2u) a.runs[threadIdx.x] = 0u;
  for (uint32_t i = lo + threadIdx.x; i < hi; i += kBatch * kSortThreads) {
    uint32_t key[kBatch];
#pragma unroll
    for (uint32_t r = 0; r < kBatch; ++r)
      if (i + r * kSortThreads < hi) key[r] = sort_key<FIRST>(a, i + r * kSortThreads, a.err);
#pragma unroll
    for (uint32_t r = 0; r < kBatch; ++r)
      if (i + r * kSortThreads < hi) atomicAdd(&bin[(key[r] >> a.shift) & (a.bins - 1u)], 1u);
  }
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < a.bins; b += kSortThreads) a.counts[(uint64_t)blockIdx.x * a.bins + b] = bin[b];
}

// One stable scatter: a warp owns a contiguous part of the block's chunk and
// counters of its own, so entries of one digit keep their order.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(const SortArgs a) {
  extern __shared__ __align__(16) uint32_t warp_bin[];  // kSortWarps x bins: counts, then next places
  __shared__ uint32_t warp_sum[kSortWarps];
  if (blockIdx.x >= a.blocks) return clear_share(a);
  const uint32_t tid = threadIdx.x, warp = tid / 32u, lane = tid % 32u;
  const uint32_t part = a.chunk / kSortWarps;  // a multiple of 32
  const uint32_t lo = min(a.count, blockIdx.x * a.chunk + warp * part), hi = min(a.count, lo + part);
  uint32_t* mine = warp_bin + warp * a.bins;
  uint32_t key[kBatch], pos[kBatch];
  auto load = [&](uint32_t i) {
#pragma unroll
    for (uint32_t r = 0; r < kBatch; ++r) {
      const uint32_t at = i + r * 32u + lane;
      key[r] = at < hi ? sort_key<FIRST>(a, at, a.err) : 0u;
      pos[r] = FIRST || at >= hi ? at : a.pos[at];
    }
  };
  load(lo);
  for (uint32_t i = tid; i < kSortWarps * a.bins; i += kSortThreads) warp_bin[i] = 0;
  // This block's first place for each digit: entries of smaller digits
  // anywhere, and of this digit in earlier blocks.  Thread t has digits
  // 2t and 2t + 1.
  uint32_t total[2] = {0, 0}, before[2] = {0, 0};
  if (2u * tid < a.bins) {
    const uint2* c = reinterpret_cast<const uint2*>(a.counts) + tid;
#pragma unroll 8
    for (uint32_t b = 0; b < a.blocks; ++b) {
      const uint2 n = c[(uint64_t)b * (a.bins / 2u)];
      if (b < blockIdx.x) {
        before[0] += n.x;
        before[1] += n.y;
      }
      total[0] += n.x;
      total[1] += n.y;
    }
  }
  uint32_t sum = total[0] + total[1];
#pragma unroll
  for (uint32_t o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) warp_sum[warp] = sum;
  __syncthreads();
  uint32_t base = sum - total[0] - total[1];
  for (uint32_t w = 0; w < warp; ++w) base += warp_sum[w];
  // counts of each warp's part
  const bool once = part <= kBatch * 32u;  // then keys, positions and equals stay in registers
  uint32_t same[kBatch];
  auto digit = [&](uint32_t i, uint32_t r) {
    return i + r * 32u + lane < hi ? (key[r] >> a.shift) & (a.bins - 1u) : a.bins;
  };
  for (uint32_t i = lo; i < hi; i += kBatch * 32u) {
    if (i != lo) load(i);
#pragma unroll
    for (uint32_t r = 0; r < kBatch; ++r) {
      if (i + r * 32u >= hi) break;
      const uint32_t d = digit(i, r);
      same[r] = __match_any_sync(0xffffffffu, d);
      if (d < a.bins && lane == (uint32_t)__ffs(same[r]) - 1u) mine[d] += __popc(same[r]);
      __syncwarp();
    }
  }
  __syncthreads();
  if (2u * tid < a.bins) {
    uint2 n[kSortWarps];
#pragma unroll
    for (uint32_t w = 0; w < kSortWarps; ++w) n[w] = *reinterpret_cast<const uint2*>(warp_bin + w * a.bins + 2u * tid);
    uint2 place = make_uint2(base + before[0], base + total[0] + before[1]);
#pragma unroll
    for (uint32_t w = 0; w < kSortWarps; ++w) {
      *reinterpret_cast<uint2*>(warp_bin + w * a.bins + 2u * tid) = place;
      place.x += n[w].x;
      place.y += n[w].y;
    }
  }
  __syncthreads();
  for (uint32_t i = lo; i < hi; i += kBatch * 32u) {
    if (!once) load(i);
#pragma unroll
    for (uint32_t r = 0; r < kBatch; ++r) {
      if (i + r * 32u >= hi) break;
      const uint32_t d = digit(i, r);
      if (!once) same[r] = __match_any_sync(0xffffffffu, d);
      const uint32_t rank = __popc(same[r] & ((1u << lane) - 1u));
      const bool in = d < a.bins;
      const uint32_t place = in ? mine[d] + rank : 0u;
      __syncwarp();
      if (in && rank == 0) mine[d] += __popc(same[r]);
      __syncwarp();
      if (in) {
        a.out_keys[place] = key[r];
        a.out_pos[place] = pos[r];
      }
    }
  }
}

// Up to 16384 entries: one cluster of CTAs sorts them in its shared memory,
// every pass in the same launch, an entry a thread.  Per pass each warp counts
// its entries' digits, the CTAs read one another's totals, and every entry goes
// to its place, in whichever CTA that is (the last pass: to global memory).  One
// launch instead of two a pass, each nearly all latency: into 20000 rows of 128
// f32 the gradient of 8192 entries takes 17 us instead of 22, of 16384 22
// instead of 24.5.
constexpr uint32_t kClusterChunk = 1024, kClusterWarps = kClusterChunk / 32;
constexpr uint32_t kClusterMost = 16u * kClusterChunk;

__global__ void __launch_bounds__(kClusterChunk)
    sort_cluster_kernel(const SortArgs a, uint32_t passes, uint32_t digit_bits) {
  extern __shared__ uint16_t warp_digits[];  // warps x bins
  __shared__ uint2 entry[2][kClusterChunk];
  __shared__ uint32_t hist[1u << kMaxDigitBits], first_place[1u << kMaxDigitBits];
  __shared__ uint32_t warp_sum[kClusterWarps];
  if (blockIdx.x >= a.blocks) return clear_share(a);  // whole clusters
  const uint32_t ctas = a.blocks, bins = 1u << digit_bits;
  const uint32_t tid = threadIdx.x, warp = tid / 32u, lane = tid % 32u, rank = cluster_ctarank();
  const uint32_t at = rank * kClusterChunk + tid;
  uint16_t* mine = warp_digits + warp * bins;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (rank == 0 && tid < 2u) a.runs[tid] = 0u;
  cluster_sync();  // every CTA has started
  for (uint32_t pass = 0; pass < passes; ++pass) {
    const bool in = at < a.count;
    uint2 e = make_uint2(0u, 0u);  // (key, position)
    if (in) e = pass ? entry[(pass - 1u) & 1u][tid] : make_uint2(id_key(a.ids, a.id_bits, at, a.table_rows, a.err), at);
    for (uint32_t i = lane; i < bins; i += 32u) mine[i] = 0;
    __syncwarp();
    const uint32_t d = in ? (e.x >> (pass * digit_bits)) & (bins - 1u) : bins;
    const uint32_t same = __match_any_sync(0xffffffffu, d), before_me = __popc(same & ((1u << lane) - 1u));
    if (in && before_me == 0u) mine[d] = (uint16_t)__popc(same);
    __syncthreads();
    // thread t: digit t.  The warps' counts become places among this CTA's.
    if (tid < bins) {
      uint32_t n = 0;
#pragma unroll 8
      for (uint32_t w = 0; w < kClusterWarps; ++w) {
        const uint32_t c = warp_digits[w * bins + tid];
        warp_digits[w * bins + tid] = (uint16_t)n;
        n += c;
      }
      hist[tid] = n;
    }
    cluster_sync();  // and all entries of the last pass have been read
    uint32_t total = 0, before = 0;
    if (tid < bins) {
      for (uint32_t r = 0; r < ctas; ++r) {
        uint32_t n;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(n) : "r"(mapa_shared(&hist[tid], r)) : "memory");
        total += n;
        if (r < rank) before += n;
      }
    }
    uint32_t sum = total;
#pragma unroll
    for (uint32_t o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31u) warp_sum[warp] = sum;
    __syncthreads();
    uint32_t base = warp_sum[lane];
#pragma unroll
    for (uint32_t o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, base, o);
      if (lane >= o) base += v;
    }
    base = __shfl_sync(0xffffffffu, base, (warp + 31u) % 32u);  // of the warps before
    if (tid < bins) first_place[tid] = (warp ? base : 0u) + sum - total + before;
    __syncthreads();
    if (in) {
      const uint32_t place = first_place[d] + mine[d] + before_me;
      if (pass + 1u == passes) {
        a.out_keys[place] = e.x;
        a.out_pos[place] = e.y;
      } else {
        const uint32_t to = mapa_shared(&entry[pass & 1u][place % kClusterChunk], place / kClusterChunk);
        asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(to), "r"(e.x), "r"(e.y) : "memory");
      }
    }
    cluster_sync();  // the entries have arrived; nobody reads another's counts any more
  }
}

// ------------------------------------------------------------------- sums

struct SumArgs {
  const uint32_t* keys;
  const uint32_t* pos;
  float* parts;           // tiles x 2 x part_stride: run from the tile before, run into the tile after
  uint32_t* runs;         // numbers of short and of long runs that cross tiles, then the tiles that they start in:
                          // short from the front, long from the back
  uint32_t part_stride;
  uint32_t count, tile, tiles, chunks, table_rows;  // tile: entries of one
};

template <class O, int VE>
__device__ __forceinline__ Vec<O, VE>* grad_at(const tessa_lookup_grad_args& a, uint32_t row, uint32_t c) {
  return reinterpret_cast<Vec<O, VE>*>(static_cast<O*>(a.grad) + (uint64_t)row * a.grad_stride + c);
}

// ACC: `old`, read some time before, is what the sum is added to.
template <bool ACC, class O, int VE>
__device__ __forceinline__ void store_row(const tessa_lookup_grad_args& a, uint32_t row, uint32_t c,
                                          const float (&s)[VE], const Vec<O, VE>& old) {
  Vec<O, VE> o;
#pragma unroll
  for (int i = 0; i < VE; ++i) o.v[i] = from_f32<O>(ACC ? to_f32(old.v[i]) + a.scale * s[i] : a.scale * s[i]);
  *grad_at<O, VE>(a, row, c) = o;
}

// One warp: the TILE sorted entries of a tile, 32 * VE columns.
template <class T, class O, int VE, bool ACC, uint32_t TILE>
__global__ void __launch_bounds__(256) sum_tiles_kernel(const tessa_lookup_grad_args a, const SumArgs s) {
  const uint64_t w = (uint64_t)blockIdx.x * 8u + threadIdx.x / 32u;
  const uint32_t tile = (uint32_t)(w / s.chunks), lane = threadIdx.x % 32u;
  after_the_last();
  if (tile >= s.tiles) return;
  const uint32_t col = (uint32_t)(w % s.chunks) * 32u * VE + lane * VE;
  const bool in = col < a.dim;
  const uint32_t first = tile * TILE, e = first + lane;
  const bool here = lane < TILE && e < s.count;
  const uint32_t key = here ? s.keys[e] : s.table_rows;
  const uint32_t pos = here ? s.pos[e] : 0u;
  const uint32_t valid = __popc(__ballot_sync(0xffffffffu, key < s.table_rows));  // padding is sorted last
  if (valid == 0) return;
  const uint32_t prev = first ? s.keys[first - 1u] : s.table_rows;
  const uint32_t next = first + TILE < s.count ? s.keys[first + TILE] : s.table_rows;
  const uint32_t after = __shfl_down_sync(0xffffffffu, key, 1);
  const uint32_t ends = __ballot_sync(0xffffffffu, lane == TILE - 1u || after != key);
  const T* dout = static_cast<const T*>(a.dout) + col;
  float acc[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
  bool from_before = __shfl_sync(0xffffffffu, key, 0) == prev;  // the current run began in an earlier tile
  // Rows under way, against registers: 262144 rows of 768 bf16 206 us with four,
  // 232 with eight, 216 with two; adding to the gradient 195 with two, 239 with
  // four, 327 with eight.
  constexpr uint32_t kRows = ACC ? (VE < 2 ? 8 : 16 / VE) : VE == 8 ? 4 : 8;
#pragma unroll 1
  for (uint32_t b = 0; b < valid; b += kRows) {
    Vec<T, VE> x[kRows];
    Vec<O, VE> old[kRows];
#pragma unroll
    for (uint32_t q = 0; q < kRows; ++q) {
      const uint32_t p = __shfl_sync(0xffffffffu, pos, b + q);
      if (in && b + q < valid) x[q] = *reinterpret_cast<const Vec<T, VE>*>(dout + (uint64_t)p * a.dout_stride);
      if constexpr (ACC) {
        const uint32_t row = __shfl_sync(0xffffffffu, key, b + q);
        if (in && b + q < valid && (ends >> (b + q) & 1u)) old[q] = *grad_at<O, VE>(a, row, col);
      }
    }
#pragma unroll
    for (uint32_t q = 0; q < kRows; ++q) {
      if (b + q >= valid) break;
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] += to_f32(x[q].v[i]);
      if (ends >> (b + q) & 1u) {
        const uint32_t row = __shfl_sync(0xffffffffu, key, b + q);
        const bool goes_on = b + q == TILE - 1u && next == row;
        if (goes_on && !from_before && lane == 0 && w % s.chunks == 0) {
          const uint64_t far = (uint64_t)first + kLongRun * TILE;
          if (far < s.count && s.keys[far] == row) s.runs[1u + s.tiles - atomicAdd(s.runs + 1, 1u)] = tile;
          else s.runs[2u + atomicAdd(s.runs, 1u)] = tile;
        }
        if (in) {
          if (from_before || goes_on) {
            float* part = s.parts + ((uint64_t)tile * 2u + (from_before ? 0u : 1u)) * s.part_stride + col;
#pragma unroll
            for (int i = 0; i < VE; ++i) part[i] = acc[i];
          } else {
            store_row<ACC, O, VE>(a, row, col, acc, old[q]);
          }
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
        from_before = false;
      }
    }
  }
}

// The runs that cross tiles, in whatever order they were noted, 128 columns at
// a time; a run's parts are added in the order of the tiles -- the first
// tile's, then one of each later tile it reaches.  A short run is a warp's.  Of
// a long one warp r of a block adds parts r, r + 8, ..., and the warps' sums
// are added in order.
template <class O, bool ACC>
__global__ void __launch_bounds__(256) sum_parts_kernel(const tessa_lookup_grad_args a, const SumArgs s) {
  const uint32_t pieces = (s.part_stride + 127u) / 128u;
  const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
  __shared__ float4 sums[256];
  after_the_last();
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](const float4& v) {
    acc.x += v.x;
    acc.y += v.y;
    acc.z += v.z;
    acc.w += v.w;
  };
  auto part = [&](uint32_t tile, uint32_t j, uint32_t col) {
    const uint64_t p = j ? ((uint64_t)tile + j) * 2u : (uint64_t)tile * 2u + 1u;
    return *reinterpret_cast<const float4*>(s.parts + p * s.part_stride + col);
  };
  Vec<O, 1> old[4];
  auto load_old = [&](uint32_t row, uint32_t col) {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      if (ACC && col + i < a.dim) old[i] = *grad_at<O, 1>(a, row, col + i);
  };
  auto store = [&](uint32_t row, uint32_t col) {
    const float v[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const float one[1] = {v[i]};
      if (col + i < a.dim) store_row<ACC, O, 1>(a, row, col + i, one, old[i]);
    }
  };
  const uint64_t shorts = (uint64_t)s.runs[0] * pieces, longs = (uint64_t)s.runs[1] * pieces;
  for (uint64_t item = (uint64_t)blockIdx.x * 8u + warp; item < shorts; item += (uint64_t)gridDim.x * 8u) {
    const uint32_t tile = s.runs[2u + item / pieces], row = s.keys[(tile + 1u) * s.tile - 1u];
    const uint32_t col = (uint32_t)(item % pieces) * 128u + lane * 4u;
    load_old(row, col);
    // later tiles that begin with the run: at most kLongRun
    uint32_t more = 0;
#pragma unroll
    for (uint32_t q = 0; q < kLongRun; q += 32u) {
      const uint64_t at = ((uint64_t)tile + 1u + q + lane) * s.tile;
      more += __popc(__ballot_sync(0xffffffffu, at < s.count && s.keys[at] == row));
    }
    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (col >= s.part_stride) continue;
#pragma unroll 4
    for (uint32_t j = 0; j <= more; ++j) add(part(tile, j, col));
    store(row, col);
  }
  for (uint64_t item = blockIdx.x; item < longs; item += gridDim.x) {
    const uint32_t tile = s.runs[1u + s.tiles - item / pieces], row = s.keys[(tile + 1u) * s.tile - 1u];
    uint32_t more = 0;
    while (true) {
      const uint64_t at = ((uint64_t)tile + 1u + more + threadIdx.x) * s.tile;
      const uint32_t got = __syncthreads_count(at < s.count && s.keys[at] == row);
      more += got;
      if (got < 256u) break;
    }
    const uint32_t col = (uint32_t)(item % pieces) * 128u + lane * 4u;
    if (warp == 0) load_old(row, col);
    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (col < s.part_stride) {
#pragma unroll 8
      for (uint32_t j = warp; j <= more; j += 8u) add(part(tile, j, col));
    }
    sums[threadIdx.x] = acc;
    __syncthreads();
    if (warp == 0 && col < s.part_stride) {
      for (uint32_t q = 1; q < 8u; ++q) add(sums[q * 32u + lane]);
      store(row, col);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------ few ids, one launch

// Up to 4096 entries: a block keeps all keys in shared memory, and a warp
// has one entry.  If no earlier one has its key, the warp sums the rows of all
// that have, in order; more than 32 of them are shared by the block's warps,
// each a part of the entries, whose sums are added in order.  Blocks behind
// these clear the rows that no id names, which they mark in a bitmap, so one
// launch does it all: 256 ids over 20000 x 128 f32 4.2 us, by sorting 11.5; over
// 200000 19 and 23, mostly clearing.  Bound by the latency of three dependent
// reads, and by an id's rows where it has many.
constexpr uint32_t kFewWarps = 8;

template <class T, class O, int VE, bool ACC>
__global__ void __launch_bounds__(256) few_ids_kernel(const tessa_lookup_grad_args a, uint32_t sum_blocks, uint32_t* err) {
  extern __shared__ __align__(16) uint32_t few_smem[];
  const uint32_t tid = threadIdx.x, warp = tid / 32u, lane = tid % 32u, count = (uint32_t)a.count;
  const uint32_t none = (uint32_t)a.table_rows;
  auto key_of = [&](uint32_t i) {
    const int64_t id = a.id_bits == 32 ? (int64_t)static_cast<const int32_t*>(a.ids)[i]
                                       : static_cast<const int64_t*>(a.ids)[i];
    const bool ok = id >= 0 && (uint64_t)id < a.table_rows;
    if (!ok && id != -1 && blockIdx.x == 0) report(err, TESSA_DEVERR_BAD_ROW);
    return ok ? (uint32_t)id : none;
  };
  if (blockIdx.x >= sum_blocks) {
    // rows [first, first + rows) of the table, vectors of VE
    const uint32_t parts = gridDim.x - sum_blocks, part = blockIdx.x - sum_blocks;
    const uint32_t per = (uint32_t)((a.table_rows + parts - 1u) / parts);
    const uint64_t first = (uint64_t)part * per;
    if (first >= a.table_rows) return;
    const uint32_t rows = (uint32_t)min((uint64_t)per, a.table_rows - first);
    for (uint32_t i = tid; i < (rows + 31u) / 32u; i += 256u) few_smem[i] = 0u;
    __syncthreads();
    for (uint32_t i = tid; i < count; i += 256u) {
      const uint64_t r = (uint64_t)key_of(i) - first;  // (past the end for padding and other blocks' rows)
      if (r < rows) atomicOr(few_smem + r / 32u, 1u << (r % 32u));
    }
    __syncthreads();
    const uint32_t vecs = a.dim / VE;
    Vec<O, VE> zero;
#pragma unroll
    for (int i = 0; i < VE; ++i) zero.v[i] = from_f32<O>(0.0f);
    for (uint64_t i = tid; i < (uint64_t)rows * vecs; i += 256u) {
      const uint32_t r = (uint32_t)(i / vecs), v = (uint32_t)(i - (uint64_t)r * vecs);
      if (!(few_smem[r / 32u] >> (r % 32u) & 1u)) *grad_at<O, VE>(a, (uint32_t)first + r, v * VE) = zero;
    }
    return;
  }

  const uint32_t padded = (count + 127u) / 128u * 128u;
  uint32_t* keys = few_smem;
  __shared__ uint32_t shared_entry[kFewWarps];  // entries whose key many have
  __shared__ float part_sum[kFewWarps][32 * VE];
  for (uint32_t i = tid; i < padded; i += 256u) keys[i] = i < count ? key_of(i) : none;
  __syncthreads();
  const uint4* four = reinterpret_cast<const uint4*>(keys);
  // bits 0..3: which of keys [base + 4 lane, + 4) are k, at or behind `from`
  auto matches = [&](uint32_t base, uint32_t k, uint32_t from) {
    const uint4 q = four[base / 4u + lane];
    const uint32_t m = (q.x == k ? 1u : 0u) | (q.y == k ? 2u : 0u) | (q.z == k ? 4u : 0u) | (q.w == k ? 8u : 0u);
    const uint32_t j = base + 4u * lane;
    return j >= from ? m : from - j < 4u ? m & (15u << (from - j)) : 0u;
  };
  const T* dout = static_cast<const T*>(a.dout);
  // adds the rows at lanes' positions 0 .. n - 1, in order, columns col ..
  auto add_rows = [&](float (&acc)[VE], uint32_t mine, uint32_t n, uint32_t col) {
    for (uint32_t b = 0; b < n; b += 4u) {
      Vec<T, VE> x[4];
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q) {
        const uint32_t j = __shfl_sync(0xffffffffu, mine, (b + q) % 32u);
        if (b + q < n && col < a.dim) x[q] = *reinterpret_cast<const Vec<T, VE>*>(dout + (uint64_t)j * a.dout_stride + col);
      }
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q) {
        if (b + q >= n || col >= a.dim) break;
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[i] += to_f32(x[q].v[i]);
      }
    }
  };
  const uint32_t t = blockIdx.x * kFewWarps + warp;
  const uint32_t k = t < count ? keys[t] : none;
  bool first = k != none;
  for (uint32_t base = 0; first && base < t; base += 128u) {
    const uint32_t m = matches(base, k, 0u), j = base + 4u * lane;
    const uint32_t earlier = j >= t ? 0u : t - j < 4u ? m & ((1u << (t - j)) - 1u) : m;
    first = !__any_sync(0xffffffffu, earlier != 0u);
  }
  uint32_t found = 0, mine = 0;  // lane i: position of the i-th
  if (first) {
    for (uint32_t base = t / 128u * 128u; base < count; base += 128u) {
      const uint32_t m = matches(base, k, t);
      for (uint32_t lanes = __ballot_sync(0xffffffffu, m != 0u); lanes; lanes &= lanes - 1u) {
        const uint32_t l = __ffs(lanes) - 1u;
        for (uint32_t bits = __shfl_sync(0xffffffffu, m, l); bits; bits &= bits - 1u, ++found)
          if (lane == found) mine = base + 4u * l + __ffs(bits) - 1u;
      }
    }
  }
  if (lane == 0) shared_entry[warp] = found > 32u ? t : 0xffffffffu;
  if (found && found <= 32u) {
    for (uint32_t c0 = 0; c0 < a.dim; c0 += 32u * VE) {
      const uint32_t col = c0 + lane * VE;
      Vec<O, VE> old;
      if (ACC && col < a.dim) old = *grad_at<O, VE>(a, k, col);
      float acc[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
      add_rows(acc, mine, found, col);
      if (col < a.dim) store_row<ACC, O, VE>(a, k, col, acc, old);
    }
  }
  __syncthreads();
  for (uint32_t e = 0; e < kFewWarps; ++e) {
    const uint32_t from = shared_entry[e];
    if (from == 0xffffffffu) continue;
    const uint32_t key = keys[from];
    // this warp's part of the entries, a multiple of 128
    const uint32_t per = (padded / 128u + kFewWarps - 1u) / kFewWarps * 128u;
    const uint32_t lo = warp * per, hi = min(padded, lo + per);
    for (uint32_t c0 = 0; c0 < a.dim; c0 += 32u * VE) {
      const uint32_t col = c0 + lane * VE;
      float acc[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
      uint32_t n = 0, at = 0;
      for (uint32_t base = lo; base < hi; base += 128u) {
        const uint32_t m = matches(base, key, from);
        for (uint32_t lanes = __ballot_sync(0xffffffffu, m != 0u); lanes; lanes &= lanes - 1u) {
          const uint32_t l = __ffs(lanes) - 1u;
          for (uint32_t bits = __shfl_sync(0xffffffffu, m, l); bits; bits &= bits - 1u) {
            if (lane == n) at = base + 4u * l + __ffs(bits) - 1u;
            if (++n == 32u) {
              add_rows(acc, at, 32u, col);
              n = 0;
            }
          }
        }
      }
      add_rows(acc, at, n, col);
#pragma unroll
      for (int i = 0; i < VE; ++i) part_sum[warp][lane * VE + i] = acc[i];
      __syncthreads();
      if (warp == 0 && col < a.dim) {
        Vec<O, VE> old;
        if (ACC) old = *grad_at<O, VE>(a, key, col);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          acc[i] = part_sum[0][lane * VE + i];
          for (uint32_t w = 1; w < kFewWarps; ++w) acc[i] += part_sum[w][lane * VE + i];
        }
        store_row<ACC, O, VE>(a, key, col, acc, old);
      }
      __syncthreads();
    }
  }
}

template <class F>
cudaError_t with_width(uint32_t ve, F f) {
  switch (ve) {
    case 8: return f(std::integral_constant<int, 8>());
    case 4: return f(std::integral_constant<int, 4>());
    case 2: return f(std::integral_constant<int, 2>());
    default: return f(std::integral_constant<int, 1>());
  }
}

inline uint64_t align256(uint64_t n) { return (n + 255) / 256 * 256; }

constexpr uint64_t kBeside = 100ull << 20;  // bytes of a gradient that is cleared beside the sort

struct GradSpace {
  uint64_t keys[2], pos[2], counts, runs, parts, bytes;
};

inline GradSpace grad_space(uint64_t count, uint64_t table_rows, uint32_t dim) {
  const SortPlan p = sort_plan(count, table_rows);
  GradSpace g;
  uint64_t at = 0;
  auto take = [&](uint64_t n) {
    const uint64_t here = at;
    at += align256(n);
    return here;
  };
  for (int i = 0; i < 2; ++i) g.keys[i] = take(count * 4);
  for (int i = 0; i < 2; ++i) g.pos[i] = take(count * 4);
  g.counts = take((uint64_t)p.blocks * (1u << kMaxDigitBits) * 4);
  const uint64_t tiles = div_up(count, count <= kFewIds ? kShortTile : kTile);
  g.runs = take((2 + tiles) * 4);
  g.parts = take(tiles * 2 * ((dim + 3u) / 4u * 4u) * 4);
  g.bytes = at;
  return g;
}

}  // namespace train

cudaError_t launch_embedding_lookup(const tessa_lookup_args& a, const AsyncCtx& c, cudaStream_t stream) {
  using namespace train;
  const uint32_t eb = type_bytes(a.dtype), ob = type_bytes(a.out_dtype);
  const uint32_t most = 16u / (eb > ob ? eb : ob);
  const uint32_t vt = vector_elems(a.table, a.table_rows, a.dim, a.table_stride, eb, most);
  const uint32_t ve = vector_elems(a.out, a.count, a.dim, a.out_stride, ob, vt);
  uint32_t lanes = 1;
  while (lanes < 32u && lanes * ve < a.dim) lanes <<= 1;
  const uint32_t grid = (uint32_t)div_up(a.count, 256u / lanes);
  return with_type(a.dtype, [&](auto t) {
    return with_type(a.out_dtype, [&](auto o) {
      return with_width(ve, [&](auto w) {
        lookup_kernel<decltype(t), decltype(o), decltype(w)::value><<<grid, 256, 0, stream>>>(a, lanes, c.err);
        return cudaGetLastError();
      });
    });
  });
}

uint64_t embedding_grad_workspace(uint64_t count, uint64_t table_rows, uint32_t dim) {
  return count && !train::unsorted(count, dim) ? train::grad_space(count, table_rows, dim).bytes : 0;
}

cudaError_t launch_embedding_grad(const tessa_lookup_grad_args& a, void* workspace, const AsyncCtx& c,
                                  cudaStream_t stream) {
  using namespace train;
  const uint32_t eb = type_bytes(a.dtype), ob = type_bytes(a.grad_dtype);
  // The rows that no id names are zero.  Where stores at a kernel's rate are
  // through before the sort, which leaves most SMs idle, blocks beside it clear
  // them (200000 rows, 16384 ids: 64 columns of bf16 25 us instead of 29, 128 of
  // f32 39 instead of 43; 120000 x 256 f32, 117 MB, 46 either way).  A larger
  // gradient is cleared first, at the memory's rate.
  const uint64_t row_bytes = (uint64_t)a.dim * ob, bytes = a.table_rows * row_bytes;
  const uint32_t widest = 16u / (eb > ob ? eb : ob);
  uint32_t ve = vector_elems(a.dout, a.count, a.dim, a.dout_stride, eb, widest);
  ve = vector_elems(a.grad, a.table_rows, a.dim, a.grad_stride, ob, ve);
  const bool few = a.count > 0 && unsorted(a.count, a.dim);
  const bool whole = a.table_rows == 1 || a.grad_stride == a.dim;
  const bool beside = !few && !a.accumulate && a.count > 0 && whole && bytes <= kBeside && bytes % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(a.grad) % 16 == 0;
  const bool clears = few && !a.accumulate && bytes <= kBeside;
  if (!a.accumulate && !beside && !clears) {
    const cudaError_t e = whole ? cudaMemsetAsync(a.grad, 0, bytes, stream)
                                : cudaMemset2DAsync(a.grad, a.grad_stride * ob, 0, row_bytes, a.table_rows, stream);
    if (e != cudaSuccess) return e;
  }
  if (a.count == 0) return cudaSuccess;
  if (few) {
    const uint32_t sums = (uint32_t)div_up(a.count, kFewWarps);
    // a block clears 32 KB at least; its bitmap is of a part of the rows
    const uint64_t want = div_up(bytes, 32768), most = (uint64_t)c.sm_count * 4;
    const uint32_t clear = clears ? (uint32_t)(want < most ? want : most) : 0u;
    const uint64_t keys = div_up(a.count, 128) * 512, map = clear ? div_up(div_up(a.table_rows, clear), 32) * 4 : 0;
    const uint32_t smem = (uint32_t)(keys > map ? keys : map);
    return with_type(a.dtype, [&](auto t) {
      return with_type(a.grad_dtype, [&](auto o) {
        return with_width(ve, [&](auto w) {
          constexpr int VE = decltype(w)::value;
          if (a.accumulate)
            few_ids_kernel<decltype(t), decltype(o), VE, true><<<sums, 256, smem, stream>>>(a, sums, c.err);
          else
            few_ids_kernel<decltype(t), decltype(o), VE, false><<<sums + clear, 256, smem, stream>>>(a, sums, c.err);
          return cudaGetLastError();
        });
      });
    });
  }
  const GradSpace g = grad_space(a.count, a.table_rows, a.dim);
  const SortPlan p = sort_plan(a.count, a.table_rows);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  auto at = [&](uint64_t off) { return reinterpret_cast<uint32_t*>(ws + off); };
  SortArgs s = {};
  s.ids = a.ids;
  s.id_bits = a.id_bits;
  s.table_rows = a.table_rows;
  s.count = (uint32_t)a.count;
  s.counts = at(g.counts);
  s.runs = at(g.runs);
  s.chunk = p.chunk;
  s.err = c.err;
  s.clear = static_cast<uint4*>(a.grad);
  // blocks for this launch's share, of `launches`
  auto share = [&](uint32_t launch, uint32_t launches) {
    if (!beside) return 0u;
    const uint64_t all = bytes / 16, lo = all * launch / launches, hi = all * (launch + 1) / launches;
    s.clear = static_cast<uint4*>(a.grad) + lo;
    s.clear_count = hi - lo;
    const uint64_t want = div_up(s.clear_count, 4096);
    return (uint32_t)(want < (uint64_t)c.sm_count ? want : (uint64_t)c.sm_count);
  };
  uint32_t out = 0;
  if (a.count <= kClusterMost) {
    const uint32_t ctas = (uint32_t)div_up(a.count, kClusterChunk);
    s.out_keys = at(g.keys[0]);
    s.out_pos = at(g.pos[0]);
    static SmemRaised raised, wide;
    cudaError_t e = raise_smem(sort_cluster_kernel, c.device, kClusterWarps * 2 << kMaxDigitBits, raised);
    const uint64_t bit = 1ull << (c.device & 63);
    if (e == cudaSuccess && !(wide.devices.load(std::memory_order_relaxed) & bit)) {
      e = cudaFuncSetAttribute(sort_cluster_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e == cudaSuccess) wide.devices.fetch_or(bit, std::memory_order_relaxed);
    }
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    s.blocks = ctas;
    cfg.gridDim = dim3(ctas + share(0, 1) / ctas * ctas);
    if (beside && cfg.gridDim.x == ctas) cfg.gridDim.x += ctas;
    cfg.blockDim = dim3(kClusterChunk);
    cfg.dynamicSmemBytes = kClusterWarps * 2u << p.digit_bits;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, sort_cluster_kernel, s, p.passes, p.digit_bits);
    if (e != cudaSuccess) return e;
  } else {
    s.blocks = p.blocks;
    s.bins = 1u << p.digit_bits;
    if (s.bins < 2) s.bins = 2;
    const uint32_t smem = kSortWarps * s.bins * 4u;
    static SmemRaised raised[2];
    constexpr int kMost = kSortWarps * (1 << kMaxDigitBits) * 4;
    cudaError_t e = raise_smem(sort_scatter_kernel<true>, c.device, kMost, raised[0]);
    if (e == cudaSuccess) e = raise_smem(sort_scatter_kernel<false>, c.device, kMost, raised[1]);
    if (e != cudaSuccess) return e;
    for (uint32_t pass = 0; pass < p.passes; ++pass) {
      out = pass & 1u;
      s.keys = at(g.keys[out ^ 1u]);
      s.pos = at(g.pos[out ^ 1u]);
      s.out_keys = at(g.keys[out]);
      s.out_pos = at(g.pos[out]);
      s.shift = pass * p.digit_bits;
      const uint32_t launches = 2 * p.passes, count_blocks = p.blocks + share(2 * pass, launches);
      if (pass == 0) sort_count_kernel<true><<<count_blocks, kSortThreads, 0, stream>>>(s);
      else sort_count_kernel<false><<<count_blocks, kSortThreads, 0, stream>>>(s);
      const uint32_t scatter_blocks = p.blocks + share(2 * pass + 1, launches);
      if (pass == 0) sort_scatter_kernel<true><<<scatter_blocks, kSortThreads, smem, stream>>>(s);
      else sort_scatter_kernel<false><<<scatter_blocks, kSortThreads, smem, stream>>>(s);
    }
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;

  SumArgs m = {};
  m.keys = at(g.keys[out]);
  m.pos = at(g.pos[out]);
  m.parts = reinterpret_cast<float*>(ws + g.parts);
  m.runs = at(g.runs);
  m.part_stride = (a.dim + 3u) / 4u * 4u;
  m.count = (uint32_t)a.count;
  m.tile = a.count <= kFewIds ? kShortTile : kTile;
  m.tiles = (uint32_t)div_up(a.count, m.tile);
  m.table_rows = (uint32_t)a.table_rows;
  while (ve > 1 && 32u * ve > a.dim) ve >>= 1;  // narrow rows: every lane a column rather than wide accesses
  m.chunks = (uint32_t)div_up(a.dim, 32u * ve);
  const uint32_t grid = (uint32_t)div_up((uint64_t)m.tiles * m.chunks, 8);
  return with_type(a.dtype, [&](auto t) {
    return with_type(a.grad_dtype, [&](auto o) {
      return with_width(ve, [&](auto w) {
        constexpr int VE = decltype(w)::value;
        const bool ahead = a.count <= kClusterMost;
        auto tiles = [&](auto tile, auto add) {
          return launch_after(ahead, sum_tiles_kernel<decltype(t), decltype(o), VE, decltype(add)::value, decltype(tile)::value>,
                              grid, 256, stream, a, m);
        };
        auto either = [&](auto tile) { return a.accumulate ? tiles(tile, std::true_type()) : tiles(tile, std::false_type()); };
        cudaError_t e = m.tile == kTile ? either(std::integral_constant<uint32_t, kTile>())
                                        : either(std::integral_constant<uint32_t, kShortTile>());
        if (e == cudaSuccess && m.tiles > 1) {
          const uint64_t items = div_up((uint64_t)m.tiles * div_up(a.dim, 128), 8), most = (uint64_t)c.sm_count * 8;
          const uint32_t blocks = (uint32_t)(items < most ? items : most);
          e = a.accumulate ? launch_after(ahead, sum_parts_kernel<decltype(o), true>, blocks, 256, stream, a, m)
                           : launch_after(ahead, sum_parts_kernel<decltype(o), false>, blocks, 256, stream, a, m);
        }
        return e;
      });
    });
  });
}

}  // namespace tessa

// Rows out of a table by id, scaled, and the gradient of that lookup.
//
// Lookup: out[t] = s * table[id_t].  A copy: bound by the bytes of the rows
// read and written.
//
// Gradient: grad[v] = s * sum_{t: id_t = v} dout[t].  Atomic adds would give
// another order, and other bits, every time, and a popular row would serialise
// them.  Here the entries (id, t) are sorted (stable radix sort, digits of at
// most 10 bits), cut into tiles of 32 sorted entries, and one warp sums a
// tile's rows run by run in f32: a run inside the tile is written at once, a
// run that crosses a tile border leaves its part in the workspace, and a last
// kernel adds each such run's parts.  Every tile holds 32 entries however
// popular one id is, so skew costs nothing but the parts.
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

constexpr uint32_t kSortThreads = 512;
constexpr uint32_t kSortWarps = kSortThreads / 32;
constexpr uint32_t kMaxDigitBits = 10;
constexpr uint32_t kSmallSort = 2048;  // entries that one block sorts in shared memory
constexpr uint32_t kTile = 32;         // sorted entries a warp sums

struct SortPlan {
  uint32_t passes, digit_bits, chunk, blocks;
};

inline SortPlan sort_plan(uint64_t count, uint64_t table_rows) {
  uint32_t bits = 1;
  while (bits < 32 && (table_rows >> bits)) ++bits;  // keys 0 .. table_rows
  SortPlan p;
  p.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digit_bits = (bits + p.passes - 1) / p.passes;
  // 4096 entries a block, more where that would be over 256 blocks: every
  // block reads all blocks' digit counts.
  p.chunk = 4096u * (uint32_t)div_up(count, 4096ull * 256ull);
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
  uint64_t table_rows;
  uint32_t count, chunk, shift, bins;
  uint32_t* err;
};

template <bool FIRST>
__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, uint32_t i, uint32_t* err) {
  return FIRST ? id_key(a.ids, a.id_bits, i, a.table_rows, err) : a.keys[i];
}

template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortArgs a) {
  __shared__ uint32_t bin[1u << kMaxDigitBits];
  for (uint32_t b = threadIdx.x; b < a.bins; b += kSortThreads) bin[b] = 0;
  __syncthreads();
  const uint32_t lo = blockIdx.x * a.chunk, hi = min(a.count, lo + a.chunk);
  for (uint32_t i = lo + threadIdx.x; i < hi; i += kSortThreads)
    atomicAdd(&bin[(sort_key<FIRST>(a, i, a.err) >> a.shift) & (a.bins - 1u)], 1u);
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < a.bins; b += kSortThreads) a.counts[(uint64_t)blockIdx.x * a.bins + b] = bin[b];
}

// One stable scatter: a warp owns a contiguous part of the block's chunk and
// counters of its own, so entries of one digit keep their order.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(const SortArgs a) {
  extern __shared__ uint32_t warp_bin[];  // kSortWarps x bins: counts, then next places
  __shared__ uint32_t warp_sum[kSortWarps];
  const uint32_t tid = threadIdx.x, warp = tid / 32u, lane = tid % 32u;
  for (uint32_t i = tid; i < kSortWarps * a.bins; i += kSortThreads) warp_bin[i] = 0;
  // This block's first place for each digit: entries of smaller digits
  // anywhere, and of this digit in earlier blocks.  Thread t has digits
  // 2t and 2t + 1.
  uint32_t total[2] = {0, 0}, before[2] = {0, 0};
  if (2u * tid < a.bins) {
    const uint2* c = reinterpret_cast<const uint2*>(a.counts) + tid;
#pragma unroll 8
    for (uint32_t b = 0; b < gridDim.x; ++b) {
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
  const uint32_t part = a.chunk / kSortWarps;  // a multiple of 32
  const uint32_t lo = min(a.count, blockIdx.x * a.chunk + warp * part), hi = min(a.count, lo + part);
  uint32_t* mine = warp_bin + warp * a.bins;
  for (uint32_t i = lo; i < hi; i += 32) {
    const bool in = i + lane < hi;
    const uint32_t d = in ? (sort_key<FIRST>(a, i + lane, a.err) >> a.shift) & (a.bins - 1u) : a.bins;
    const uint32_t same = __match_any_sync(0xffffffffu, d);
    if (in && lane == (uint32_t)__ffs(same) - 1u) mine[d] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  if (2u * tid < a.bins) {
#pragma unroll
    for (uint32_t q = 0; q < 2; ++q) {
      uint32_t place = base + (q ? total[0] : 0u) + before[q];
      for (uint32_t w = 0; w < kSortWarps; ++w) {
        uint32_t& n = warp_bin[w * a.bins + 2u * tid + q];
        const uint32_t c = n;
        n = place;
        place += c;
      }
    }
  }
  __syncthreads();
  for (uint32_t i = lo; i < hi; i += 32) {
    const bool in = i + lane < hi;
    const uint32_t key = in ? sort_key<FIRST>(a, i + lane, a.err) : 0u;
    const uint32_t d = in ? (key >> a.shift) & (a.bins - 1u) : a.bins;
    const uint32_t same = __match_any_sync(0xffffffffu, d);
    const uint32_t rank = __popc(same & ((1u << lane) - 1u));
    uint32_t place = in ? mine[d] + rank : 0u;
    __syncwarp();
    if (in && rank == 0) mine[d] += __popc(same);
    __syncwarp();
    if (in) {
      a.out_keys[place] = key;
      a.out_pos[place] = FIRST ? i + lane : a.pos[i + lane];
    }
  }
}

// Few entries: one block, a bitonic sort of (key, position) in shared memory.
__global__ void __launch_bounds__(1024) sort_small_kernel(const SortArgs a) {
  __shared__ uint64_t e[kSmallSort];
  uint32_t n = 32;
  while (n < a.count) n <<= 1;
  for (uint32_t i = threadIdx.x; i < n; i += 1024u)
    e[i] = i < a.count ? (uint64_t)id_key(a.ids, a.id_bits, i, a.table_rows, a.err) << 32 | i : ~0ull;
  for (uint32_t size = 2; size <= n; size <<= 1) {
    for (uint32_t step = size >> 1; step; step >>= 1) {
      __syncthreads();
      for (uint32_t j = threadIdx.x; j < n / 2; j += 1024u) {
        const uint32_t lo = 2u * j - (j & (step - 1u)), hi = lo + step;
        const uint64_t x = e[lo], y = e[hi];
        if ((x > y) == ((lo & size) == 0u)) {
          e[lo] = y;
          e[hi] = x;
        }
      }
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < a.count; i += 1024u) {
    a.out_keys[i] = (uint32_t)(e[i] >> 32);
    a.out_pos[i] = (uint32_t)e[i];
  }
}

// ------------------------------------------------------------------- sums

struct SumArgs {
  const uint32_t* keys;
  const uint32_t* pos;
  float* parts;           // tiles x 2 x part_stride: run from the tile before, run into the tile after
  uint32_t part_stride;
  uint32_t count, tiles, chunks, table_rows;
};

template <class O, int VE>
__device__ __forceinline__ void store_row(const tessa_lookup_grad_args& a, uint32_t row, uint32_t c,
                                          const float (&s)[VE]) {
  Vec<O, VE>* dst = reinterpret_cast<Vec<O, VE>*>(static_cast<O*>(a.grad) + (uint64_t)row * a.grad_stride + c);
  Vec<O, VE> o;
  if (a.accumulate) {
    o = *dst;
#pragma unroll
    for (int i = 0; i < VE; ++i) o.v[i] = from_f32<O>(to_f32(o.v[i]) + a.scale * s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) o.v[i] = from_f32<O>(a.scale * s[i]);
  }
  *dst = o;
}

// One warp: the 32 sorted entries of a tile, 32 * VE columns.
template <class T, class O, int VE>
__global__ void __launch_bounds__(256) sum_tiles_kernel(const tessa_lookup_grad_args a, const SumArgs s) {
  const uint64_t w = (uint64_t)blockIdx.x * 8u + threadIdx.x / 32u;
  const uint32_t tile = (uint32_t)(w / s.chunks), lane = threadIdx.x % 32u;
  if (tile >= s.tiles) return;
  const uint32_t col = (uint32_t)(w % s.chunks) * 32u * VE + lane * VE;
  const bool in = col < a.dim;
  const uint32_t first = tile * kTile, e = first + lane;
  const uint32_t key = e < s.count ? s.keys[e] : s.table_rows;
  const uint32_t pos = e < s.count ? s.pos[e] : 0u;
  const uint32_t valid = __popc(__ballot_sync(0xffffffffu, key < s.table_rows));  // padding is sorted last
  if (valid == 0) return;
  const uint32_t prev = first ? s.keys[first - 1u] : s.table_rows;
  const uint32_t next = first + kTile < s.count ? s.keys[first + kTile] : s.table_rows;
  const uint32_t after = __shfl_down_sync(0xffffffffu, key, 1);
  const uint32_t ends = __ballot_sync(0xffffffffu, lane == 31u || after != key);
  const T* dout = static_cast<const T*>(a.dout) + col;
  float acc[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
  bool from_before = __shfl_sync(0xffffffffu, key, 0) == prev;  // the current run began in an earlier tile
#pragma unroll 1
  for (uint32_t b = 0; b < valid; b += 8) {
    Vec<T, VE> x[8];
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) {
      const uint32_t p = __shfl_sync(0xffffffffu, pos, b + q);
      if (in && b + q < valid) x[q] = *reinterpret_cast<const Vec<T, VE>*>(dout + (uint64_t)p * a.dout_stride);
    }
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) {
      if (b + q >= valid) break;
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] += to_f32(x[q].v[i]);
      if (ends >> (b + q) & 1u) {
        const uint32_t row = __shfl_sync(0xffffffffu, key, b + q);
        const bool goes_on = b + q == 31u && next == row;
        if (in) {
          if (from_before || goes_on) {
            float* part = s.parts + ((uint64_t)tile * 2u + (from_before ? 0u : 1u)) * s.part_stride + col;
#pragma unroll
            for (int i = 0; i < VE; ++i) part[i] = acc[i];
          } else {
            store_row<O, VE>(a, row, col, acc);
          }
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
        from_before = false;
      }
    }
  }
}

// One block a tile: where a run starts in this tile and goes on, its parts in
// order -- this tile's, then one of each later tile it reaches.  The threads
// stand in rows of `groups` (4 columns each); row r adds parts r, r + R, ...,
// and the rows' sums are added in order.
template <class O>
__global__ void __launch_bounds__(256) sum_parts_kernel(const tessa_lookup_grad_args a, const SumArgs s) {
  const uint32_t tile = blockIdx.x, first = tile * kTile, last = first + kTile - 1u;
  if (last + 1u >= s.count) return;
  const uint32_t row = s.keys[last];
  if (row >= s.table_rows || s.keys[last + 1u] != row) return;
  if (first && s.keys[first] == row && s.keys[first - 1u] == row) return;  // began earlier
  uint32_t more = 0;  // later tiles that begin with the run
  while (true) {
    const uint64_t at = ((uint64_t)tile + 1u + more + threadIdx.x) * kTile;
    const uint32_t got = __syncthreads_count(at < s.count && s.keys[at] == row);
    more += got;
    if (got < 256u) break;
  }
  __shared__ float4 sums[256];
  const uint32_t groups = s.part_stride / 4u;
  const uint32_t width = groups < 256u ? groups : 256u, rows = 256u / width;
  const uint32_t r = threadIdx.x / width;
  for (uint32_t g0 = 0; g0 < groups; g0 += width) {
    const uint32_t g = g0 + threadIdx.x % width;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r < rows && g < groups) {
#pragma unroll 8
      for (uint32_t j = r; j <= more; j += rows) {
        const uint64_t part = j ? ((uint64_t)tile + j) * 2u : (uint64_t)tile * 2u + 1u;
        const float4 v = *reinterpret_cast<const float4*>(s.parts + part * s.part_stride + g * 4u);
        acc.x += v.x;
        acc.y += v.y;
        acc.z += v.z;
        acc.w += v.w;
      }
    }
    __syncthreads();
    sums[threadIdx.x] = acc;
    __syncthreads();
    if (r == 0 && g < groups) {
      for (uint32_t q = 1; q < rows; ++q) {
        const float4 v = sums[q * width + threadIdx.x];
        acc.x += v.x;
        acc.y += v.y;
        acc.z += v.z;
        acc.w += v.w;
      }
      const float v[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const float one[1] = {v[i]};
        if (g * 4u + i < a.dim) store_row<O, 1>(a, row, g * 4u + i, one);
      }
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

struct GradSpace {
  uint64_t keys[2], pos[2], counts, parts, bytes;
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
  g.parts = take(div_up(count, kTile) * 2 * ((dim + 3u) / 4u * 4u) * 4);
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
  return train::grad_space(count, table_rows, dim).bytes;
}

cudaError_t launch_embedding_grad(const tessa_lookup_grad_args& a, void* workspace, const AsyncCtx& c,
                                  cudaStream_t stream) {
  using namespace train;
  const uint32_t eb = type_bytes(a.dtype), ob = type_bytes(a.grad_dtype);
  if (!a.accumulate) {
    cudaError_t e = cudaMemset2DAsync(a.grad, (a.table_rows > 1 ? a.grad_stride : a.dim) * ob, 0, (size_t)a.dim * ob,
                                      a.table_rows, stream);
    if (e != cudaSuccess) return e;
  }
  if (a.count == 0) return cudaSuccess;
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
  s.chunk = p.chunk;
  s.err = c.err;
  uint32_t out = 0;
  if (a.count <= kSmallSort) {
    s.out_keys = at(g.keys[0]);
    s.out_pos = at(g.pos[0]);
    sort_small_kernel<<<1, 1024, 0, stream>>>(s);
  } else {
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
      if (pass == 0) {
        sort_count_kernel<true><<<p.blocks, kSortThreads, 0, stream>>>(s);
        sort_scatter_kernel<true><<<p.blocks, kSortThreads, smem, stream>>>(s);
      } else {
        sort_count_kernel<false><<<p.blocks, kSortThreads, 0, stream>>>(s);
        sort_scatter_kernel<false><<<p.blocks, kSortThreads, smem, stream>>>(s);
      }
    }
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;

  SumArgs m = {};
  m.keys = at(g.keys[out]);
  m.pos = at(g.pos[out]);
  m.parts = reinterpret_cast<float*>(ws + g.parts);
  m.part_stride = (a.dim + 3u) / 4u * 4u;
  m.count = (uint32_t)a.count;
  m.tiles = (uint32_t)div_up(a.count, kTile);
  m.table_rows = (uint32_t)a.table_rows;
  const uint32_t most = 16u / (eb > ob ? eb : ob);
  uint32_t ve = vector_elems(a.dout, a.count, a.dim, a.dout_stride, eb, most);
  ve = vector_elems(a.grad, a.table_rows, a.dim, a.grad_stride, ob, ve);
  while (ve > 1 && 32u * ve > a.dim) ve >>= 1;  // narrow rows: every lane a column rather than wide accesses
  m.chunks = (uint32_t)div_up(a.dim, 32u * ve);
  const uint32_t grid = (uint32_t)div_up((uint64_t)m.tiles * m.chunks, 8);
  return with_type(a.dtype, [&](auto t) {
    return with_type(a.grad_dtype, [&](auto o) {
      return with_width(ve, [&](auto w) {
        sum_tiles_kernel<decltype(t), decltype(o), decltype(w)::value><<<grid, 256, 0, stream>>>(a, m);
        if (m.tiles > 1) sum_parts_kernel<decltype(o)><<<m.tiles, 256, 0, stream>>>(a, m);
        return cudaGetLastError();
      });
    });
  });
}

}  // namespace tessa

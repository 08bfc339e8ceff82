// C ABI of libtessa_sm100.so: contexts, argument validation, host-side
// planning (tile tables), device scratch, the host-buffer entry points and the
// replay session that mirrors TessaCudaReplaySession (reference
// CB:34597-35305).  No exception or abort crosses the ABI: every entry point
// returns TESSA_OK or a negative TESSA_ERR_* code and records a message for
// tessa_last_error_message().
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <new>
#include <numeric>
#include <string>
#include <vector>

#include "common.cuh"

#include "kernels.h"

using namespace tessa;

namespace {

thread_local std::string g_last_error;

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

#define CUDA_TRY(expr)                                                                        \
  do {                                                                                        \
    cudaError_t _e = (expr);                                                                  \
    if (_e != cudaSuccess)                                                                    \
      return fail(_e == cudaErrorMemoryAllocation ? TESSA_ERR_OOM : TESSA_ERR_CUDA, "%s: %s (%s:%d)", #expr, \
                  cudaGetErrorString(_e), __FILE__, __LINE__);                                 \
  } while (0)

#define TRY(expr)              \
  do {                         \
    int _r = (expr);           \
    if (_r != TESSA_OK) return _r; \
  } while (0)

constexpr uint64_t kDefaultTimeoutNs = 2000000000ull;  // bounded device waits: 2 s
// A pipeline's drain after a wait gives up waits, under the same limit, for
// its in-flight copies and MMAs (microseconds); the floor keeps the limit far
// above that, the ceiling keeps a stuck kernel from holding the GPU long.
constexpr uint64_t kMinTimeoutNs = 10000000ull;      // 10 ms
constexpr uint64_t kMaxTimeoutNs = 60000000000ull;   // 60 s
constexpr uint64_t kDefaultHostBatchBytes = 128ull << 20;  // codes per batch of the host-buffer pipeline
constexpr uint64_t kMaxHostBatches = 64;

// Grow-only device buffer.
struct DevBuf {
  void* ptr = nullptr;
  size_t bytes = 0;
  int ensure(size_t need) {
    if (need <= bytes) return TESSA_OK;
    if (ptr) cudaFree(ptr);
    ptr = nullptr;
    bytes = 0;
    if (need == 0) return TESSA_OK;
    cudaError_t e = cudaMalloc(&ptr, need);
    if (e != cudaSuccess) {
      ptr = nullptr;
      return fail(e == cudaErrorMemoryAllocation ? TESSA_ERR_OOM : TESSA_ERR_CUDA, "cudaMalloc(%zu): %s", need,
                  cudaGetErrorString(e));
    }
    bytes = need;
    return TESSA_OK;
  }
  void release() {
    if (ptr) cudaFree(ptr);
    ptr = nullptr;
    bytes = 0;
  }
  template <class T>
  T* as() const {
    return reinterpret_cast<T*>(ptr);
  }
};

int map_device_error(uint32_t bits) {
  if (bits == 0) return TESSA_OK;
  if (bits & TESSA_DEVERR_TIMEOUT) return fail(TESSA_ERR_TIMEOUT, "device wait timed out (error bits 0x%x)", bits);
  if (bits & TESSA_DEVERR_BAD_ROW) return fail(TESSA_ERR_BAD_ROW, "row id outside resident rows (0x%x)", bits);
  if (bits & TESSA_DEVERR_NONFINITE) return fail(TESSA_ERR_NONFINITE, "non-finite quantizer input (0x%x)", bits);
  return fail(TESSA_ERR_BAD_TASK, "malformed task descriptor on device (0x%x)", bits);
}

// Host-side leaf plan: (leaf, first row) per 128-row tile plus device copies
// of the leaf layout.  Cached by content so repeated calls on the same layout
// upload nothing.
struct LeafPlan {
  std::vector<uint64_t> starts;
  std::vector<uint64_t> sizes;
  uint64_t leaf_rows = 0;
  uint32_t num_tiles = 0;
  uint32_t num_pairs = 0;  // 256-row tile pairs for the two-CTA leaf kernel
  DevBuf d_starts, d_sizes, d_tiles, d_pairs;
  bool valid = false;

  int build(const uint64_t* h_starts, const uint64_t* h_sizes, uint64_t leaf_count, uint64_t rows, cudaStream_t st) {
    if (valid && leaf_count == starts.size() && rows == leaf_rows &&
        (leaf_count == 0 || (memcmp(h_starts, starts.data(), leaf_count * 8) == 0 &&
                             memcmp(h_sizes, sizes.data(), leaf_count * 8) == 0)))
      return TESSA_OK;
    valid = false;
    std::vector<uint32_t> sz32(leaf_count);
    std::vector<uint2> tiles, pairs;
    for (uint64_t l = 0; l < leaf_count; ++l) {
      if (h_sizes[l] > 0x7fffffffull || h_starts[l] > rows || h_sizes[l] > rows - h_starts[l])
        return fail(TESSA_ERR_INVALID_ARG, "leaf %llu [start %llu, size %llu] outside %llu member rows",
                    (unsigned long long)l, (unsigned long long)h_starts[l], (unsigned long long)h_sizes[l],
                    (unsigned long long)rows);
      if (h_starts[l] + h_sizes[l] > 0x7fffffffull)
        return fail(TESSA_ERR_UNSUPPORTED, "leaf member rows beyond 2^31 are not supported");
      if (h_sizes[l] > kMaxLeafRows)
        return fail(TESSA_ERR_UNSUPPORTED, "leaf %llu has %llu rows; at most %llu are supported", (unsigned long long)l,
                    (unsigned long long)h_sizes[l], (unsigned long long)kMaxLeafRows);
      sz32[l] = (uint32_t)h_sizes[l];
      for (uint64_t r0 = 0; r0 < h_sizes[l]; r0 += 128) tiles.push_back(make_uint2((uint32_t)l, (uint32_t)r0));
      for (uint64_t r0 = 0; r0 < h_sizes[l]; r0 += 256) pairs.push_back(make_uint2((uint32_t)l, (uint32_t)r0));
    }
    if (tiles.size() > 0xffffffffull) return fail(TESSA_ERR_UNSUPPORTED, "too many leaf tiles");
    TRY(d_starts.ensure(leaf_count * 8 + 8));
    TRY(d_sizes.ensure(leaf_count * 4 + 4));
    TRY(d_tiles.ensure(tiles.size() * 8 + 8));
    TRY(d_pairs.ensure(pairs.size() * 8 + 8));
    if (leaf_count) {
      CUDA_TRY(cudaMemcpyAsync(d_starts.ptr, h_starts, leaf_count * 8, cudaMemcpyHostToDevice, st));
      CUDA_TRY(cudaMemcpyAsync(d_sizes.ptr, sz32.data(), leaf_count * 4, cudaMemcpyHostToDevice, st));
    }
    if (!tiles.empty())
      CUDA_TRY(cudaMemcpyAsync(d_tiles.ptr, tiles.data(), tiles.size() * 8, cudaMemcpyHostToDevice, st));
    if (!pairs.empty())
      CUDA_TRY(cudaMemcpyAsync(d_pairs.ptr, pairs.data(), pairs.size() * 8, cudaMemcpyHostToDevice, st));
    CUDA_TRY(cudaStreamSynchronize(st));
    starts.assign(h_starts, h_starts + leaf_count);
    sizes.assign(h_sizes, h_sizes + leaf_count);
    leaf_rows = rows;
    num_tiles = (uint32_t)tiles.size();
    num_pairs = (uint32_t)pairs.size();
    valid = true;
    return TESSA_OK;
  }
  void release() {
    d_starts.release();
    d_sizes.release();
    d_tiles.release();
    d_pairs.release();
    valid = false;
  }
};

// Host-side assignment plan: (task, first row) per 128-row work item plus
// device copies of the task arrays.
struct AssignPlan {
  DevBuf d_moff, d_mcnt, d_loff, d_lcnt, d_rh, d_out, d_work;
  uint32_t num_work = 0;
  uint32_t task_count = 0;
  uint32_t max_leaders = 0;  // largest leader count of any task
  // host copy of the task arrays the device tables were built from: a call
  // with the same tasks (replay sweeps) reuses them without an upload
  std::vector<uint32_t> key32;
  std::vector<uint64_t> key64;
  uint64_t key_member_rows = 0, out_len_cached = 0;
  bool valid = false;

  bool same_tasks(const tessa_assign_args& a) const {
    const size_t n = a.task_count;
    if (!valid || n != task_count || a.member_rows != key_member_rows || key32.size() != 5 * n) return false;
    const uint32_t* cols[5] = {a.task_member_offsets, a.task_member_counts, a.task_leader_offsets,
                               a.task_leader_counts, a.task_rh};
    for (int c = 0; c < 5; ++c)
      if (n && memcmp(cols[c], key32.data() + c * n, n * 4) != 0) return false;
    return n == 0 || memcmp(a.task_output_offsets, key64.data(), n * 8) == 0;
  }

  int build(const tessa_assign_args& a, uint64_t* output_len, cudaStream_t st) {
    if (same_tasks(a)) {
      *output_len = out_len_cached;
      return TESSA_OK;
    }
    valid = false;
    std::vector<uint2> work;
    uint64_t out_len = 0;
    max_leaders = 0;
    for (uint32_t t = 0; t < a.task_count; ++t) {
      max_leaders = std::max(max_leaders, a.task_leader_counts[t]);
      if (a.task_rh[t] == 0 || a.task_rh[t] > TESSA_MAX_RH || a.task_leader_counts[t] < a.task_rh[t])
        return fail(TESSA_ERR_INVALID_ARG, "assignment task %u has invalid r_h=%u for %u leaders", t, a.task_rh[t],
                    a.task_leader_counts[t]);
      if ((uint64_t)a.task_member_offsets[t] + a.task_member_counts[t] > a.member_rows)
        return fail(TESSA_ERR_INVALID_ARG, "assignment task %u members outside the member array", t);
      for (uint32_t r0 = 0; r0 < a.task_member_counts[t]; r0 += 128) work.push_back(make_uint2(t, r0));
      uint64_t end = a.task_output_offsets[t] + (uint64_t)a.task_member_counts[t] * a.task_rh[t];
      if (end > out_len) out_len = end;
    }
    *output_len = out_len;
    size_t n = a.task_count;
    TRY(d_moff.ensure(n * 4 + 4));
    TRY(d_mcnt.ensure(n * 4 + 4));
    TRY(d_loff.ensure(n * 4 + 4));
    TRY(d_lcnt.ensure(n * 4 + 4));
    TRY(d_rh.ensure(n * 4 + 4));
    TRY(d_out.ensure(n * 8 + 8));
    TRY(d_work.ensure(work.size() * 8 + 8));
    if (n) {
      CUDA_TRY(cudaMemcpyAsync(d_moff.ptr, a.task_member_offsets, n * 4, cudaMemcpyHostToDevice, st));
      CUDA_TRY(cudaMemcpyAsync(d_mcnt.ptr, a.task_member_counts, n * 4, cudaMemcpyHostToDevice, st));
      CUDA_TRY(cudaMemcpyAsync(d_loff.ptr, a.task_leader_offsets, n * 4, cudaMemcpyHostToDevice, st));
      CUDA_TRY(cudaMemcpyAsync(d_lcnt.ptr, a.task_leader_counts, n * 4, cudaMemcpyHostToDevice, st));
      CUDA_TRY(cudaMemcpyAsync(d_rh.ptr, a.task_rh, n * 4, cudaMemcpyHostToDevice, st));
      CUDA_TRY(cudaMemcpyAsync(d_out.ptr, a.task_output_offsets, n * 8, cudaMemcpyHostToDevice, st));
    }
    if (!work.empty())
      CUDA_TRY(cudaMemcpyAsync(d_work.ptr, work.data(), work.size() * 8, cudaMemcpyHostToDevice, st));
    CUDA_TRY(cudaStreamSynchronize(st));
    num_work = (uint32_t)work.size();
    task_count = a.task_count;
    key32.resize(5 * n);
    key64.assign(a.task_output_offsets, a.task_output_offsets + n);
    const uint32_t* cols[5] = {a.task_member_offsets, a.task_member_counts, a.task_leader_offsets,
                               a.task_leader_counts, a.task_rh};
    for (int c = 0; c < 5; ++c)
      if (n) memcpy(key32.data() + c * n, cols[c], n * 4);
    key_member_rows = a.member_rows;
    out_len_cached = out_len;
    valid = true;
    return TESSA_OK;
  }
  void release() {
    valid = false;
    d_moff.release();
    d_mcnt.release();
    d_loff.release();
    d_lcnt.release();
    d_rh.release();
    d_out.release();
    d_work.release();
  }
};

}  // namespace

int tessa::set_last_error(int code, const char* message) { return fail(code, "%s", message); }

struct tessa_ctx {
  int device = -1;
  int sm_count = 0;
  cudaStream_t stream = nullptr;
  DevBuf d_err;         // one uint32 error word
  DevBuf gather;        // leaf-ordered codes scratch
  DevBuf fallback;      // exact-fallback row list: count + (leaf, row) entries
  DevBuf dump;          // column-split leaf kernel: per-row zone dump
  LeafPlan leaf_plan;
  AssignPlan assign_plan;
  // staging for host-buffer entry points
  DevBuf h_codes, h_scales, h_norms, h_gids, h_members, h_ids, h_dists, h_x;
  uint64_t timeout_ns = kDefaultTimeoutNs;
  uint64_t last_fallback_rows = 0;  // rows of the last leaf call recomputed by the exact fallback
  // batched host-buffer pipeline: copy-in and copy-out streams, per-batch
  // events and fallback-row counters (created on first use)
  cudaStream_t stream_in = nullptr, stream_out = nullptr;
  std::vector<cudaEvent_t> ev_in, ev_done;
  DevBuf fb_counts;
  uint64_t host_batch_bytes = kDefaultHostBatchBytes;
  // global-D0 staging: leader payload, tie keys, key -> leader, top-k keys,
  // and the host form's extra staging
  DevBuf d0_lcodes, d0_lscales, d0_lnorms, d0_keys, d0_k2l, d0_okeys, d0_dists, d0_lvec, d0_lids, d0_child,
      d0_point;
  DevBuf e_starts, e_sizes;  // leaf layout of an edge-hash call
  cudaEvent_t d0_ev[5] = {nullptr, nullptr, nullptr, nullptr, nullptr};  // phase boundaries of a D0 call
  tessa_d0_profile d0_prof = {};
  SubtreeState* subtree = nullptr;  // subtree partition scratch (created on first use)
  DevBuf g_temp;                    // record grouping: sort and scan scratch
  DevBuf probe;                     // bounded-wait probe: elapsed time
  SubmitRing* ring = nullptr;       // subtree submissions (created on first use)
  uint32_t leaf_kernel = 1;         // 0: column-split kernel on CTA pairs where it applies, 1: one CTA per tile
  uint32_t* async_err = nullptr;    // pinned, mapped error word of the calls that do not wait
  uint32_t* async_err_dev = nullptr;
};

namespace {

int bind(tessa_ctx* ctx) {
  if (!ctx) return fail(TESSA_ERR_INVALID_ARG, "null context");
  CUDA_TRY(cudaSetDevice(ctx->device));
  return TESSA_OK;
}

int read_err(tessa_ctx* ctx, cudaStream_t st, uint32_t* bits) {
  CUDA_TRY(cudaMemcpyAsync(bits, ctx->d_err.ptr, 4, cudaMemcpyDeviceToHost, st));
  CUDA_TRY(cudaStreamSynchronize(st));
  return TESSA_OK;
}

int clear_err(tessa_ctx* ctx, cudaStream_t st) {
  CUDA_TRY(cudaMemsetAsync(ctx->d_err.ptr, 0, 4, st));
  return TESSA_OK;
}

// The error word of the calls that do not wait.
int make_async_word(tessa_ctx* ctx) {
  void *p = nullptr, *d = nullptr;
  CUDA_TRY(cudaHostAlloc(&p, 64, cudaHostAllocMapped));
  memset(p, 0, 64);
  ctx->async_err = static_cast<uint32_t*>(p);
  CUDA_TRY(cudaHostGetDevicePointer(&d, p, 0));
  ctx->async_err_dev = static_cast<uint32_t*>(d);
  return TESSA_OK;
}

// Error bits that kernels of the calls that do not wait have left so far;
// taking them clears the word.  Threads may share the context: each bit is
// taken by one of them.
int take_async_error(tessa_ctx* ctx) {
  if (__atomic_load_n(ctx->async_err, __ATOMIC_RELAXED) == 0) return TESSA_OK;
  const uint32_t bits = __atomic_exchange_n(ctx->async_err, 0u, __ATOMIC_ACQ_REL);
  return bits ? map_device_error(bits) : TESSA_OK;
}

// Blocked scans: the inner loops have no early exit, so they vectorise.
bool members_identity(const uint32_t* m, uint64_t n) {
  for (uint64_t b = 0; b < n; b += 4096) {
    const uint64_t e = n - b < 4096 ? n : b + 4096;
    uint32_t diff = 0;
    for (uint64_t i = b; i < e; ++i) diff |= m[i] ^ (uint32_t)i;
    if (diff) return false;
  }
  return true;
}

// Index of the first entry >= bound, or n.
uint64_t first_at_or_above(const uint32_t* m, uint64_t n, uint64_t bound) {
  if (bound > 0xffffffffull) return n;
  for (uint64_t b = 0; b < n; b += 4096) {
    const uint64_t e = n - b < 4096 ? n : b + 4096;
    uint32_t mx = 0;
    for (uint64_t i = b; i < e; ++i) mx = m[i] > mx ? m[i] : mx;
    if (mx >= bound)
      for (uint64_t i = b; i < e; ++i)
        if (m[i] >= bound) return i;
  }
  return n;
}

// Leaves in ascending start order with disjoint row ranges.
bool leaves_ordered(const uint64_t* starts, const uint64_t* sizes, uint64_t n) {
  uint64_t end = 0;
  for (uint64_t l = 0; l < n; ++l) {
    if (starts[l] < end) return false;
    end = starts[l] + sizes[l];
  }
  return true;
}

int validate_leaf(const tessa_leaf_args* a) {
  if (!a) return fail(TESSA_ERR_INVALID_ARG, "null leaf args");
  if (a->k == 0 || a->k > TESSA_MAX_LEAF_K) return fail(TESSA_ERR_INVALID_ARG, "leaf k=%u outside 1..%d", a->k, TESSA_MAX_LEAF_K);
  if (a->padded_dim == 0 || a->padded_dim % 16 != 0)
    return fail(TESSA_ERR_INVALID_ARG, "padded_dim=%u must be a positive multiple of 16", a->padded_dim);
  if (a->padded_dim > TESSA_MAX_PADDED_DIM || leaf_num_bstages(a->padded_dim) == 0)
    return fail(TESSA_ERR_UNSUPPORTED, "padded_dim=%u above the supported %d", a->padded_dim, TESSA_MAX_PADDED_DIM);
  if (a->resident_rows > 0xffffffffull) return fail(TESSA_ERR_UNSUPPORTED, "more than 2^32 resident rows");
  if (a->leaf_count && (!a->leaf_starts || !a->leaf_sizes))
    return fail(TESSA_ERR_INVALID_ARG, "null leaf layout");
  if (a->leaf_rows && (!a->leaf_members || !a->codes || !a->scales || !a->norms || !a->global_ids || !a->topk_ids ||
                       !a->topk_dists))
    return fail(TESSA_ERR_INVALID_ARG, "null leaf data pointer");
  return TESSA_OK;
}

// Leaf op on device pointers (layout arrays on the host).
// Launches the leaf kernel (and its exact fallback) over tiles
// [tile0, tile0 + ntiles) of the current leaf plan on `st`, without waiting.
// The fallback-row count of this launch lands in *d_fb_count.
// Rows [row0, row0 + nrows) of the leaf-ordered space hold every leaf of the
// launch (the range of the column-split kernel's zone dump).
int leaf_launch_tiles(tessa_ctx* ctx, const tessa_leaf_args* a, const int8_t* lc, uint32_t tile0, uint32_t ntiles,
                      uint32_t* d_fb_count, cudaStream_t st, uint64_t row0, uint64_t nrows) {
  if (ntiles == 0) return TESSA_OK;
  LeafLaunch L;
  uint32_t ring = 0, log_cap = 0;
  if (nrows && leaf_split_plan(a->padded_dim, a->k, &ring, &log_cap)) {
    TRY(ctx->dump.ensure(leaf_dump_bytes(nrows, a->k)));
    L.d_dump = ctx->dump.ptr;
    L.dump_row0 = row0;
    L.dump_rows = nrows;
  }
  L.leaf_codes = lc;
  L.leaf_rows = a->leaf_rows;
  L.padded_dim = a->padded_dim;
  L.scales = a->scales;
  L.norms = a->norms;
  L.global_ids = a->global_ids;
  L.members = a->leaf_members;
  L.d_leaf_starts = ctx->leaf_plan.d_starts.as<uint64_t>();
  L.d_leaf_sizes = ctx->leaf_plan.d_sizes.as<uint32_t>();
  L.d_tiles = ctx->leaf_plan.d_tiles.as<uint2>() + tile0;
  L.num_tiles = ntiles;
  if (ctx->leaf_kernel == 0 && tile0 == 0 && ntiles == ctx->leaf_plan.num_tiles && L.d_dump) {
    L.d_pairs = ctx->leaf_plan.d_pairs.as<uint2>();
    L.num_pairs = ctx->leaf_plan.num_pairs;
  }
  L.k = a->k;
  L.out_ids = a->topk_ids;
  L.out_dists = a->topk_dists;
  L.d_err = ctx->d_err.as<uint32_t>();
  L.d_fb_count = d_fb_count;
  L.d_fb_list = reinterpret_cast<uint2*>(ctx->fallback.as<uint8_t>() + 16);
  L.fb_capacity = (uint32_t)a->leaf_rows;
  L.resident_rows = a->resident_rows;
  L.timeout_ns = ctx->timeout_ns;
  L.sm_count = ctx->sm_count;
  int r = launch_leaf_topk_sq8(L, st);
  if (r != TESSA_OK) return fail(r, "leaf kernel launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  return TESSA_OK;
}

int leaf_device(tessa_ctx* ctx, const tessa_leaf_args* a, cudaStream_t st) {
  TRY(ctx->leaf_plan.build(a->leaf_starts, a->leaf_sizes, a->leaf_count, a->leaf_rows, st));
  if (ctx->leaf_plan.num_tiles == 0) return TESSA_OK;
  const int8_t* lc = a->leaf_ordered_codes;
  if (!lc) {
    TRY(ctx->gather.ensure((size_t)a->leaf_rows * a->padded_dim));
    TRY(launch_gather_rows(a->codes, a->leaf_members, a->leaf_rows, a->padded_dim, a->resident_rows,
                           ctx->gather.as<int8_t>(), ctx->sm_count, st));
    lc = ctx->gather.as<int8_t>();
  }
  TRY(clear_err(ctx, st));
  TRY(ctx->fallback.ensure(16 + (size_t)a->leaf_rows * 8));
  uint32_t* d_fb = ctx->fallback.as<uint32_t>();
  TRY(leaf_launch_tiles(ctx, a, lc, 0, ctx->leaf_plan.num_tiles, d_fb, st, 0, a->leaf_rows));
  uint32_t fb = 0;
  CUDA_TRY(cudaMemcpyAsync(&fb, d_fb, 4, cudaMemcpyDeviceToHost, st));
  uint32_t bits = 0;
  TRY(read_err(ctx, st, &bits));
  ctx->last_fallback_rows = fb;
  return map_device_error(bits);
}

// Host-buffer leaf call when the members are the identity and the leaves are
// ordered and disjoint (the layout a contiguous subtree build produces): the
// member rows split into batches of whole leaves, and batch b's upload (copy
// stream), leaf kernel (compute stream) and download (second copy stream)
// overlap the neighbouring batches', so the call approaches the slowest of
// the three instead of their sum.  Only rows [0, leaf_rows) travel: identity
// members reference no other resident row.
int leaf_host_pipelined(tessa_ctx* ctx, const tessa_leaf_args* a) {
  const uint64_t M = a->leaf_rows, P = a->padded_dim, K = a->k;
  cudaStream_t st = ctx->stream;
  if (!ctx->stream_in) CUDA_TRY(cudaStreamCreateWithFlags(&ctx->stream_in, cudaStreamNonBlocking));
  if (!ctx->stream_out) CUDA_TRY(cudaStreamCreateWithFlags(&ctx->stream_out, cudaStreamNonBlocking));
  TRY(ctx->h_codes.ensure(M * P + 16));
  TRY(ctx->h_scales.ensure(M * 4 + 4));
  TRY(ctx->h_norms.ensure(M * 4 + 4));
  TRY(ctx->h_gids.ensure(M * 4 + 4));
  TRY(ctx->h_members.ensure(M * 4 + 4));
  TRY(ctx->h_ids.ensure(M * K * 4 + 4));
  TRY(ctx->h_dists.ensure(M * K * 4 + 4));
  TRY(ctx->fallback.ensure(16 + M * 8));
  TRY(ctx->leaf_plan.build(a->leaf_starts, a->leaf_sizes, a->leaf_count, M, st));

  struct Batch {
    uint64_t r0, r1;
    uint32_t t0, nt;
  };
  std::vector<Batch> batches;
  const uint64_t per_batch = ctx->host_batch_bytes / P;
  const uint64_t min_rows = (M + kMaxHostBatches - 1) / kMaxHostBatches;
  const uint64_t target = per_batch > min_rows ? per_batch : (min_rows ? min_rows : 1);
  uint64_t r0 = 0;
  uint32_t t = 0, t0 = 0;
  for (uint64_t l = 0; l < a->leaf_count; ++l) {
    t += (uint32_t)((a->leaf_sizes[l] + 127) / 128);
    const uint64_t end = a->leaf_starts[l] + a->leaf_sizes[l];
    const bool last = l + 1 == a->leaf_count;
    if (last || end - r0 >= target) {
      batches.push_back({r0, last ? M : end, t0, t - t0});
      r0 = end;
      t0 = t;
    }
  }
  const size_t nb = batches.size();
  while (ctx->ev_in.size() < nb) {
    cudaEvent_t e;
    CUDA_TRY(cudaEventCreateWithFlags(&e, cudaEventDisableTiming));
    ctx->ev_in.push_back(e);
  }
  while (ctx->ev_done.size() < nb) {
    cudaEvent_t e;
    CUDA_TRY(cudaEventCreateWithFlags(&e, cudaEventDisableTiming));
    ctx->ev_done.push_back(e);
  }
  TRY(ctx->fb_counts.ensure(nb * 4));
  {
    // size the zone dump for the largest batch before any copy is queued
    uint64_t max_rows = 0;
    for (const Batch& B : batches) max_rows = B.r1 - B.r0 > max_rows ? B.r1 - B.r0 : max_rows;
    uint32_t ring = 0, log_cap = 0;
    if (max_rows && leaf_split_plan((uint32_t)P, (uint32_t)K, &ring, &log_cap))
      TRY(ctx->dump.ensure(leaf_dump_bytes(max_rows, (uint32_t)K)));
  }

  tessa_leaf_args d = *a;
  d.codes = ctx->h_codes.as<int8_t>();
  d.scales = ctx->h_scales.as<float>();
  d.norms = ctx->h_norms.as<float>();
  d.global_ids = ctx->h_gids.as<uint32_t>();
  d.leaf_members = ctx->h_members.as<uint32_t>();
  d.topk_ids = ctx->h_ids.as<uint32_t>();
  d.topk_dists = ctx->h_dists.as<float>();
  d.leaf_ordered_codes = d.codes;
  d.resident_rows = M;

  auto issue = [&]() -> int {
    TRY(clear_err(ctx, st));
    CUDA_TRY(cudaMemsetAsync(ctx->fb_counts.ptr, 0, nb * 4, st));
    for (size_t b = 0; b < nb; ++b) {
      const Batch& B = batches[b];
      const uint64_t n = B.r1 - B.r0;
      cudaStream_t si = ctx->stream_in, so = ctx->stream_out;
      CUDA_TRY(cudaMemcpyAsync(ctx->h_codes.as<int8_t>() + B.r0 * P, a->codes + B.r0 * P, n * P,
                               cudaMemcpyHostToDevice, si));
      CUDA_TRY(cudaMemcpyAsync(ctx->h_scales.as<float>() + B.r0, a->scales + B.r0, n * 4, cudaMemcpyHostToDevice, si));
      CUDA_TRY(cudaMemcpyAsync(ctx->h_norms.as<float>() + B.r0, a->norms + B.r0, n * 4, cudaMemcpyHostToDevice, si));
      CUDA_TRY(cudaMemcpyAsync(ctx->h_gids.as<uint32_t>() + B.r0, a->global_ids + B.r0, n * 4,
                               cudaMemcpyHostToDevice, si));
      CUDA_TRY(cudaMemcpyAsync(ctx->h_members.as<uint32_t>() + B.r0, a->leaf_members + B.r0, n * 4,
                               cudaMemcpyHostToDevice, si));
      CUDA_TRY(cudaEventRecord(ctx->ev_in[b], si));
      CUDA_TRY(cudaStreamWaitEvent(st, ctx->ev_in[b], 0));
      TRY(leaf_launch_tiles(ctx, &d, d.codes, B.t0, B.nt, ctx->fb_counts.as<uint32_t>() + b, st, B.r0, B.r1 - B.r0));
      CUDA_TRY(cudaEventRecord(ctx->ev_done[b], st));
      CUDA_TRY(cudaStreamWaitEvent(so, ctx->ev_done[b], 0));
      CUDA_TRY(cudaMemcpyAsync(a->topk_ids + B.r0 * K, ctx->h_ids.as<uint32_t>() + B.r0 * K, n * K * 4,
                               cudaMemcpyDeviceToHost, so));
      CUDA_TRY(cudaMemcpyAsync(a->topk_dists + B.r0 * K, ctx->h_dists.as<float>() + B.r0 * K, n * K * 4,
                               cudaMemcpyDeviceToHost, so));
    }
    return TESSA_OK;
  };
  const int r = issue();
  // drain every stream before reporting, on success and failure alike
  const cudaError_t e_in = cudaStreamSynchronize(ctx->stream_in);
  const cudaError_t e_st = cudaStreamSynchronize(st);
  const cudaError_t e_out = cudaStreamSynchronize(ctx->stream_out);
  if (r != TESSA_OK) return r;
  for (cudaError_t e : {e_in, e_st, e_out})
    if (e != cudaSuccess) return fail(TESSA_ERR_CUDA, "leaf pipeline: %s", cudaGetErrorString(e));
  std::vector<uint32_t> fb(nb);
  CUDA_TRY(cudaMemcpyAsync(fb.data(), ctx->fb_counts.ptr, nb * 4, cudaMemcpyDeviceToHost, st));
  uint32_t bits = 0;
  TRY(read_err(ctx, st, &bits));
  uint64_t total = 0;
  for (uint32_t c : fb) total += c;
  ctx->last_fallback_rows = total;
  return map_device_error(bits);
}

// ------------------------------------------------------------- global D0

int validate_d0(const tessa_d0_args* a) {
  if (!a) return fail(TESSA_ERR_INVALID_ARG, "null D0 args");
  // P/dco_sq_int8.rs:1932-1960 (messages as the reference's)
  if (a->rows == 0) return fail(TESSA_ERR_INVALID_ARG, "SQ GPU-D0 staging requires at least one input row");
  if (a->dim == 0) return fail(TESSA_ERR_INVALID_ARG, "SQ GPU-D0 staging requires dim > 0");
  if (a->leader_count == 0)
    return fail(TESSA_ERR_INVALID_ARG, "SQ GPU-D0 staging requires at least one global D0 leader");
  if (a->fanout_top == 0 || a->fanout_top > a->leader_count || a->fanout_top > 32)
    return fail(TESSA_ERR_INVALID_ARG,
                "SQ GPU-D0 staging fanout must be in 1..=min(32, leaders), got fanout=%u leaders=%u", a->fanout_top,
                a->leader_count);
  if (!a->raw_vectors || !a->global_ids || !a->leader_ids || !a->codes || !a->scales || !a->norms ||
      !a->child_ids || !a->point_ids)
    return fail(TESSA_ERR_INVALID_ARG, "null D0 data pointer");
  if (!a->leader_codes && !a->leader_vectors)
    return fail(TESSA_ERR_INVALID_ARG, "D0 leaders need leader_vectors or a leader payload");
  if (a->leader_codes && (!a->leader_scales || !a->leader_norms))
    return fail(TESSA_ERR_INVALID_ARG, "D0 leader payload without scales or norms");
  const uint64_t P = ((uint64_t)a->dim + 15) / 16 * 16;
  if (P > TESSA_MAX_PADDED_DIM || leaf_num_bstages((uint32_t)P) == 0)
    return fail(TESSA_ERR_UNSUPPORTED, "padded_dim=%llu above the supported %d", (unsigned long long)P,
                TESSA_MAX_PADDED_DIM);
  if (a->rows > kMaxRectRows) return fail(TESSA_ERR_UNSUPPORTED, "more than %llu D0 rows in one call",
                                          (unsigned long long)kMaxRectRows);
  return TESSA_OK;
}

// Tie keys of the leaders: key[j] = rank of (leader_ids[j], j) in
// lexicographic order.  "key_a < key_b" orders two leaders exactly as their
// ids do and breaks equal ids by index (the earlier leader first, as the
// sequential reading of the reference's stable order does), so the keys are
// distinct and the eps/id rule on keys is the rule on ids.
void d0_tie_keys(const uint32_t* ids, uint32_t n, std::vector<uint32_t>& key, std::vector<uint32_t>& key_to_leader) {
  key_to_leader.resize(n);
  std::iota(key_to_leader.begin(), key_to_leader.end(), 0u);
  std::stable_sort(key_to_leader.begin(), key_to_leader.end(),
                   [ids](uint32_t a, uint32_t b) { return ids[a] < ids[b]; });
  key.resize(n);
  for (uint32_t r = 0; r < n; ++r) key[key_to_leader[r]] = r;
}

// Leader side of a D0 call: tie keys to the device, leaders quantized unless a
// payload is given.  Sets the leader code / scale / norm pointers to use.
int d0_prepare(tessa_ctx* ctx, const tessa_d0_args* a, const uint32_t* h_leader_ids, cudaStream_t st,
               const int8_t** lc, const float** ls, const float** ln) {
  const uint32_t dim = a->dim, L = a->leader_count;
  const uint32_t P = (dim + 15u) / 16u * 16u;
  std::vector<uint32_t> key, k2l;
  d0_tie_keys(h_leader_ids, L, key, k2l);
  TRY(ctx->d0_keys.ensure((size_t)L * 4));
  TRY(ctx->d0_k2l.ensure((size_t)L * 4));
  CUDA_TRY(cudaMemcpyAsync(ctx->d0_keys.ptr, key.data(), (size_t)L * 4, cudaMemcpyHostToDevice, st));
  CUDA_TRY(cudaMemcpyAsync(ctx->d0_k2l.ptr, k2l.data(), (size_t)L * 4, cudaMemcpyHostToDevice, st));
  *lc = a->leader_codes;
  *ls = a->leader_scales;
  *ln = a->leader_norms;
  if (!*lc) {
    TRY(ctx->d0_lcodes.ensure((size_t)L * P));
    TRY(ctx->d0_lscales.ensure((size_t)L * 4));
    TRY(ctx->d0_lnorms.ensure((size_t)L * 4));
    TRY(launch_quantize_sq8(a->leader_vectors, L, dim, P, 8, ctx->d0_lcodes.as<int8_t>(), ctx->d0_lscales.as<float>(),
                            ctx->d0_lnorms.as<float>(), ctx->d_err.as<uint32_t>(), st));
    *lc = ctx->d0_lcodes.as<int8_t>();
    *ls = ctx->d0_lscales.as<float>();
    *ln = ctx->d0_lnorms.as<float>();
  }
  // The pageable key vectors must be consumed before they go out of scope.
  CUDA_TRY(cudaStreamSynchronize(st));
  return TESSA_OK;
}

// Row side of a D0 call over a->rows rows (all pointers of `a` already at the
// batch's first row): quantize, assign (top-fanout keys into okeys / dists),
// fragments.  ev, if given, receives three events: after quantize, after
// assignment, after fragments.  Does not wait.
int d0_rows(tessa_ctx* ctx, const tessa_d0_args* a, const int8_t* lc, const float* ls, const float* ln,
            uint32_t* okeys, float* dists, uint32_t* d_fb_count, cudaStream_t st, cudaEvent_t* ev) {
  const uint64_t rows = a->rows;
  const uint32_t dim = a->dim, L = a->leader_count, f = a->fanout_top;
  const uint32_t P = (dim + 15u) / 16u * 16u;
  TRY(launch_quantize_sq8(a->raw_vectors, rows, dim, P, 8, a->codes, a->scales, a->norms, ctx->d_err.as<uint32_t>(),
                          st));
  if (ev) CUDA_TRY(cudaEventRecord(ev[0], st));
  RectLaunch R;
  R.row_codes = a->codes;
  R.rows = rows;
  R.padded_dim = P;
  R.row_scales = a->scales;
  R.row_norms = a->norms;
  R.col_codes = lc;
  R.cols = L;
  R.col_scales = ls;
  R.col_norms = ln;
  R.col_keys = ctx->d0_keys.as<uint32_t>();
  R.k = f;
  R.out_keys = okeys;
  R.out_dists = dists;
  R.d_err = ctx->d_err.as<uint32_t>();
  R.d_fb_count = d_fb_count;
  R.d_fb_list = reinterpret_cast<uint2*>(ctx->fallback.as<uint8_t>() + 16);
  R.fb_capacity = (uint32_t)(rows < 0xffffffffull ? rows : 0xffffffffull);
  R.timeout_ns = ctx->timeout_ns;
  R.sm_count = ctx->sm_count;
  int r = launch_rect_topk_sq8(R, st);
  if (r != TESSA_OK) return fail(r, "D0 assignment launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  if (ev) CUDA_TRY(cudaEventRecord(ev[1], st));
  r = launch_d0_fragments(okeys, ctx->d0_k2l.as<uint32_t>(), a->global_ids, rows, f, L, a->child_ids, a->point_ids,
                          ctx->d_err.as<uint32_t>(), ctx->sm_count, st);
  if (r != TESSA_OK) return fail(r, "D0 fragment launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  if (ev) CUDA_TRY(cudaEventRecord(ev[2], st));
  return TESSA_OK;
}

int d0_status(uint32_t bits) {
  if (bits & TESSA_DEVERR_NONFINITE)
    return fail(TESSA_ERR_NONFINITE, "SQ GPU-D0 staging: non-finite input or distance (0x%x)", bits);
  return map_device_error(bits);
}

// Device-pointer D0 staging; h_leader_ids is a host copy of the leader ids.
int d0_device(tessa_ctx* ctx, const tessa_d0_args* a, const uint32_t* h_leader_ids, cudaStream_t st) {
  const uint64_t rows = a->rows;
  const uint32_t L = a->leader_count, f = a->fanout_top;
  TRY(ctx->d0_okeys.ensure(rows * f * 4));
  TRY(ctx->fallback.ensure(16 + rows * 8));
  if (!a->dists) TRY(ctx->d0_dists.ensure(rows * f * 4));
  for (cudaEvent_t& e : ctx->d0_ev)
    if (!e) CUDA_TRY(cudaEventCreate(&e));
  TRY(clear_err(ctx, st));
  CUDA_TRY(cudaEventRecord(ctx->d0_ev[0], st));
  const int8_t* lc;
  const float* ls;
  const float* ln;
  TRY(d0_prepare(ctx, a, h_leader_ids, st, &lc, &ls, &ln));
  CUDA_TRY(cudaEventRecord(ctx->d0_ev[1], st));
  uint32_t* d_fb = ctx->fallback.as<uint32_t>();
  TRY(d0_rows(ctx, a, lc, ls, ln, ctx->d0_okeys.as<uint32_t>(), a->dists ? a->dists : ctx->d0_dists.as<float>(),
              d_fb, st, &ctx->d0_ev[2]));
  uint32_t fb = 0;
  CUDA_TRY(cudaMemcpyAsync(&fb, d_fb, 4, cudaMemcpyDeviceToHost, st));
  uint32_t bits = 0;
  TRY(read_err(ctx, st, &bits));
  ctx->last_fallback_rows = fb;
  float ms[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < 4; ++i) CUDA_TRY(cudaEventElapsedTime(&ms[i], ctx->d0_ev[i], ctx->d0_ev[i + 1]));
  tessa_d0_profile& pr = ctx->d0_prof;
  pr.leader_quantize_ms = a->leader_codes ? 0.0 : ms[0];
  pr.quantize_ms = ms[1];
  pr.assign_ms = ms[2];
  pr.fragment_ms = ms[3];
  pr.rows = rows;
  pr.fallback_rows = fb;
  pr.leaders = L;
  pr.fanout = f;
  pr.padded_dim = (a->dim + 15u) / 16u * 16u;
  return d0_status(bits);
}

int assign_device(tessa_ctx* ctx, uint32_t source, const tessa_assign_args* a, cudaStream_t st) {
  if (!a) return fail(TESSA_ERR_INVALID_ARG, "null assignment args");
  if (source != TESSA_ASSIGN_FP32 && source != TESSA_ASSIGN_SQ8)
    return fail(TESSA_ERR_INVALID_ARG, "unknown assignment source %u", source);
  if (source == TESSA_ASSIGN_SQ8 && (a->padded_dim == 0 || a->padded_dim % 16 != 0))
    return fail(TESSA_ERR_INVALID_ARG, "padded_dim=%u must be a positive multiple of 16", a->padded_dim);
  if (source == TESSA_ASSIGN_SQ8 && (reinterpret_cast<uintptr_t>(a->codes) & 15u) != 0u)
    return fail(TESSA_ERR_INVALID_ARG, "SQ8 codes must start on a 16-byte boundary");
  if (a->task_count && (!a->task_member_offsets || !a->task_member_counts || !a->task_leader_offsets ||
                        !a->task_leader_counts || !a->task_rh || !a->task_output_offsets))
    return fail(TESSA_ERR_INVALID_ARG, "null task array");
  uint64_t out_len = 0;
  TRY(ctx->assign_plan.build(*a, &out_len, st));
  if (ctx->assign_plan.num_work == 0) return TESSA_OK;
  TRY(clear_err(ctx, st));
  assign::Params p;
  p.x = a->x;
  p.raw_norms = a->raw_norms;
  p.codes = a->codes;
  p.scales = a->scales;
  p.sq8_norms = a->sq8_norms;
  p.global_ids = a->global_ids;
  p.resident_rows = a->resident_rows;
  p.dim = a->dim;
  p.padded_dim = a->padded_dim;
  p.members = a->members;
  p.leaders = a->leaders;
  p.t_moff = ctx->assign_plan.d_moff.as<uint32_t>();
  p.t_mcnt = ctx->assign_plan.d_mcnt.as<uint32_t>();
  p.t_loff = ctx->assign_plan.d_loff.as<uint32_t>();
  p.t_lcnt = ctx->assign_plan.d_lcnt.as<uint32_t>();
  p.t_rh = ctx->assign_plan.d_rh.as<uint32_t>();
  p.t_out = ctx->assign_plan.d_out.as<uint64_t>();
  p.work = ctx->assign_plan.d_work.as<uint2>();
  p.num_work = ctx->assign_plan.num_work;
  p.fused = 1u;
  p.out_ids = a->out_ids;
  p.out_dists = a->out_dists;
  p.err_word = ctx->d_err.as<uint32_t>();
  p.timeout_ns = ctx->timeout_ns;
  TRY(launch_assign(p, source == TESSA_ASSIGN_SQ8, ctx->assign_plan.max_leaders, ctx->sm_count, st));
  uint32_t bits = 0;
  TRY(read_err(ctx, st, &bits));
  return map_device_error(bits);
}

}  // namespace

int tessa::ctx_sm_count(const tessa_ctx* ctx) { return ctx->sm_count; }

int tessa::async_begin(tessa_ctx* ctx, AsyncCtx* out) {
  CUDA_TRY((cudaError_t)out->scope.enter(ctx->device));
  TRY(take_async_error(ctx));
  out->device = ctx->device;
  out->sm_count = ctx->sm_count;
  out->timeout_ns = ctx->timeout_ns;
  out->err = ctx->async_err_dev;
  return TESSA_OK;
}

extern "C" {

int tessa_async_status(tessa_ctx* ctx, void* stream) {
  if (!ctx) return fail(TESSA_ERR_INVALID_ARG, "null context");
  DeviceScope<CudaDevices> scope;
  CUDA_TRY((cudaError_t)scope.enter(ctx->device));
  CUDA_TRY(cudaStreamSynchronize((cudaStream_t)stream));
  return take_async_error(ctx);
}

int tessa_abi_version(void) { return TESSA_ABI_VERSION; }

const char* tessa_strerror(int code) {
  switch (code) {
    case TESSA_OK: return "ok";
    case TESSA_ERR_INVALID_ARG: return "invalid argument";
    case TESSA_ERR_CUDA: return "CUDA error";
    case TESSA_ERR_OOM: return "out of memory";
    case TESSA_ERR_TIMEOUT: return "device wait timed out";
    case TESSA_ERR_BAD_ROW: return "row id outside resident rows";
    case TESSA_ERR_UNSUPPORTED: return "unsupported shape or mode";
    case TESSA_ERR_NONFINITE: return "non-finite input";
    case TESSA_ERR_NO_DEVICE: return "no usable sm_100 device";
    case TESSA_ERR_BAD_TASK: return "malformed task descriptor";
    case TESSA_ERR_PARTITION: return "subtree partition cannot finish";
    case TESSA_ERR_AGAIN: return "not now (no free slot, or still running)";
    default: return "unknown error";
  }
}

const char* tessa_last_error_message(void) { return g_last_error.c_str(); }

int tessa_create(int device, tessa_ctx** out) {
  if (!out) return fail(TESSA_ERR_INVALID_ARG, "null output pointer");
  *out = nullptr;
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) return fail(TESSA_ERR_NO_DEVICE, "no CUDA device");
  if (device < 0 || device >= n) return fail(TESSA_ERR_INVALID_ARG, "device %d outside 0..%d", device, n - 1);
  cudaDeviceProp prop;
  CUDA_TRY(cudaGetDeviceProperties(&prop, device));
  if (prop.major != 10)
    return fail(TESSA_ERR_NO_DEVICE, "device %d is sm_%d%d; this library is built for sm_100a", device, prop.major,
                prop.minor);
  tessa_ctx* ctx = new (std::nothrow) tessa_ctx();
  if (!ctx) return fail(TESSA_ERR_OOM, "context allocation failed");
  ctx->device = device;
  ctx->sm_count = prop.multiProcessorCount;
  int r = bind(ctx);
  if (r == TESSA_OK) {
    if (cudaStreamCreateWithFlags(&ctx->stream, cudaStreamNonBlocking) != cudaSuccess) r = fail(TESSA_ERR_CUDA, "stream create failed");
  }
  if (r == TESSA_OK) r = ctx->d_err.ensure(4);
  if (r == TESSA_OK) r = make_async_word(ctx);
  if (r != TESSA_OK) {
    tessa_destroy(ctx);
    return r;
  }
  *out = ctx;
  return TESSA_OK;
}

void tessa_destroy(tessa_ctx* ctx) {
  if (!ctx) return;
  DeviceScope<CudaDevices> scope;
  scope.enter(ctx->device);
  submit_ring_destroy(ctx->ring);  // waits for queued submissions
  ctx->ring = nullptr;
  if (ctx->stream) cudaStreamSynchronize(ctx->stream);
  ctx->d_err.release();
  ctx->gather.release();
  ctx->fallback.release();
  ctx->dump.release();
  ctx->leaf_plan.release();
  ctx->assign_plan.release();
  DevBuf* bufs[] = {&ctx->h_codes, &ctx->h_scales, &ctx->h_norms, &ctx->h_gids, &ctx->h_members,
                    &ctx->h_ids, &ctx->h_dists, &ctx->h_x, &ctx->fb_counts, &ctx->d0_lcodes,
                    &ctx->d0_lscales, &ctx->d0_lnorms, &ctx->d0_keys, &ctx->d0_k2l, &ctx->d0_okeys,
                    &ctx->d0_dists, &ctx->d0_lvec, &ctx->d0_lids, &ctx->d0_child, &ctx->d0_point,
                    &ctx->e_starts, &ctx->e_sizes};
  for (DevBuf* b : bufs) b->release();
  subtree_state_free(ctx->subtree);
  ctx->subtree = nullptr;
  ctx->g_temp.release();
  ctx->probe.release();
  for (cudaStream_t s : {ctx->stream_in, ctx->stream_out})
    if (s) {
      cudaStreamSynchronize(s);
      cudaStreamDestroy(s);
    }
  if (ctx->async_err) {
    cudaDeviceSynchronize();  // kernels in flight may still write the word
    cudaFreeHost(ctx->async_err);
  }
  for (cudaEvent_t e : ctx->d0_ev)
    if (e) cudaEventDestroy(e);
  for (cudaEvent_t e : ctx->ev_in) cudaEventDestroy(e);
  for (cudaEvent_t e : ctx->ev_done) cudaEventDestroy(e);
  if (ctx->stream) cudaStreamDestroy(ctx->stream);
  delete ctx;
}

int tessa_ctx_device(const tessa_ctx* ctx) { return ctx ? ctx->device : -1; }

int tessa_ctx_device_bytes(const tessa_ctx* ctx, uint64_t* bytes) {
  if (!ctx || !bytes) return fail(TESSA_ERR_INVALID_ARG, "null argument");
  const DevBuf* bufs[] = {&ctx->d_err, &ctx->gather, &ctx->fallback, &ctx->dump, &ctx->leaf_plan.d_starts,
                          &ctx->leaf_plan.d_sizes, &ctx->leaf_plan.d_tiles, &ctx->assign_plan.d_moff,
                          &ctx->assign_plan.d_mcnt, &ctx->assign_plan.d_loff, &ctx->assign_plan.d_lcnt,
                          &ctx->assign_plan.d_rh, &ctx->assign_plan.d_out, &ctx->assign_plan.d_work, &ctx->h_codes,
                          &ctx->h_scales, &ctx->h_norms, &ctx->h_gids, &ctx->h_members, &ctx->h_ids, &ctx->h_dists,
                          &ctx->h_x, &ctx->fb_counts, &ctx->d0_lcodes, &ctx->d0_lscales, &ctx->d0_lnorms,
                          &ctx->d0_keys, &ctx->d0_k2l, &ctx->d0_okeys, &ctx->d0_dists, &ctx->d0_lvec, &ctx->d0_lids,
                          &ctx->d0_child, &ctx->d0_point, &ctx->e_starts, &ctx->e_sizes};
  uint64_t n = 0;
  for (const DevBuf* b : bufs) n += b->bytes;
  *bytes = n;
  return TESSA_OK;
}

int tessa_leaf_last_fallback_rows(const tessa_ctx* ctx, uint64_t* rows) {
  if (!ctx || !rows) return fail(TESSA_ERR_INVALID_ARG, "null argument");
  *rows = ctx->last_fallback_rows;
  return TESSA_OK;
}

int tessa_quantize_sq8(tessa_ctx* ctx, const float* x, uint64_t rows, uint32_t dim, uint32_t k_align, uint32_t bits,
                       int8_t* codes, float* scales, float* norms, void* stream) {
  TRY(bind(ctx));
  if (bits < 2 || bits > 8) return fail(TESSA_ERR_INVALID_ARG, "SQ-int8 bits=%u outside 2..8", bits);
  if (dim == 0) return fail(TESSA_ERR_INVALID_ARG, "SQ-int8 quantization requires dim > 0");
  if (k_align == 0) k_align = 1;
  uint64_t padded = ((uint64_t)dim + k_align - 1) / k_align * k_align;
  if (padded > 0xffffffffull) return fail(TESSA_ERR_UNSUPPORTED, "padded_dim=%llu too large", (unsigned long long)padded);
  if (rows && (!x || !codes || !scales || !norms)) return fail(TESSA_ERR_INVALID_ARG, "null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  TRY(clear_err(ctx, st));
  TRY(launch_quantize_sq8(x, rows, dim, (uint32_t)padded, bits, codes, scales, norms, ctx->d_err.as<uint32_t>(), st));
  uint32_t b = 0;
  TRY(read_err(ctx, st, &b));
  return map_device_error(b);
}

int tessa_quantize_sq8_host(tessa_ctx* ctx, const float* x, uint64_t rows, uint32_t dim, uint32_t k_align,
                            uint32_t bits, int8_t* codes, float* scales, float* norms) {
  TRY(bind(ctx));
  if (dim == 0) return fail(TESSA_ERR_INVALID_ARG, "SQ-int8 quantization requires dim > 0");
  uint32_t ka = k_align ? k_align : 1;
  uint64_t padded = ((uint64_t)dim + ka - 1) / ka * ka;
  cudaStream_t st = ctx->stream;
  TRY(ctx->h_x.ensure(rows * dim * 4 + 4));
  TRY(ctx->h_codes.ensure(rows * padded + 16));
  TRY(ctx->h_scales.ensure(rows * 4 + 4));
  TRY(ctx->h_norms.ensure(rows * 4 + 4));
  if (rows) CUDA_TRY(cudaMemcpyAsync(ctx->h_x.ptr, x, rows * dim * 4, cudaMemcpyHostToDevice, st));
  TRY(tessa_quantize_sq8(ctx, ctx->h_x.as<float>(), rows, dim, k_align, bits, ctx->h_codes.as<int8_t>(),
                         ctx->h_scales.as<float>(), ctx->h_norms.as<float>(), st));
  if (rows) {
    CUDA_TRY(cudaMemcpyAsync(codes, ctx->h_codes.ptr, rows * padded, cudaMemcpyDeviceToHost, st));
    CUDA_TRY(cudaMemcpyAsync(scales, ctx->h_scales.ptr, rows * 4, cudaMemcpyDeviceToHost, st));
    CUDA_TRY(cudaMemcpyAsync(norms, ctx->h_norms.ptr, rows * 4, cudaMemcpyDeviceToHost, st));
  }
  CUDA_TRY(cudaStreamSynchronize(st));
  return TESSA_OK;
}

int tessa_leaf_topk_sq8(tessa_ctx* ctx, const tessa_leaf_args* args, void* stream) {
  TRY(bind(ctx));
  TRY(validate_leaf(args));
  return leaf_device(ctx, args, (cudaStream_t)stream);
}

int tessa_set_host_batch_bytes(tessa_ctx* ctx, uint64_t bytes) {
  if (!ctx) return fail(TESSA_ERR_INVALID_ARG, "null context");
  ctx->host_batch_bytes = bytes ? bytes : kDefaultHostBatchBytes;
  return TESSA_OK;
}

int tessa_leaf_topk_sq8_host(tessa_ctx* ctx, const tessa_leaf_args* a) {
  TRY(bind(ctx));
  TRY(validate_leaf(a));
  const uint64_t R = a->resident_rows, M = a->leaf_rows, P = a->padded_dim;
  const bool ident = (M <= R) && members_identity(a->leaf_members, M);
  if (!ident) {
    uint64_t i = first_at_or_above(a->leaf_members, M, R);
    if (i < M)
      return fail(TESSA_ERR_BAD_ROW, "leaf member %llu = %u outside %llu resident rows", (unsigned long long)i,
                  a->leaf_members[i], (unsigned long long)R);
  }
  if (ident && a->leaf_count && leaves_ordered(a->leaf_starts, a->leaf_sizes, a->leaf_count))
    return leaf_host_pipelined(ctx, a);
  cudaStream_t st = ctx->stream;
  TRY(ctx->h_codes.ensure(R * P + 16));
  TRY(ctx->h_scales.ensure(R * 4 + 4));
  TRY(ctx->h_norms.ensure(R * 4 + 4));
  TRY(ctx->h_gids.ensure(R * 4 + 4));
  TRY(ctx->h_members.ensure(M * 4 + 4));
  TRY(ctx->h_ids.ensure(M * a->k * 4 + 4));
  TRY(ctx->h_dists.ensure(M * a->k * 4 + 4));
  if (R) {
    CUDA_TRY(cudaMemcpyAsync(ctx->h_codes.ptr, a->codes, R * P, cudaMemcpyHostToDevice, st));
    CUDA_TRY(cudaMemcpyAsync(ctx->h_scales.ptr, a->scales, R * 4, cudaMemcpyHostToDevice, st));
    CUDA_TRY(cudaMemcpyAsync(ctx->h_norms.ptr, a->norms, R * 4, cudaMemcpyHostToDevice, st));
    CUDA_TRY(cudaMemcpyAsync(ctx->h_gids.ptr, a->global_ids, R * 4, cudaMemcpyHostToDevice, st));
  }
  if (M) CUDA_TRY(cudaMemcpyAsync(ctx->h_members.ptr, a->leaf_members, M * 4, cudaMemcpyHostToDevice, st));
  tessa_leaf_args d = *a;
  d.codes = ctx->h_codes.as<int8_t>();
  d.scales = ctx->h_scales.as<float>();
  d.norms = ctx->h_norms.as<float>();
  d.global_ids = ctx->h_gids.as<uint32_t>();
  d.leaf_members = ctx->h_members.as<uint32_t>();
  d.topk_ids = ctx->h_ids.as<uint32_t>();
  d.topk_dists = ctx->h_dists.as<float>();
  d.leaf_ordered_codes = ident ? d.codes : nullptr;
  TRY(leaf_device(ctx, &d, st));
  if (M) {
    CUDA_TRY(cudaMemcpyAsync(a->topk_ids, ctx->h_ids.ptr, M * a->k * 4, cudaMemcpyDeviceToHost, st));
    CUDA_TRY(cudaMemcpyAsync(a->topk_dists, ctx->h_dists.ptr, M * a->k * 4, cudaMemcpyDeviceToHost, st));
  }
  CUDA_TRY(cudaStreamSynchronize(st));
  return TESSA_OK;
}

int tessa_d0_last_profile(const tessa_ctx* ctx, tessa_d0_profile* out) {
  if (!ctx || !out) return fail(TESSA_ERR_INVALID_ARG, "null argument");
  *out = ctx->d0_prof;
  return TESSA_OK;
}

int tessa_quantize_sq8_assign_d0(tessa_ctx* ctx, const tessa_d0_args* a, void* stream) {
  TRY(bind(ctx));
  TRY(validate_d0(a));
  cudaStream_t st = (cudaStream_t)stream;
  cudaPointerAttributes attr;
  CUDA_TRY(cudaPointerGetAttributes(&attr, a->leader_ids));
  if (attr.type != cudaMemoryTypeDevice) return d0_device(ctx, a, a->leader_ids, st);
  std::vector<uint32_t> ids(a->leader_count);
  CUDA_TRY(cudaMemcpyAsync(ids.data(), a->leader_ids, ids.size() * 4, cudaMemcpyDeviceToHost, st));
  CUDA_TRY(cudaStreamSynchronize(st));
  return d0_device(ctx, a, ids.data(), st);
}

// Host-buffer D0 staging.  Leaders are prepared once; the rows then go in
// batches of about host_batch_bytes of f32 whose upload (copy stream), device
// work (compute stream) and download (second copy stream) overlap those of the
// neighbouring batches, ordered by events.
int tessa_quantize_sq8_assign_d0_host(tessa_ctx* ctx, const tessa_d0_args* a) {
  TRY(bind(ctx));
  TRY(validate_d0(a));
  cudaStream_t st = ctx->stream;
  const uint64_t rows = a->rows, L = a->leader_count, f = a->fanout_top, dim = a->dim;
  const uint64_t P = (dim + 15) / 16 * 16;
  if (!ctx->stream_in) CUDA_TRY(cudaStreamCreateWithFlags(&ctx->stream_in, cudaStreamNonBlocking));
  if (!ctx->stream_out) CUDA_TRY(cudaStreamCreateWithFlags(&ctx->stream_out, cudaStreamNonBlocking));
  TRY(ctx->h_x.ensure(rows * dim * 4));
  TRY(ctx->h_gids.ensure(rows * 4));
  TRY(ctx->h_codes.ensure(rows * P));
  TRY(ctx->h_scales.ensure(rows * 4));
  TRY(ctx->h_norms.ensure(rows * 4));
  TRY(ctx->d0_child.ensure(rows * f * 4));
  TRY(ctx->d0_point.ensure(rows * f * 4));
  TRY(ctx->h_dists.ensure(rows * f * 4));
  TRY(ctx->d0_okeys.ensure(rows * f * 4));
  TRY(ctx->fallback.ensure(16 + rows * 8));
  tessa_d0_args d = *a;
  if (a->leader_codes) {
    TRY(ctx->d0_lcodes.ensure(L * P));
    TRY(ctx->d0_lscales.ensure(L * 4));
    TRY(ctx->d0_lnorms.ensure(L * 4));
    CUDA_TRY(cudaMemcpyAsync(ctx->d0_lcodes.ptr, a->leader_codes, L * P, cudaMemcpyHostToDevice, st));
    CUDA_TRY(cudaMemcpyAsync(ctx->d0_lscales.ptr, a->leader_scales, L * 4, cudaMemcpyHostToDevice, st));
    CUDA_TRY(cudaMemcpyAsync(ctx->d0_lnorms.ptr, a->leader_norms, L * 4, cudaMemcpyHostToDevice, st));
    d.leader_codes = ctx->d0_lcodes.as<int8_t>();
    d.leader_scales = ctx->d0_lscales.as<float>();
    d.leader_norms = ctx->d0_lnorms.as<float>();
    d.leader_vectors = nullptr;
  } else {
    TRY(ctx->d0_lvec.ensure(L * dim * 4));
    CUDA_TRY(cudaMemcpyAsync(ctx->d0_lvec.ptr, a->leader_vectors, L * dim * 4, cudaMemcpyHostToDevice, st));
    d.leader_vectors = ctx->d0_lvec.as<float>();
  }
  TRY(clear_err(ctx, st));
  const int8_t* lc;
  const float* ls;
  const float* ln;
  TRY(d0_prepare(ctx, &d, a->leader_ids, st, &lc, &ls, &ln));

  const uint64_t per_batch = ctx->host_batch_bytes / (dim * 4);
  const uint64_t min_rows = (rows + kMaxHostBatches - 1) / kMaxHostBatches;
  const uint64_t brows = per_batch > min_rows ? per_batch : (min_rows ? min_rows : 1);
  const size_t nb = (size_t)((rows + brows - 1) / brows);
  while (ctx->ev_in.size() < nb) {
    cudaEvent_t e;
    CUDA_TRY(cudaEventCreateWithFlags(&e, cudaEventDisableTiming));
    ctx->ev_in.push_back(e);
  }
  while (ctx->ev_done.size() < nb) {
    cudaEvent_t e;
    CUDA_TRY(cudaEventCreateWithFlags(&e, cudaEventDisableTiming));
    ctx->ev_done.push_back(e);
  }
  TRY(ctx->fb_counts.ensure(nb * 4));
  CUDA_TRY(cudaMemsetAsync(ctx->fb_counts.ptr, 0, nb * 4, st));

  auto issue = [&]() -> int {
    for (size_t b = 0; b < nb; ++b) {
      const uint64_t r0 = b * brows, n = rows - r0 < brows ? rows - r0 : brows;
      cudaStream_t si = ctx->stream_in, so = ctx->stream_out;
      tessa_d0_args v = d;
      v.rows = n;
      v.raw_vectors = ctx->h_x.as<float>() + r0 * dim;
      v.global_ids = ctx->h_gids.as<uint32_t>() + r0;
      v.codes = ctx->h_codes.as<int8_t>() + r0 * P;
      v.scales = ctx->h_scales.as<float>() + r0;
      v.norms = ctx->h_norms.as<float>() + r0;
      v.child_ids = ctx->d0_child.as<uint32_t>() + r0 * f;
      v.point_ids = ctx->d0_point.as<uint32_t>() + r0 * f;
      v.dists = ctx->h_dists.as<float>() + r0 * f;
      CUDA_TRY(cudaMemcpyAsync(const_cast<float*>(v.raw_vectors), a->raw_vectors + r0 * dim, n * dim * 4,
                               cudaMemcpyHostToDevice, si));
      CUDA_TRY(cudaMemcpyAsync(const_cast<uint32_t*>(v.global_ids), a->global_ids + r0, n * 4,
                               cudaMemcpyHostToDevice, si));
      CUDA_TRY(cudaEventRecord(ctx->ev_in[b], si));
      CUDA_TRY(cudaStreamWaitEvent(st, ctx->ev_in[b], 0));
      TRY(d0_rows(ctx, &v, lc, ls, ln, ctx->d0_okeys.as<uint32_t>() + r0 * f, v.dists,
                  ctx->fb_counts.as<uint32_t>() + b, st, nullptr));
      CUDA_TRY(cudaEventRecord(ctx->ev_done[b], st));
      CUDA_TRY(cudaStreamWaitEvent(so, ctx->ev_done[b], 0));
      CUDA_TRY(cudaMemcpyAsync(a->codes + r0 * P, v.codes, n * P, cudaMemcpyDeviceToHost, so));
      CUDA_TRY(cudaMemcpyAsync(a->scales + r0, v.scales, n * 4, cudaMemcpyDeviceToHost, so));
      CUDA_TRY(cudaMemcpyAsync(a->norms + r0, v.norms, n * 4, cudaMemcpyDeviceToHost, so));
      CUDA_TRY(cudaMemcpyAsync(a->child_ids + r0 * f, v.child_ids, n * f * 4, cudaMemcpyDeviceToHost, so));
      CUDA_TRY(cudaMemcpyAsync(a->point_ids + r0 * f, v.point_ids, n * f * 4, cudaMemcpyDeviceToHost, so));
      if (a->dists) CUDA_TRY(cudaMemcpyAsync(a->dists + r0 * f, v.dists, n * f * 4, cudaMemcpyDeviceToHost, so));
    }
    return TESSA_OK;
  };
  const int r = issue();
  const cudaError_t e_in = cudaStreamSynchronize(ctx->stream_in);
  const cudaError_t e_st = cudaStreamSynchronize(st);
  const cudaError_t e_out = cudaStreamSynchronize(ctx->stream_out);
  if (r != TESSA_OK) return r;
  for (cudaError_t e : {e_in, e_st, e_out})
    if (e != cudaSuccess) return fail(TESSA_ERR_CUDA, "D0 pipeline: %s", cudaGetErrorString(e));
  std::vector<uint32_t> fb(nb);
  CUDA_TRY(cudaMemcpyAsync(fb.data(), ctx->fb_counts.ptr, nb * 4, cudaMemcpyDeviceToHost, st));
  uint32_t bits = 0;
  TRY(read_err(ctx, st, &bits));
  uint64_t total = 0;
  for (uint32_t c : fb) total += c;
  ctx->last_fallback_rows = total;
  tessa_d0_profile& pr = ctx->d0_prof;
  pr = tessa_d0_profile{};  // phases overlap across batches: no per-phase times
  pr.rows = rows;
  pr.fallback_rows = total;
  pr.leaders = (uint32_t)L;
  pr.fanout = (uint32_t)f;
  pr.padded_dim = (uint32_t)P;
  return d0_status(bits);
}

int tessa_sketch_rows(tessa_ctx* ctx, const float* x, uint64_t rows, uint32_t dim, const float* hyperplanes,
                      uint32_t m, float* sketches, void* stream) {
  TRY(bind(ctx));
  if (m == 0 || m > TESSA_MAX_HASH_BITS)
    return fail(TESSA_ERR_INVALID_ARG, "sketch width m=%u outside 1..%d", m, TESSA_MAX_HASH_BITS);
  if (dim == 0) return fail(TESSA_ERR_INVALID_ARG, "sketches require dim > 0");
  if (rows && (!x || !hyperplanes || !sketches)) return fail(TESSA_ERR_INVALID_ARG, "null pointer");
  const int r = launch_sketch_rows(x, rows, dim, hyperplanes, m, sketches, ctx->sm_count, (cudaStream_t)stream);
  if (r != TESSA_OK) return fail(r, "sketch launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  return TESSA_OK;
}

int tessa_edge_hashes(tessa_ctx* ctx, const uint32_t* point_ids, const uint32_t* topk_ids, uint64_t rows, uint32_t k,
                      const uint64_t* leaf_starts, const uint64_t* leaf_sizes, uint64_t leaf_count,
                      const float* sketches, uint64_t sketch_rows, uint32_t sketch_width, uint32_t m_bits,
                      uint16_t* hash_fwd, uint16_t* hash_rev, void* stream) {
  TRY(bind(ctx));
  if (m_bits == 0 || m_bits > TESSA_MAX_HASH_BITS || m_bits > sketch_width)
    return fail(TESSA_ERR_INVALID_ARG, "m_bits=%u outside 1..min(%d, sketch width %u)", m_bits, TESSA_MAX_HASH_BITS,
                sketch_width);
  if (rows && k && (!point_ids || !topk_ids || !sketches || !hash_fwd || !hash_rev))
    return fail(TESSA_ERR_INVALID_ARG, "null pointer");
  if (leaf_count && (!leaf_starts || !leaf_sizes)) return fail(TESSA_ERR_INVALID_ARG, "null leaf layout");
  uint64_t max_rows = 0;
  for (uint64_t l = 0; l < leaf_count; ++l) {
    if (leaf_starts[l] > rows || leaf_sizes[l] > rows - leaf_starts[l])
      return fail(TESSA_ERR_INVALID_ARG, "leaf %llu [start %llu, size %llu] outside %llu rows", (unsigned long long)l,
                  (unsigned long long)leaf_starts[l], (unsigned long long)leaf_sizes[l], (unsigned long long)rows);
    max_rows = std::max(max_rows, leaf_sizes[l]);
  }
  cudaStream_t st = (cudaStream_t)stream;
  TRY(clear_err(ctx, st));
  uint32_t log2cap = 0;
  const bool staged = leaf_count > 0 && leaf_count <= 0xffffffffull && max_rows <= 0xffffffull &&
                      max_rows * k <= 0xffffffffull &&  // slot indices within a leaf are 32-bit
                      leaf_edge_smem((uint32_t)max_rows, m_bits, &log2cap) <= kLeafEdgeSmemMax;
  int r;
  if (staged) {
    std::vector<uint32_t> sz32(leaf_count);
    for (uint64_t l = 0; l < leaf_count; ++l) sz32[l] = (uint32_t)leaf_sizes[l];
    TRY(ctx->e_starts.ensure(leaf_count * 8));
    TRY(ctx->e_sizes.ensure(leaf_count * 4));
    CUDA_TRY(cudaMemcpyAsync(ctx->e_starts.ptr, leaf_starts, leaf_count * 8, cudaMemcpyHostToDevice, st));
    CUDA_TRY(cudaMemcpyAsync(ctx->e_sizes.ptr, sz32.data(), leaf_count * 4, cudaMemcpyHostToDevice, st));
    r = launch_leaf_edge_hashes(point_ids, topk_ids, ctx->e_starts.as<uint64_t>(), ctx->e_sizes.as<uint32_t>(),
                                (uint32_t)leaf_count, (uint32_t)max_rows, k, sketches, sketch_rows, sketch_width,
                                m_bits, hash_fwd, hash_rev, ctx->d_err.as<uint32_t>(), ctx->sm_count, st);
  } else {
    r = launch_edge_hashes(point_ids, topk_ids, rows, k, sketches, sketch_rows, sketch_width, m_bits, hash_fwd,
                           hash_rev, ctx->d_err.as<uint32_t>(), ctx->sm_count, st);
  }
  if (r != TESSA_OK) return fail(r, "edge hash launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  uint32_t bits = 0;
  TRY(read_err(ctx, st, &bits));  // synchronises: the pageable size vector outlives the copy
  if (bits & TESSA_DEVERR_BAD_ROW) return fail(TESSA_ERR_BAD_ROW, "leaf slot or row id outside the sketch store");
  if (bits & TESSA_DEVERR_BAD_TASK)
    return fail(TESSA_ERR_BAD_TASK, "a leaf slot references a point outside its leaf");
  return map_device_error(bits);
}

int tessa_expand_edges(const uint32_t* point_ids, const uint32_t* topk_ids, const float* topk_dists,
                       const uint16_t* hash_fwd, const uint16_t* hash_rev, uint64_t rows, uint32_t k, uint32_t threads,
                       uint32_t* edge_p, uint32_t* edge_c, uint16_t* edge_hash, float* edge_dist, uint64_t capacity,
                       uint64_t* edge_count) {
  if (!edge_count) return fail(TESSA_ERR_INVALID_ARG, "null edge_count");
  *edge_count = 0;
  if (rows && k && (!point_ids || !topk_ids || !topk_dists || !hash_fwd || !hash_rev))
    return fail(TESSA_ERR_INVALID_ARG, "null input pointer");
  if (edge_p && (!edge_c || !edge_hash || !edge_dist)) return fail(TESSA_ERR_INVALID_ARG, "null output pointer");
  *edge_count = expand_edges_host(point_ids, topk_ids, topk_dists, hash_fwd, hash_rev, rows, k, edge_p, edge_c,
                                  edge_hash, edge_dist, capacity, threads);
  if (edge_p && *edge_count > capacity)
    return fail(TESSA_ERR_INVALID_ARG, "edge capacity %llu below the %llu edges", (unsigned long long)capacity,
                (unsigned long long)*edge_count);
  return TESSA_OK;
}

int tessa_membership_digests(tessa_ctx* ctx, const uint32_t* ids, const uint32_t* global_ids,
                             const uint64_t* leaf_starts, const uint64_t* leaf_sizes, uint64_t leaf_count,
                             uint64_t* out_sum, uint64_t* out_xor, void* stream) {
  TRY(bind(ctx));
  if (leaf_count == 0) return TESSA_OK;
  if (!ids || !leaf_starts || !leaf_sizes || !out_sum || !out_xor) return fail(TESSA_ERR_INVALID_ARG, "null pointer");
  if (leaf_count > 0xffffffffull) return fail(TESSA_ERR_UNSUPPORTED, "more than 2^32 leaves");
  cudaStream_t st = (cudaStream_t)stream;
  TRY(ctx->e_starts.ensure(leaf_count * 8));
  TRY(ctx->e_sizes.ensure(leaf_count * 8));
  CUDA_TRY(cudaMemcpyAsync(ctx->e_starts.ptr, leaf_starts, leaf_count * 8, cudaMemcpyHostToDevice, st));
  CUDA_TRY(cudaMemcpyAsync(ctx->e_sizes.ptr, leaf_sizes, leaf_count * 8, cudaMemcpyHostToDevice, st));
  const int r = launch_membership_digests(ids, global_ids, ctx->e_starts.as<uint64_t>(), ctx->e_sizes.as<uint64_t>(),
                                          (uint32_t)leaf_count, out_sum, out_xor, ctx->sm_count, st);
  if (r != TESSA_OK) return fail(r, "digest launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  CUDA_TRY(cudaStreamSynchronize(st));
  return TESSA_OK;
}

int tessa_graph_search(const float* data, uint64_t n, uint32_t dim, const uint64_t* offsets,
                       const uint32_t* neighbors, uint32_t start, const float* queries, uint64_t nq, uint32_t k,
                       uint32_t l, uint32_t threads, uint32_t* out_ids, uint64_t* comparisons) {
  if (nq == 0) return TESSA_OK;
  if (!data || !offsets || !queries || !out_ids || (offsets[n] && !neighbors))
    return fail(TESSA_ERR_INVALID_ARG, "null pointer");
  if (n == 0 || dim == 0 || k == 0) return fail(TESSA_ERR_INVALID_ARG, "graph search needs n, dim and k > 0");
  if (start >= n) return fail(TESSA_ERR_INVALID_ARG, "start node %u outside %llu points", start, (unsigned long long)n);
  for (uint64_t v = 0; v < n; ++v)
    if (offsets[v] > offsets[v + 1]) return fail(TESSA_ERR_INVALID_ARG, "graph offsets decrease at node %llu",
                                                 (unsigned long long)v);
  const uint64_t c = graph_search_host(data, n, dim, offsets, neighbors, start, queries, nq, k, l, threads, out_ids);
  if (comparisons) *comparisons = c;
  return TESSA_OK;
}

int tessa_assign(tessa_ctx* ctx, uint32_t source, const tessa_assign_args* args, void* stream) {
  TRY(bind(ctx));
  return assign_device(ctx, source, args, (cudaStream_t)stream);
}

}  // extern "C"

// ------------------------------------------------------------ replay session

struct tessa_replay_session {
  tessa_ctx* ctx = nullptr;
  uint32_t dim = 0, padded_dim = 0, leaf_k = 0;
  uint64_t resident_rows = 0, leaf_rows = 0, assign_out_len = 0;
  DevBuf gids, x, raw_norms, codes, scales, sq8_norms, amembers, aleaders, lmembers, aids, adists, lids, ldists;
  bool leaf_identity = false;
  std::vector<uint32_t> t_moff, t_mcnt, t_loff, t_lcnt, t_rh;
  std::vector<uint64_t> t_out, leaf_starts, leaf_sizes;
  uint64_t amember_rows = 0;
  cudaEvent_t ev[6] = {};
};

namespace {

template <class T>
int upload(DevBuf& b, const T* h, uint64_t n, cudaStream_t st) {
  TRY(b.ensure(n * sizeof(T) + 16));
  if (n) CUDA_TRY(cudaMemcpyAsync(b.ptr, h, n * sizeof(T), cudaMemcpyHostToDevice, st));
  return TESSA_OK;
}

bool mode_uses_sq8(uint32_t m) { return m >= TESSA_MODE_A2_SQ8_DP4A_BATCH1; }
bool mode_replays_leaf(uint32_t m) { return m <= TESSA_MODE_A3_SQ8_WMMA_BATCH8; }

}  // namespace

extern "C" {

int tessa_replay_session_create(int device, const tessa_prepared_replay* p, tessa_replay_session** out) {
  if (!out || !p) return fail(TESSA_ERR_INVALID_ARG, "null argument");
  *out = nullptr;
  if (p->resident_rows == 0 || p->task_count == 0 || p->leaf_count == 0)
    return fail(TESSA_ERR_INVALID_ARG, "prepared replay tasks must be non-empty");
  tessa_ctx* ctx = nullptr;
  TRY(tessa_create(device, &ctx));
  tessa_replay_session* s = new (std::nothrow) tessa_replay_session();
  if (!s) {
    tessa_destroy(ctx);
    return fail(TESSA_ERR_OOM, "session allocation failed");
  }
  s->ctx = ctx;
  auto cleanup = [&](int r) {
    tessa_replay_session_destroy(s);
    return r;
  };
  cudaStream_t st = ctx->stream;
  s->dim = p->dim;
  s->padded_dim = p->padded_dim;
  s->leaf_k = p->leaf_k;
  s->resident_rows = p->resident_rows;
  s->leaf_rows = p->leaf_rows;
  s->assign_out_len = p->assignment_output_len;
  s->amember_rows = p->assignment_member_rows;
  int r;
  if ((r = upload(s->gids, p->global_ids, p->resident_rows, st)) ||
      (r = upload(s->x, p->vectors, p->resident_rows * p->dim, st)) ||
      (r = upload(s->raw_norms, p->raw_norms, p->resident_rows, st)) ||
      (r = upload(s->codes, p->sq8_codes, p->resident_rows * p->padded_dim, st)) ||
      (r = upload(s->scales, p->sq8_scales, p->resident_rows, st)) ||
      (r = upload(s->sq8_norms, p->sq8_norms, p->resident_rows, st)) ||
      (r = upload(s->amembers, p->assignment_members, p->assignment_member_rows, st)) ||
      (r = upload(s->aleaders, p->assignment_leaders, p->assignment_leader_rows, st)) ||
      (r = upload(s->lmembers, p->leaf_members, p->leaf_rows, st)))
    return cleanup(r);
  if ((r = s->aids.ensure(p->assignment_output_len * 4 + 4)) || (r = s->adists.ensure(p->assignment_output_len * 4 + 4)) ||
      (r = s->lids.ensure(p->leaf_rows * p->leaf_k * 4 + 4)) || (r = s->ldists.ensure(p->leaf_rows * p->leaf_k * 4 + 4)))
    return cleanup(r);
  for (uint64_t i = 0; i < p->leaf_rows; ++i)
    if (p->leaf_members[i] >= p->resident_rows) return cleanup(fail(TESSA_ERR_BAD_ROW, "leaf member outside resident rows"));
  for (uint64_t i = 0; i < p->assignment_member_rows; ++i)
    if (p->assignment_members[i] >= p->resident_rows) return cleanup(fail(TESSA_ERR_BAD_ROW, "assignment member outside resident rows"));
  for (uint64_t i = 0; i < p->assignment_leader_rows; ++i)
    if (p->assignment_leaders[i] >= p->resident_rows) return cleanup(fail(TESSA_ERR_BAD_ROW, "assignment leader outside resident rows"));
  s->leaf_identity = p->leaf_rows <= p->resident_rows && members_identity(p->leaf_members, p->leaf_rows);
  s->t_moff.assign(p->task_member_offsets, p->task_member_offsets + p->task_count);
  s->t_mcnt.assign(p->task_member_counts, p->task_member_counts + p->task_count);
  s->t_loff.assign(p->task_leader_offsets, p->task_leader_offsets + p->task_count);
  s->t_lcnt.assign(p->task_leader_counts, p->task_leader_counts + p->task_count);
  s->t_rh.assign(p->task_rh, p->task_rh + p->task_count);
  s->t_out.assign(p->task_output_offsets, p->task_output_offsets + p->task_count);
  s->leaf_starts.assign(p->leaf_starts, p->leaf_starts + p->leaf_count);
  s->leaf_sizes.assign(p->leaf_sizes, p->leaf_sizes + p->leaf_count);
  for (auto& e : s->ev)
    if (cudaEventCreate(&e) != cudaSuccess) return cleanup(fail(TESSA_ERR_CUDA, "event create failed"));
  if (cudaStreamSynchronize(st) != cudaSuccess) return cleanup(fail(TESSA_ERR_CUDA, "upload failed"));
  *out = s;
  return TESSA_OK;
}

int tessa_replay_run_mode(tessa_replay_session* s, uint32_t mode, tessa_mode_result* res) {
  if (!s || !res) return fail(TESSA_ERR_INVALID_ARG, "null argument");
  if (mode > TESSA_MODE_SQ8_WMMA_BATCH1) return fail(TESSA_ERR_INVALID_ARG, "unknown replay mode %u", mode);
  if (mode_replays_leaf(mode) && !mode_uses_sq8(mode))
    return fail(TESSA_ERR_UNSUPPORTED,
                "mode %u replays raw FP32/TF32 leaf tasks; only the SQ8 leaf operator is built (use modes 2-5)", mode);
  tessa_ctx* ctx = s->ctx;
  TRY(bind(ctx));
  cudaStream_t st = ctx->stream;
  // clear outputs as run_mode does (CB:34849-34889): ids 0xffffffff, dists FLT_MAX
  std::vector<uint32_t> fill_id(1, 0xffffffffu);
  CUDA_TRY(cudaMemsetAsync(s->aids.ptr, 0xff, s->assign_out_len * 4, st));
  {
    std::vector<float> fmax(s->assign_out_len, 3.402823466e+38F);
    if (!fmax.empty()) CUDA_TRY(cudaMemcpyAsync(s->adists.ptr, fmax.data(), fmax.size() * 4, cudaMemcpyHostToDevice, st));
    CUDA_TRY(cudaStreamSynchronize(st));
  }
  bool leaf = mode_replays_leaf(mode);
  if (leaf) {
    CUDA_TRY(cudaMemsetAsync(s->lids.ptr, 0xff, s->leaf_rows * s->leaf_k * 4, st));
    std::vector<float> fmax(s->leaf_rows * s->leaf_k, 3.402823466e+38F);
    if (!fmax.empty()) CUDA_TRY(cudaMemcpyAsync(s->ldists.ptr, fmax.data(), fmax.size() * 4, cudaMemcpyHostToDevice, st));
    CUDA_TRY(cudaStreamSynchronize(st));
  }
  tessa_assign_args aa;
  memset(&aa, 0, sizeof(aa));
  aa.x = s->x.as<float>();
  aa.raw_norms = s->raw_norms.as<float>();
  aa.codes = s->codes.as<int8_t>();
  aa.scales = s->scales.as<float>();
  aa.sq8_norms = s->sq8_norms.as<float>();
  aa.global_ids = s->gids.as<uint32_t>();
  aa.resident_rows = s->resident_rows;
  aa.dim = s->dim;
  aa.padded_dim = s->padded_dim;
  aa.members = s->amembers.as<uint32_t>();
  aa.leaders = s->aleaders.as<uint32_t>();
  aa.task_member_offsets = s->t_moff.data();
  aa.task_member_counts = s->t_mcnt.data();
  aa.task_leader_offsets = s->t_loff.data();
  aa.task_leader_counts = s->t_lcnt.data();
  aa.task_rh = s->t_rh.data();
  aa.task_output_offsets = s->t_out.data();
  aa.task_count = (uint32_t)s->t_moff.size();
  aa.member_rows = s->amember_rows;
  aa.out_ids = s->aids.as<uint32_t>();
  aa.out_dists = s->adists.as<float>();
  uint64_t err_bits = 0;
  CUDA_TRY(cudaEventRecord(s->ev[0], st));
  CUDA_TRY(cudaEventRecord(s->ev[1], st));
  int r = assign_device(ctx, mode_uses_sq8(mode) ? TESSA_ASSIGN_SQ8 : TESSA_ASSIGN_FP32, &aa, st);
  if (r == TESSA_ERR_TIMEOUT || r == TESSA_ERR_BAD_ROW || r == TESSA_ERR_BAD_TASK) err_bits |= 1;
  TRY(r);
  CUDA_TRY(cudaEventRecord(s->ev[2], st));
  if (leaf) {
    CUDA_TRY(cudaEventRecord(s->ev[3], st));
    tessa_leaf_args la;
    memset(&la, 0, sizeof(la));
    la.codes = s->codes.as<int8_t>();
    la.scales = s->scales.as<float>();
    la.norms = s->sq8_norms.as<float>();
    la.global_ids = s->gids.as<uint32_t>();
    la.resident_rows = s->resident_rows;
    la.padded_dim = s->padded_dim;
    la.k = s->leaf_k;
    la.leaf_members = s->lmembers.as<uint32_t>();
    la.leaf_starts = s->leaf_starts.data();
    la.leaf_sizes = s->leaf_sizes.data();
    la.leaf_count = s->leaf_starts.size();
    la.leaf_rows = s->leaf_rows;
    la.topk_ids = s->lids.as<uint32_t>();
    la.topk_dists = s->ldists.as<float>();
    la.leaf_ordered_codes = s->leaf_identity ? la.codes : nullptr;
    TRY(validate_leaf(&la));
    TRY(leaf_device(ctx, &la, st));
    CUDA_TRY(cudaEventRecord(s->ev[4], st));
  }
  CUDA_TRY(cudaEventRecord(s->ev[5], st));
  CUDA_TRY(cudaStreamSynchronize(st));
  float ms = 0;
  CUDA_TRY(cudaEventElapsedTime(&ms, s->ev[1], s->ev[2]));
  res->assignment_event_ms = ms;
  if (leaf) {
    CUDA_TRY(cudaEventElapsedTime(&ms, s->ev[3], s->ev[4]));
    res->leaf_event_ms = ms;
  } else {
    res->leaf_event_ms = -1.0;
  }
  CUDA_TRY(cudaEventElapsedTime(&ms, s->ev[0], s->ev[5]));
  res->total_event_ms = ms;
  res->device_error_bits = err_bits;
  if (res->assignment_ids && s->assign_out_len)
    CUDA_TRY(cudaMemcpyAsync(res->assignment_ids, s->aids.ptr, s->assign_out_len * 4, cudaMemcpyDeviceToHost, st));
  if (res->assignment_dists && s->assign_out_len)
    CUDA_TRY(cudaMemcpyAsync(res->assignment_dists, s->adists.ptr, s->assign_out_len * 4, cudaMemcpyDeviceToHost, st));
  if (leaf && res->leaf_ids)
    CUDA_TRY(cudaMemcpyAsync(res->leaf_ids, s->lids.ptr, s->leaf_rows * s->leaf_k * 4, cudaMemcpyDeviceToHost, st));
  if (leaf && res->leaf_dists)
    CUDA_TRY(cudaMemcpyAsync(res->leaf_dists, s->ldists.ptr, s->leaf_rows * s->leaf_k * 4, cudaMemcpyDeviceToHost, st));
  CUDA_TRY(cudaStreamSynchronize(st));
  return TESSA_OK;
}

void tessa_replay_session_destroy(tessa_replay_session* s) {
  if (!s) return;
  if (s->ctx) {
    cudaSetDevice(s->ctx->device);
    cudaStreamSynchronize(s->ctx->stream);
  }
  for (auto& e : s->ev)
    if (e) cudaEventDestroy(e);
  DevBuf* bufs[] = {&s->gids, &s->x, &s->raw_norms, &s->codes, &s->scales, &s->sq8_norms, &s->amembers,
                    &s->aleaders, &s->lmembers, &s->aids, &s->adists, &s->lids, &s->ldists};
  for (DevBuf* b : bufs) b->release();
  tessa_destroy(s->ctx);
  delete s;
}

}  // extern "C"

// ------------------------------------------------------ subtree partition

int tessa_subtree_partition(tessa_ctx* ctx, const tessa_subtree_args* a, tessa_subtree_result* result, void* stream) {
  TRY(bind(ctx));
  if (!a || !result) return fail(TESSA_ERR_INVALID_ARG, "null subtree arguments");
  if (a->padded_dim == 0 || a->padded_dim % 16 != 0)
    return fail(TESSA_ERR_INVALID_ARG, "padded_dim=%u must be a positive multiple of 16", a->padded_dim);
  if (a->task_count && (!a->task_offsets || !a->task_counts || !a->task_seeds || !a->task_members))
    return fail(TESSA_ERR_INVALID_ARG, "null task arrays");
  if (!a->codes || !a->scales || !a->sq8_norms || !a->leaf_rows || !a->leaf_starts || !a->leaf_sizes)
    return fail(TESSA_ERR_INVALID_ARG, "null data or output pointer");
  if (a->leaf_max == 0 || a->leaf_min == 0 || a->max_depth == 0 || a->max_leaders < 2)
    return fail(TESSA_ERR_INVALID_ARG, "leaf_max, leaf_min, max_depth must be positive and max_leaders >= 2");
  if (a->fanout_second == 0 || a->fanout_second > TESSA_MAX_RH)
    return fail(TESSA_ERR_INVALID_ARG, "fanout_second=%u outside 1..4 (GPU_PERSISTENT_FANOUT_OVER_32)",
                a->fanout_second);
  if (a->small_node_limit > 4096 || a->small_node_limit < 2)
    return fail(TESSA_ERR_UNSUPPORTED, "small_node_limit=%u outside 2..4096", a->small_node_limit);
  if (a->leaf_max > a->small_node_limit)
    return fail(TESSA_ERR_UNSUPPORTED, "leaf_max=%u above small_node_limit=%u (GPU_PERSISTENT_QUEUE_ROW_OVERFLOW)",
                a->leaf_max, a->small_node_limit);
  if (!(a->psamp_fraction > 0.0f) || !(a->psamp_fraction <= 1.0f))
    return fail(TESSA_ERR_INVALID_ARG, "psamp_fraction outside (0, 1]");
  if (a->resident_rows > 0xffffffffull) return fail(TESSA_ERR_UNSUPPORTED, "resident rows beyond 2^32");
  uint64_t total = 0;
  for (uint32_t t = 0; t < a->task_count; ++t) {
    if (a->task_offsets[t] + a->task_counts[t] > a->member_rows)
      return fail(TESSA_ERR_INVALID_ARG, "subtree task %u rows outside task_members", t);
    total += a->task_counts[t];
  }
  // arena positions are 32-bit: the tasks' rows, each in at most fanout_second leaves
  if ((uint64_t)a->fanout_second * total >= 0xfffffff0ull)
    return fail(TESSA_ERR_UNSUPPORTED, "fanout_second * task rows beyond 2^32");
  if (!ctx->subtree) {
    ctx->subtree = subtree_state_new();
    if (!ctx->subtree) return fail(TESSA_ERR_OOM, "subtree state allocation failed");
  }
  cudaStream_t st = (cudaStream_t)stream;  // NULL: the legacy default stream
  TRY(clear_err(ctx, st));
  SubtreeStats stats{};
  const int rc = subtree_partition(ctx->subtree, *a, &stats, ctx->d_err.as<uint32_t>(), ctx->sm_count,
                                   ctx->timeout_ns, st);
  if (rc != TESSA_OK) return rc;
  result->leaf_count = stats.leaf_count;
  result->leaf_rows_used = stats.leaf_rows_used;
  result->rounds = stats.rounds;
  result->large_assignments = stats.large_assignments;
  result->retries = stats.retries;
  result->balanced = stats.balanced;
  result->small_nodes = stats.small_nodes;
  result->kernel_launches = stats.launches;
  result->assign_ms = stats.assign_ms;
  result->scatter_ms = stats.scatter_ms;
  result->small_ms = stats.small_ms;
  result->wall_ms = stats.wall_ms;
  result->host_prep_ms = stats.host_prep_ms;
  result->host_decide_ms = stats.host_decide_ms;
  result->sync_wait_ms = stats.sync_wait_ms;
  return TESSA_OK;
}

// ------------------------------------------------- subtree submissions

int tessa_subtree_submit(tessa_ctx* ctx, const tessa_subtree_request* req, uint64_t* ticket, void* stream) {
  TRY(bind(ctx));
  if (!req || !ticket) return fail(TESSA_ERR_INVALID_ARG, "null request or ticket");
  const tessa_subtree_args& a = req->partition;
  if (req->k == 0 || req->k > TESSA_MAX_LEAF_K)
    return fail(TESSA_ERR_INVALID_ARG, "k=%u outside 1..%d", req->k, TESSA_MAX_LEAF_K);
  if (!req->global_ids || !a.codes || !a.scales || !a.sq8_norms || !a.task_members)
    return fail(TESSA_ERR_INVALID_ARG, "null device input");
  if (a.task_count && (!a.task_offsets || !a.task_counts || !a.task_seeds))
    return fail(TESSA_ERR_INVALID_ARG, "null task array");
  if (!ctx->ring) TRY(submit_ring_create(ctx->device, &ctx->ring));
  return submit_ring_submit(ctx->ring, req, ticket, (cudaStream_t)stream);
}

int tessa_subtree_poll(tessa_ctx* ctx, uint64_t ticket, int wait, tessa_compact_view* view) {
  if (!ctx || !view) return fail(TESSA_ERR_INVALID_ARG, "null context or view");
  if (!ctx->ring) return fail(TESSA_ERR_INVALID_ARG, "no submission on this context");
  return submit_ring_poll(ctx->ring, ticket, wait, view);
}

int tessa_subtree_release(tessa_ctx* ctx, uint64_t ticket) {
  if (!ctx) return fail(TESSA_ERR_INVALID_ARG, "null context");
  if (!ctx->ring) return fail(TESSA_ERR_INVALID_ARG, "no submission on this context");
  return submit_ring_release(ctx->ring, ticket);
}

// ----------------------------------------------------- record grouping

int tessa_group_edges(tessa_ctx* ctx, const uint32_t* point_ids, const uint32_t* topk_ids, const float* topk_dists,
                      const uint16_t* hash_fwd, const uint16_t* hash_rev, uint64_t rows, uint32_t k,
                      uint64_t num_points, uint64_t* offsets, tessa_edge* edges, uint64_t edge_capacity,
                      void* stream) {
  TRY(bind(ctx));
  if (!offsets || (rows && (!point_ids || !topk_ids || !topk_dists || !hash_fwd || !hash_rev || !edges)))
    return fail(TESSA_ERR_INVALID_ARG, "null record or output pointer");
  if (k == 0 || k > TESSA_MAX_LEAF_K) return fail(TESSA_ERR_INVALID_ARG, "k=%u outside 1..%d", k, TESSA_MAX_LEAF_K);
  if (num_points == 0 || num_points > 0xffffffffull) return fail(TESSA_ERR_INVALID_ARG, "num_points outside 1..2^32");
  if (edge_capacity < 2 * rows * (uint64_t)k)
    return fail(TESSA_ERR_INVALID_ARG, "edge_capacity %llu below 2 * rows * k = %llu",
                (unsigned long long)edge_capacity, (unsigned long long)(2 * rows * (uint64_t)k));
  const uint64_t m = 2 * rows * (uint64_t)k;
  if (m >= 0xffffffffull)
    return fail(TESSA_ERR_UNSUPPORTED, "2 * rows * k = %llu edges in one batch; at most 2^32 - 1 (split the batch)",
                (unsigned long long)m);
  cudaStream_t st = (cudaStream_t)stream;  // NULL: the legacy default stream
  TRY(ctx->g_temp.ensure(group_edges_scratch_bytes(m, num_points)));
  TRY(clear_err(ctx, st));
  GroupEdgesCall g{point_ids, topk_ids, topk_dists, hash_fwd, hash_rev, rows, k, num_points, offsets,
                   edges, ctx->g_temp.ptr, ctx->g_temp.bytes, ctx->d_err.as<uint32_t>(), ctx->sm_count};
  const int rc = group_edges(g, st);
  if (rc != TESSA_OK) return fail(rc, "edge grouping failed (code %d)", rc);
  uint32_t bits = 0;
  TRY(read_err(ctx, st, &bits));
  return map_device_error(bits);
}

// ------------------------------------------------ device reservoirs

namespace {

int reduce_common(tessa_ctx* ctx, ReservoirCall& r, uint64_t* slot_count, void* stream) {
  if (!r.out_offsets || !slot_count) return fail(TESSA_ERR_INVALID_ARG, "null output offsets or slot count");
  if (r.l_max == 0 || r.l_max > 255) return fail(TESSA_ERR_INVALID_ARG, "l_max=%u outside 1..255", r.l_max);
  if (r.num_points == 0 || r.num_points > 0xffffffffull)
    return fail(TESSA_ERR_INVALID_ARG, "num_points outside 1..2^32");
  if (r.edges >= 0xffffffffull)
    return fail(TESSA_ERR_UNSUPPORTED, "%llu edges in one reduction; at most 2^32 - 1 (reduce in pieces and merge "
                "the reservoirs)", (unsigned long long)r.edges);
  if (r.capacity && !r.out_neighbors && !r.out_slots)
    return fail(TESSA_ERR_INVALID_ARG, "slot capacity given without an output array");
  cudaStream_t st = (cudaStream_t)stream;  // NULL: the legacy default stream
  TRY(ctx->g_temp.ensure(reservoir_scratch_bytes(r.edges, r.num_points)));
  TRY(clear_err(ctx, st));
  r.temp = ctx->g_temp.ptr;
  r.temp_bytes = ctx->g_temp.bytes;
  r.d_err = ctx->d_err.as<uint32_t>();
  r.sm_count = ctx->sm_count;
  const int rc = reduce_reservoirs(r, st);
  if (rc != TESSA_OK) return fail(rc, "reservoir reduction failed (code %d)", rc);
  uint32_t bits = 0;
  TRY(read_err(ctx, st, &bits));
  TRY(map_device_error(bits));
  uint64_t total = 0;
  if (cudaMemcpyAsync(&total, r.out_offsets + r.num_points, 8, cudaMemcpyDeviceToHost, st) != cudaSuccess ||
      cudaStreamSynchronize(st) != cudaSuccess)
    return fail(TESSA_ERR_CUDA, "reading the slot total failed");
  *slot_count = total;
  if (total > r.capacity && (r.out_neighbors || r.out_slots))
    return fail(TESSA_ERR_INVALID_ARG, "slot capacity %llu below the slot total %llu",
                (unsigned long long)r.capacity, (unsigned long long)total);
  return TESSA_OK;
}

}  // namespace

int tessa_reduce_records(tessa_ctx* ctx, const uint32_t* point_ids, const uint32_t* topk_ids, const float* topk_dists,
                         const uint16_t* hash_fwd, const uint16_t* hash_rev, uint64_t rows, uint32_t k,
                         uint64_t num_points, uint32_t l_max, uint64_t* out_offsets, uint32_t* out_neighbors,
                         tessa_edge* out_slots, uint64_t slot_capacity, uint64_t* slot_count, void* stream) {
  TRY(bind(ctx));
  if (rows && (!point_ids || !topk_ids || !topk_dists || !hash_fwd || !hash_rev))
    return fail(TESSA_ERR_INVALID_ARG, "null record pointer");
  if (k == 0 || k > TESSA_MAX_LEAF_K) return fail(TESSA_ERR_INVALID_ARG, "k=%u outside 1..%d", k, TESSA_MAX_LEAF_K);
  ReservoirCall r{};
  r.point_ids = point_ids;
  r.topk_ids = topk_ids;
  r.topk_dists = topk_dists;
  r.hash_fwd = hash_fwd;
  r.hash_rev = hash_rev;
  r.rows = rows;
  r.k = k;
  r.edges = 2 * rows * (uint64_t)k;
  r.num_points = num_points;
  r.l_max = l_max;
  r.out_offsets = out_offsets;
  r.out_neighbors = out_neighbors;
  r.out_slots = out_slots;
  r.capacity = slot_capacity;
  return reduce_common(ctx, r, slot_count, stream);
}

int tessa_reduce_grouped(tessa_ctx* ctx, uint32_t groups, const uint64_t* const* group_offsets,
                         const tessa_edge* const* group_edges, const uint64_t* group_edge_counts,
                         uint64_t num_points, uint32_t l_max, uint64_t* out_offsets, uint32_t* out_neighbors,
                         tessa_edge* out_slots, uint64_t slot_capacity, uint64_t* slot_count, void* stream) {
  TRY(bind(ctx));
  if (groups == 0 || !group_offsets || !group_edges || !group_edge_counts)
    return fail(TESSA_ERR_INVALID_ARG, "no groups, or a null group array");
  ReservoirCall r{};
  uint64_t m = 0;
  for (uint32_t g = 0; g < groups; ++g) {
    if (!group_offsets[g] || (group_edge_counts[g] && !group_edges[g]))
      return fail(TESSA_ERR_INVALID_ARG, "group %u: null offsets or edges", g);
    m += group_edge_counts[g];
  }
  r.groups = groups;
  r.group_offsets = group_offsets;
  r.group_edges = group_edges;
  r.group_counts = group_edge_counts;
  r.edges = m;
  r.num_points = num_points;
  r.l_max = l_max;
  r.out_offsets = out_offsets;
  r.out_neighbors = out_neighbors;
  r.out_slots = out_slots;
  r.capacity = slot_capacity;
  return reduce_common(ctx, r, slot_count, stream);
}

// --------------------------------------------------- bounded-wait probe

namespace {

// Two waiters on barriers that nothing arrives on: warp 0 with the probe's
// limit, warp 1 with a limit far beyond it.  Warp 0 gives up first, records
// the timeout and raises the CTA's abort flag; warp 1 must then leave at its
// next check instead of running to its own limit -- the way every role of a
// pipeline drains after one of its waits gives up.
__global__ void wait_probe_kernel(uint32_t* err_word, uint64_t timeout_ns, unsigned long long* elapsed_ns) {
  __shared__ __align__(8) uint64_t bars[2];
  __shared__ uint32_t abort_word;
  volatile uint32_t* abort_flag = &abort_word;
  if (threadIdx.x == 0) {
    mbar_init(&bars[0], 1);
    mbar_init(&bars[1], 1);
    abort_word = 0u;
    fence_barrier_init();
  }
  __syncthreads();
  const uint64_t t0 = global_timer_ns();
  if (threadIdx.x == 0) mbar_wait(&bars[0], 0u, abort_flag, err_word, timeout_ns);
  if (threadIdx.x == 32) mbar_wait(&bars[1], 0u, abort_flag, err_word, 20ull * timeout_ns + 2000000000ull);
  __syncthreads();
  if (threadIdx.x == 0) *elapsed_ns = global_timer_ns() - t0;
}

}  // namespace

int tessa_set_leaf_kernel(tessa_ctx* ctx, uint32_t mode) {
  if (!ctx) return fail(TESSA_ERR_INVALID_ARG, "null context");
  if (mode > 1) return fail(TESSA_ERR_INVALID_ARG, "leaf kernel mode %u outside 0..1", mode);
  ctx->leaf_kernel = mode;
  return TESSA_OK;
}

int tessa_set_wait_timeout_ns(tessa_ctx* ctx, uint64_t timeout_ns) {
  if (!ctx) return fail(TESSA_ERR_INVALID_ARG, "null context");
  if (timeout_ns == 0) {
    ctx->timeout_ns = kDefaultTimeoutNs;
    return TESSA_OK;
  }
  if (timeout_ns < kMinTimeoutNs || timeout_ns > kMaxTimeoutNs)
    return fail(TESSA_ERR_INVALID_ARG, "wait limit %llu ns outside %llu..%llu ns", (unsigned long long)timeout_ns,
                (unsigned long long)kMinTimeoutNs, (unsigned long long)kMaxTimeoutNs);
  ctx->timeout_ns = timeout_ns;
  return TESSA_OK;
}

int tessa_check_bounded_wait(tessa_ctx* ctx, uint64_t timeout_ns, uint64_t* elapsed_ns, void* stream) {
  TRY(bind(ctx));
  if (timeout_ns < 1000ull || timeout_ns > kMaxTimeoutNs)
    return fail(TESSA_ERR_INVALID_ARG, "probe limit %llu ns outside 1000..%llu ns", (unsigned long long)timeout_ns,
                (unsigned long long)kMaxTimeoutNs);
  cudaStream_t st = (cudaStream_t)stream;  // NULL: the legacy default stream
  TRY(ctx->probe.ensure(8));
  TRY(clear_err(ctx, st));
  wait_probe_kernel<<<1, 64, 0, st>>>(ctx->d_err.as<uint32_t>(), timeout_ns,
                                       ctx->probe.as<unsigned long long>());
  CUDA_TRY(cudaGetLastError());
  uint64_t ns = 0;
  CUDA_TRY(cudaMemcpyAsync(&ns, ctx->probe.ptr, 8, cudaMemcpyDeviceToHost, st));
  uint32_t bits = 0;
  TRY(read_err(ctx, st, &bits));
  if (elapsed_ns) *elapsed_ns = ns;
  return map_device_error(bits);
}

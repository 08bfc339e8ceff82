// Distillation from a teacher's top-k list: loss and gradient over all vocab
// logits of a row.
//
//   q = softmax(z / tau), p = softmax of the list, P_v = sum of p_j with id_j = v
//   loss = tau^2 sum_j p_j (log p_j - log q[id_j]),  dz_v = w tau (q_v - P_v)
//
// q needs the row's maximum and sum before its first gradient can be written,
// so a plain form reads the row two or three times.  Here a cluster of CTAs
// holds a row: each CTA streams its slice once, keeping the running maximum m
// and sum of exp((z - m) / tau) per thread and the raw values in shared
// memory, the CTAs exchange (m, sum) through distributed shared memory, and
// the gradient is written from shared memory: one read and one write of the
// row, the bytes that the operator cannot do without.  The dense part ignores
// the list; the few entries of the list are then rewritten by the CTA that
// owns them (a thread of the same CTA wrote them before the barrier).
//
// One warp of each CTA stands beside the stream: it reads the list, gathers
// the listed logits, and makes p and P while the others read the row.
#include "train_common.cuh"

namespace tessa {
namespace train {

// 2^x to within 2 ulp for normal results, smaller ones flushed to zero.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// (maximum, sum of 2^((x - maximum) c)) of a set; the empty set is (-inf, 0).
struct Stat {
  float m, s;
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ Stat join(Stat a, Stat b, float c) {
  const float m = fmaxf(a.m, b.m), base = base_of(m);
  return {m, a.s * ex2((a.m - base) * c) + b.s * ex2((b.m - base) * c)};
}

struct DistillPlan {
  uint32_t cluster;     // CTAs a row
  uint32_t keep_bytes;  // shared memory for the slice (0: the second pass reads the row again)
};

constexpr uint32_t kNoEntry = 0xffffffffu;
constexpr uint32_t kMaxKeep = 200u << 10;  // the largest slice a CTA keeps, beside the longest list

template <class T, int WARPS>
__global__ void __launch_bounds__((WARPS + 1) * 32)
    distill_kernel(const tessa_distill_args a, const DistillPlan plan, uint32_t* err) {
  constexpr uint32_t VE = 16u / sizeof(T);
  constexpr uint32_t NT = WARPS * 32u;
  extern __shared__ __align__(16) uint8_t smem[];
  const uint32_t k4 = (a.k + 3u) / 4u * 4u;
  uint32_t* l_id = reinterpret_cast<uint32_t*>(smem);          // the entry's id, kNoEntry if it takes no part
  float* l_p = reinterpret_cast<float*>(smem) + k4;            // p_j
  float* l_z = l_p + k4;                                       // the student's logit
  float* l_own = l_z + k4;                                     // P of the id at its first entry, -1 elsewhere
  Vec<T, VE>* kept = reinterpret_cast<Vec<T, VE>*>(l_own + k4);
  __shared__ Stat warp_stat[WARPS];
  __shared__ Stat cta_stat[16];
  __shared__ float l_sum;  // 0: the list has no entry
  __shared__ float l_max;

  const uint32_t tid = threadIdx.x, warp = tid / 32u, lane = tid % 32u;
  const uint32_t C = plan.cluster, rank = C > 1 ? blockIdx.x % C : 0u;
  const uint64_t row = blockIdx.x / C;
  const float c = 1.44269504088896341f / a.temperature;
  const T* z = static_cast<const T*>(a.logits) + row * a.stride;
  // 16-byte body of the row, split by rank; what stands before and after it
  // (less than a vector each) belongs to rank 0.
  const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(z) % 16u);
  uint64_t head = off ? (16u - off) / sizeof(T) : 0u;
  if (head > a.vocab) head = a.vocab;
  const uint64_t body = (a.vocab - head) / VE, tail0 = head + body * VE;
  const uint64_t lo = body * rank / C, hi = body * (rank + 1) / C;
  const uint32_t n = (uint32_t)(hi - lo);
  const Vec<T, VE>* zv = reinterpret_cast<const Vec<T, VE>*>(z + head) + lo;
  // the thread's element of head or tail, if any
  uint64_t extra = a.vocab;
  if (rank == 0) {
    if (tid < head) extra = tid;
    else if (tid >= 32u && tid - 32u < a.vocab - tail0) extra = tail0 + (tid - 32u);
  }
  const bool keep = plan.keep_bytes != 0;
  // a peer's shared memory may be written once the peer has started
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  float ze = -INFINITY;

  if (warp < WARPS) {
    Stat st = {-INFINITY, 0.0f};
    if (extra < a.vocab) {
      ze = to_f32(z[extra]);
      st.m = ze;
      st.s = ex2((ze - base_of(ze)) * c);
    }
    for (uint32_t i = tid; i < n; i += 4u * NT) {
      Vec<T, VE> x[4];
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u)
        if (i + u * NT < n) x[u] = zv[i + u * NT];
      float top = st.m;
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u)
        if (i + u * NT < n) {
          if (keep) kept[i + u * NT] = x[u];
#pragma unroll
          for (uint32_t v = 0; v < VE; ++v) top = fmaxf(top, to_f32(x[u].v[v]));
        }
      const float base = base_of(top);
      if (top > st.m) st.s *= ex2((st.m - base) * c);
      st.m = top;
      float sum = 0.0f;
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u)
        if (i + u * NT < n) {
#pragma unroll
          for (uint32_t v = 0; v < VE; ++v) sum += ex2((to_f32(x[u].v[v]) - base) * c);
        }
      st.s += sum;
    }
#pragma unroll
    for (uint32_t o = 16; o; o >>= 1) {
      const Stat b = {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o)};
      st = join(st, b, c);
    }
    if (lane == 0) warp_stat[warp] = st;
  } else {
    // ------------------------------------------------ the teacher's list
    float top = -INFINITY;
    for (uint32_t j = lane; j < k4; j += 32u) {
      uint32_t id = kNoEntry;
      float t = -INFINITY;
      if (j < a.k) {
        const uint64_t at = row * a.k + j;
        const int64_t v = a.id_bits == 32 ? (int64_t)static_cast<const int32_t*>(a.teacher_ids)[at]
                                          : static_cast<const int64_t*>(a.teacher_ids)[at];
        t = a.teacher_logits[at];
        if (v >= 0 && (uint64_t)v < a.vocab) {
          if (t != -INFINITY) id = (uint32_t)v;
        } else if (v != -1) {
          report(err, TESSA_DEVERR_BAD_ROW);
        }
      }
      l_id[j] = id;
      l_p[j] = t;
      if (id != kNoEntry) top = fmaxf(top, t);
      const uint64_t vec = (id - head) / VE;
      const bool mine = id != kNoEntry && (id < head || id >= tail0 ? rank == 0 : vec >= lo && vec < hi);
      // rank 0 needs every listed logit for the loss
      l_z[j] = (mine || (rank == 0 && id != kNoEntry)) ? to_f32(z[id]) : 0.0f;
      l_own[j] = mine ? 0.0f : -1.0f;
    }
#pragma unroll
    for (uint32_t o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float sum = 0.0f;
    for (uint32_t j = lane; j < k4; j += 32u)
      if (l_id[j] != kNoEntry) sum += ex2((l_p[j] - top) * c);
#pragma unroll
    for (uint32_t o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      l_sum = sum;
      l_max = top;
    }
    if (a.grad) {
      __syncwarp();
      // P of each id at its first entry in this CTA's slice
      for (uint32_t j = lane; j < a.k; j += 32u) {
        if (l_own[j] < 0.0f) continue;
        const uint32_t id = l_id[j];
        float P = 0.0f;
        bool first = true;
        const uint4* ids = reinterpret_cast<const uint4*>(l_id);
        for (uint32_t i = 0; i < k4 / 4u; ++i) {
          const uint4 q = ids[i];
          const uint32_t e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (uint32_t u = 0; u < 4; ++u)
            if (e[u] == id) {
              if (i * 4u + u < j) first = false;
              P += ex2((l_p[i * 4u + u] - top) * c) / sum;
            }
        }
        l_own[j] = first ? P : -1.0f;
      }
    }
  }
  __syncthreads();
  Stat row_stat = warp_stat[0];
#pragma unroll
  for (uint32_t w = 1; w < WARPS; ++w) row_stat = join(row_stat, warp_stat[w], c);
  if (C > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid < C) {
      const uint32_t to = mapa_shared(&cta_stat[rank], tid);
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(row_stat.m), "f"(row_stat.s) : "memory");
    }
    cluster_sync();
    row_stat = cta_stat[0];
    for (uint32_t r = 1; r < C; ++r) row_stat = join(row_stat, cta_stat[r], c);
  }
  const float base = base_of(row_stat.m);
  const float inv_tau = 1.0f / a.temperature;
  const float log_s = logf(row_stat.s);
  const bool empty = row_stat.m == -INFINITY && row_stat.s == 0.0f;  // a row of NaN is not
  const bool active = l_sum != 0.0f && !empty;

  if (warp == WARPS && rank == 0) {
    float part = 0.0f;
    if (active) {
      const float log_l = logf(l_sum);
      for (uint32_t j = lane; j < a.k; j += 32u) {
        if (l_id[j] == kNoEntry) continue;
        // tau (log p - log q): no division, which could overflow a logit of the type's lowest value
        const float d = l_p[j] - l_max;
        const float p = ex2(d * c) / l_sum;
        if (p != 0.0f) part += (a.temperature * p) * ((d - (l_z[j] - base)) + a.temperature * (log_s - log_l));
      }
    }
#pragma unroll
    for (uint32_t o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if (lane == 0) {
      if (a.loss) a.loss[row] = active ? part : 0.0f;
      if (a.lse) a.lse[row] = empty ? -INFINITY : row_stat.m * inv_tau + log_s;
    }
  }
  if (!a.grad) return;

  const float wt = a.temperature * (a.row_weights ? a.row_weights[row] : 1.0f);
  const float f = active ? wt / row_stat.s : 0.0f;
  T* g = static_cast<T*>(a.grad) + row * a.grad_stride;
  const bool aligned = reinterpret_cast<uintptr_t>(g) % 16u == off;
  if (warp < WARPS) {
    for (uint32_t i = tid; i < n; i += NT) {
      const Vec<T, VE> x = keep ? kept[i] : zv[i];
      Vec<T, VE> y;
#pragma unroll
      for (uint32_t v = 0; v < VE; ++v) {
        const float q = ex2((to_f32(x.v[v]) - base) * c) * f;
        y.v[v] = from_f32<T>(active ? q : 0.0f);
      }
      T* dst = g + head + (lo + i) * VE;
      if (aligned) {
        *reinterpret_cast<Vec<T, VE>*>(dst) = y;
      } else {
#pragma unroll
        for (uint32_t v = 0; v < VE; ++v) dst[v] = y.v[v];
      }
    }
    if (extra < a.vocab) g[extra] = from_f32<T>(active ? ex2((ze - base) * c) * f : 0.0f);
  }
  if (!active) return;
  __syncthreads();
  for (uint32_t j = tid; j < a.k; j += NT + 32u)
    if (l_own[j] >= 0.0f) g[l_id[j]] = from_f32<T>(ex2((l_z[j] - base) * c) * f - wt * l_own[j]);
}

template <class T, int WARPS>
cudaError_t launch_distill_as(const tessa_distill_args& a, const DistillPlan& plan, const AsyncCtx& c,
                              cudaStream_t stream) {
  const uint32_t smem = (a.k + 3u) / 4u * 64u + plan.keep_bytes;
  static SmemRaised raised;
  cudaError_t e = raise_smem(distill_kernel<T, WARPS>, c.device, kMaxKeep + 64 * 256, raised);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((uint32_t)(a.rows * plan.cluster));
  cfg.blockDim = dim3((WARPS + 1) * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = plan.cluster;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = plan.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, distill_kernel<T, WARPS>, a, plan, c.err);
}

}  // namespace train

cudaError_t launch_distill(const tessa_distill_args& a, const AsyncCtx& c, cudaStream_t stream) {
  using namespace train;
  const uint64_t bytes = a.vocab * type_bytes(a.dtype);
  constexpr uint64_t kKeep = 96u << 10;  // a slice of this size leaves room for two CTAs an SM
  DistillPlan plan = {1, 0};
  // The fewest CTAs a row that can keep it; more while rows alone do not fill the GPU.
  while (plan.cluster < 8 && (bytes / plan.cluster > kKeep || (a.rows * plan.cluster < (uint64_t)c.sm_count * 2 &&
                                                             bytes / plan.cluster > 16384)))
    plan.cluster *= 2;
  const uint64_t slice = div_up(bytes, plan.cluster) + 16;
  if (a.grad && slice <= kMaxKeep) plan.keep_bytes = (uint32_t)(div_up(slice, 16) * 16);
  return with_type(a.dtype, [&](auto t) {
    if (slice <= 32768 + 16) return launch_distill_as<decltype(t), 8>(a, plan, c, stream);
    return launch_distill_as<decltype(t), 16>(a, plan, c, stream);
  });
}

}  // namespace tessa

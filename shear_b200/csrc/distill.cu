// Distillation from a teacher's top-k list: loss and gradient over all vocab
// logits of a row.
//
//   q = softmax(z / tau), p = softmax of the list, P_v = sum of p_j with id_j = v
//   loss = tau^2 sum_j p_j (log p_j - log q[id_j]),  dz_v = w tau (q_v - P_v)
//
// q needs the row's maximum and sum before its first gradient can be written,
// so a plain form reads the row two or three times.  Here a row is read once,
// keeping the running maximum m and sum of exp((z - m) / tau) per thread and
// the raw values in shared memory, and the gradient is written from there: one
// read and one write of the row, the bytes that the operator cannot do without.
// The dense part ignores the list; the few entries of the list are then
// rewritten (a thread of the same CTA wrote them before the barrier).
// A row that one CTA cannot keep, or one of few, is shared by a cluster of
// CTAs, each with a slice, which exchange (m, sum) through distributed shared
// memory.  Rows of a megabyte and more take two reads: the loss first, then
// the gradient, each at memory speed.
// One warp of a CTA stands beside the others: it reads the list, gathers the
// listed logits, makes p and P while they read the row, and then the loss.
//
// Measured (B200, loss and gradient, rows from DRAM): 2048 x 16384 bf16 28 us
// (4.8 TB/s of the read and the write), bound by instruction issue and the
// exponentials (two a logit at 16 a cycle and SM: 16 us); 4096 x 50000 bf16 177
// us (4.6 TB/s); 296 x 50003 f16 16 us, but 333 rows 24: two rows an SM, so 37
// of them start late; 1024 x 1M bf16 0.95 ms (4.3 TB/s; 6.4 of what the two forms
// together move); the loss alone 0.32 ms (6.4 TB/s).
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
// The difference comes first: x c alone leaves f32 for a mask of the type's
// lowest value.
struct Stat {
  float m, s;
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ Stat join(Stat a, Stat b, float c) {
  const float m = fmaxf(a.m, b.m), base = base_of(m);
  return {m, a.s * ex2((a.m - base) * c) + b.s * ex2((b.m - base) * c)};
}

// Two neighbouring values of a vector as a pair of f32: the arithmetic below
// runs on pairs (two f32 operations an instruction), and the maximum of 16-bit
// values on the values as they are.  The kernel is bound by instruction issue
// before it is bound by memory: 29 instructions a value with scalar code.
template <class T>
struct Pairs;
template <>
struct Pairs<float> {
  static __device__ __forceinline__ uint64_t get(const uint4& v, int i) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    return f2_pack(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  }
  static __device__ __forceinline__ float top(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ void put(uint4& v, int i, float a, float b) {
    uint32_t* w = &v.x;
    w[2 * i] = __float_as_uint(a);
    w[2 * i + 1] = __float_as_uint(b);
  }
};
template <>
struct Pairs<__nv_bfloat16> {
  static __device__ __forceinline__ uint64_t get(const uint4& v, int i) {
    const uint32_t w = (&v.x)[i];
    return f2_pack(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ float top(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
  static __device__ __forceinline__ void put(uint4& v, int i, float a, float b) {
    reinterpret_cast<__nv_bfloat162*>(&v)[i] = __floats2bfloat162_rn(a, b);
  }
};
template <>
struct Pairs<__half> {
  static __device__ __forceinline__ uint64_t get(const uint4& v, int i) {
    const float2 f = __half22float2(reinterpret_cast<const __half2*>(&v)[i]);
    return f2_pack(f.x, f.y);
  }
  static __device__ __forceinline__ float top(const uint4& v) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const float2 m = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
  static __device__ __forceinline__ void put(uint4& v, int i, float a, float b) {
    reinterpret_cast<__half2*>(&v)[i] = __floats2half2_rn(a, b);
  }
};

// 2^((x - base) c) of both values of a pair; neg_base = (-base, -base).
__device__ __forceinline__ uint64_t ex2_pair(uint64_t x, uint64_t neg_base, uint64_t c2) {
  float a, b;
  f2_unpack(f2_mul(f2_add(x, neg_base), c2), a, b);
  return f2_pack(ex2(a), ex2(b));
}

constexpr uint32_t kNoEntry = 0xffffffffu;
constexpr uint32_t kListBytes = 16;        // an entry's id, p, logit and P in shared memory
constexpr uint32_t kFilterBits = 15;       // of ids, for lists of more than a warp
__host__ __device__ __forceinline__ uint32_t list_bytes(uint32_t k) {
  return (k + 3u) / 4u * 4u * kListBytes + (k > 32u ? 1u << (kFilterBits - 3) : 0u);
}
constexpr uint32_t kSmemMost = 227u << 10;

// A row's list in shared memory, k4 entries (k rounded up to four).
struct List {
  uint32_t* id;  // kNoEntry where the entry takes no part
  float* t;      // the teacher's logit
  float* z;      // the student's
  float* own;    // P of the id at its first entry of this CTA's slice, -1 elsewhere
  uint32_t* filter;  // bits of ids, k > 32
  float* sums;   // maximum of t, sum of 2^((t - maximum) c): 0 if there is no entry
};
__device__ __forceinline__ List list_at(uint8_t* at, uint32_t k4, float* sums) {
  uint32_t* id = reinterpret_cast<uint32_t*>(at);
  float* f = reinterpret_cast<float*>(at);
  return {id, f + k4, f + 2u * k4, f + 3u * k4, id + 4u * k4, sums};
}

// How a row lies: its 16-byte body, and what stands before and after it (less
// than a vector each).
struct Span {
  uint32_t head, body, tail0;
};
template <class T>
__device__ __forceinline__ Span span_of_row(const T* z, uint32_t vocab) {
  constexpr uint32_t VE = 16u / sizeof(T);
  const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(z) % 16u);
  Span s;
  s.head = min(vocab, off ? (16u - off) / (uint32_t)sizeof(T) : 0u);
  s.body = (vocab - s.head) / VE;
  s.tail0 = s.head + s.body * VE;
  return s;
}

// One warp: reads row's list; [lo, lo + n) of the body, and the ends where
// `ends`, are this CTA's to write.  `every`: the logits of other CTAs' entries
// are needed too (for the loss); `parts`: P is (for a gradient).
template <class T>
__device__ __forceinline__ void read_list(const tessa_distill_args& a, uint64_t row, const T* z, const Span& s,
                                          uint32_t lo, uint32_t n, bool ends, bool every, bool parts, const List& l,
                                          float c, uint32_t lane, uint32_t* err) {
  constexpr uint32_t VE = 16u / sizeof(T);
  const uint32_t k4 = (a.k + 3u) / 4u * 4u;
  float top = -INFINITY;
  // N entries a lane at a time: their reads are under way together, and then the listed logits'.
  auto read = [&](auto count) {
    constexpr uint32_t N = decltype(count)::value;
    for (uint32_t j0 = lane; j0 < k4; j0 += 32u * N) {
      int64_t v[N];
      float t[N], x[N];
#pragma unroll
      for (uint32_t u = 0; u < N; ++u) {
        const uint32_t j = j0 + u * 32u;
        const uint64_t at = row * a.k + j;
        v[u] = -1;
        t[u] = -INFINITY;
        if (j < a.k) {
          v[u] = a.id_bits == 32 ? (int64_t)static_cast<const int32_t*>(a.teacher_ids)[at]
                                 : static_cast<const int64_t*>(a.teacher_ids)[at];
          t[u] = a.teacher_logits[at];
        }
      }
      uint32_t id[N], mine = 0;
#pragma unroll
      for (uint32_t u = 0; u < N; ++u) {
        const bool in = v[u] >= 0 && (uint64_t)v[u] < a.vocab;
        if (!in && v[u] != -1) report(err, TESSA_DEVERR_BAD_ROW);
        id[u] = in && t[u] != -INFINITY ? (uint32_t)v[u] : kNoEntry;
        if (id[u] != kNoEntry && (id[u] < s.head || id[u] >= s.tail0 ? ends : (id[u] - s.head) / VE - lo < n)) mine |= 1u << u;
        x[u] = mine >> u & 1u || (every && id[u] != kNoEntry) ? to_f32(z[id[u]]) : 0.0f;
      }
#pragma unroll
      for (uint32_t u = 0; u < N; ++u) {
        const uint32_t j = j0 + u * 32u;
        if (j >= k4) break;
        l.id[j] = id[u];
        l.t[j] = t[u];
        l.z[j] = x[u];
        l.own[j] = mine >> u & 1u ? 0.0f : -1.0f;
        if (id[u] != kNoEntry) top = fmaxf(top, t[u]);
      }
    }
  };
  // (with lists of 32 four at a time cost issue slots: 2048 x 16384 bf16 32 us
  // instead of 28; with lists of 100 one at a time: 333 x 50003
  // f16 29 us instead of 27)
  if (a.k <= 32u) read(std::integral_constant<int, 1>());
  else read(std::integral_constant<int, 4>());
#pragma unroll
  for (uint32_t o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float sum = 0.0f;
  for (uint32_t j = lane; j < k4; j += 32u)
    if (l.id[j] != kNoEntry) sum += ex2((l.t[j] - top) * c);
#pragma unroll
  for (uint32_t o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) {
    l.sums[0] = top;
    l.sums[1] = sum;
  }
  __syncwarp();
  if (!parts) return;
  // Nearly every id stands in a list once.  Lists of a warp are matched lane by
  // lane; of longer ones only the entries that find their bit of the filter
  // taken look for others, the whole warp with each (every entry with all others
  // took 8 us for a list of 100, as long as the row itself).
  if (a.k <= 32u) {
    const bool in = lane < a.k && l.own[lane] >= 0.0f;
    const uint32_t same = __match_any_sync(0xffffffffu, in ? l.id[lane] : kNoEntry);
    if (!in) return;
    float w = ex2((l.t[lane] - top) * c);
    for (uint32_t more = same & ~(1u << lane); more; more &= more - 1u) w += ex2((l.t[__ffs(more) - 1] - top) * c);
    l.own[lane] = same & ((1u << lane) - 1u) ? -1.0f : w / sum;
    return;
  }
  for (uint32_t i = lane; i < 1u << (kFilterBits - 7); i += 32u) reinterpret_cast<uint4*>(l.filter)[i] = make_uint4(0, 0, 0, 0);
  __syncwarp();
  uint32_t taken = 0;  // bit n: entry 32 n + lane
  for (uint32_t j = lane; j < a.k; j += 32u) {
    if (l.own[j] < 0.0f) continue;
    const uint32_t h = l.id[j] * 2654435769u >> (32u - kFilterBits);
    if (atomicOr(l.filter + h / 32u, 1u << (h % 32u)) >> (h % 32u) & 1u) taken |= 1u << (j / 32u);
    l.own[j] = ex2((l.t[j] - top) * c) / sum;
  }
  for (uint32_t n32 = 0; n32 * 32u < a.k; ++n32) {
    for (uint32_t todo = __ballot_sync(0xffffffffu, taken >> n32 & 1u); todo; todo &= todo - 1u) {
      const uint32_t id = l.id[n32 * 32u + __ffs(todo) - 1u];
      uint32_t first = a.k;
      float w = 0.0f;
      for (uint32_t i = lane; i < a.k; i += 32u) {
        if (l.id[i] != id) continue;
        first = min(first, i);
        w += ex2((l.t[i] - top) * c);
      }
      first = __reduce_min_sync(0xffffffffu, first);
#pragma unroll
      for (uint32_t o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
      for (uint32_t i = lane; i < a.k; i += 32u)
        if (l.id[i] == id) l.own[i] = i == first ? w / sum : -1.0f;
    }
  }
}

// One warp: the row's loss and lse.
__device__ __forceinline__ void write_loss(const tessa_distill_args& a, uint64_t row, const List& l, const Stat& st,
                                           bool active, bool empty, float c, uint32_t lane) {
  const float log_s = logf(st.s), base = base_of(st.m);
  float part = 0.0f;
  if (active) {
    const float top = l.sums[0], sum = l.sums[1], log_l = logf(sum);
    for (uint32_t j = lane; j < a.k; j += 32u) {
      if (l.id[j] == kNoEntry) continue;
      // tau (log p - log q): no division, which could overflow a logit of the type's lowest value
      const float d = l.t[j] - top;
      const float p = ex2(d * c) / sum;
      if (p != 0.0f) part += (a.temperature * p) * ((d - (l.z[j] - base)) + a.temperature * (log_s - log_l));
    }
  }
#pragma unroll
  for (uint32_t o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if (lane == 0) {
    if (a.loss) a.loss[row] = active ? part : 0.0f;
    if (a.lse) a.lse[row] = empty ? -INFINITY : base * (1.0f / a.temperature) + log_s;
  }
}

// A thread's running statistics: maximum, and two partial sums (a pair).
struct Running {
  float m = -INFINITY, s0 = 0.0f, s1 = 0.0f;
  template <class T, int N>
  __device__ __forceinline__ void take(const uint4 (&x)[N], float c, uint64_t c2) {
    float top = m;
#pragma unroll
    for (int u = 0; u < N; ++u) top = fmaxf(top, Pairs<T>::top(x[u]));
    const float base = base_of(top);
    if (top > m) {
      const float f = ex2((m - base) * c);
      s0 *= f;
      s1 *= f;
      m = top;
    }
    const uint64_t nb = f2_pack(-base, -base);
    uint64_t sum = f2_pack(s0, s1);
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int v = 0; v < (int)(8 / sizeof(T)); ++v) sum = f2_add(sum, ex2_pair(Pairs<T>::get(x[u], v), nb, c2));
    f2_unpack(sum, s0, s1);
  }
  __device__ __forceinline__ Stat stat() const { return {m, s0 + s1}; }
};

// The statistics of N lanes' sets (N a power of two; every group of N lanes):
// the maximum first, so that each set is brought to it once.
template <int N>
__device__ __forceinline__ Stat join_lanes(Stat st, float c) {
  float m = st.m;
#pragma unroll
  for (int o = N / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float s = st.s * ex2((st.m - base_of(m)) * c);
#pragma unroll
  for (int o = N / 2; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return {m, s};
}
template <int WARPS>
__device__ __forceinline__ Stat join_warps(const Stat* warp_stat, uint32_t lane, float c) {
  return join_lanes<WARPS>(warp_stat[lane % WARPS], c);
}

// Gradients of a vector without the list's part.
template <class T>
__device__ __forceinline__ uint4 gradients(const uint4& x, uint64_t nb, uint64_t c2, uint64_t f2) {
  uint4 y;
#pragma unroll
  for (int v = 0; v < (int)(8 / sizeof(T)); ++v) {
    float a0, a1;
    f2_unpack(f2_mul(ex2_pair(Pairs<T>::get(x, v), nb, c2), f2), a0, a1);
    Pairs<T>::put(y, v, a0, a1);
  }
  return y;
}
template <class T>
__device__ __forceinline__ void put_vector(T* dst, const uint4& y, bool aligned) {
  if (aligned) {
    __stcs(reinterpret_cast<uint4*>(dst), y);
  } else {
    const T* v = reinterpret_cast<const T*>(&y);
#pragma unroll
    for (uint32_t e = 0; e < 16u / sizeof(T); ++e) dst[e] = v[e];
  }
}

struct DistillPlan {
  uint32_t cluster_log2;  // CTAs a row
  uint32_t keep_bytes;    // shared memory for the slice's first part; the second pass reads the rest again
  // Loss alone, for a gradient that follows in launches of its own:
  Stat* stats;            // rows
  uint32_t* ids;          // rows x k: the list's ids at their first entries (kNoEntry elsewhere),
  float2* terms;          // their logits and P
};

template <class T, int WARPS>
__global__ void __launch_bounds__((WARPS + 1) * 32, WARPS == 16 ? 2 : WARPS == 8 ? 5 : 9)
    distill_kernel(const tessa_distill_args a, const DistillPlan plan, uint32_t* err) {
  constexpr uint32_t VE = 16u / sizeof(T), NT = WARPS * 32u;
  extern __shared__ __align__(16) uint8_t smem[];
  const uint32_t k4 = (a.k + 3u) / 4u * 4u;
  __shared__ float sums[2];
  __shared__ Stat warp_stat[WARPS];
  __shared__ Stat cta_stat[16];
  const List l = list_at(smem, k4, sums);
  uint4* kept = reinterpret_cast<uint4*>(smem + list_bytes(a.k));

  const uint32_t tid = threadIdx.x, warp = tid / 32u, lane = tid % 32u;
  const uint32_t C = 1u << plan.cluster_log2, rank = blockIdx.x & (C - 1u);
  const uint64_t row = blockIdx.x >> plan.cluster_log2;
  const uint32_t vocab = (uint32_t)a.vocab;
  const float c = 1.44269504088896341f / a.temperature;
  const uint64_t c2 = f2_pack(c, c);
  const T* z = static_cast<const T*>(a.logits) + row * a.stride;
  // the body is split by rank; the ends belong to rank 0
  const Span s = span_of_row(z, vocab);
  const uint32_t per = (s.body + C - 1u) >> plan.cluster_log2;
  const uint32_t lo = min(s.body, per * rank), n = min(s.body, lo + per) - lo;
  const uint4* zv = reinterpret_cast<const uint4*>(z + s.head) + lo;
  uint32_t extra = vocab;  // the thread's element of the ends, if any
  if (rank == 0) {
    if (tid < s.head) extra = tid;
    else if (tid >= 32u && tid - 32u < vocab - s.tail0) extra = s.tail0 + (tid - 32u);
  }
  const uint32_t keep = min(n, plan.keep_bytes / 16u);  // vectors
  // a peer's shared memory may be written once the peer has started
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  float ze = -INFINITY;
  if (warp < WARPS) {
    if (extra < vocab) ze = to_f32(z[extra]);
    Running run;
    uint32_t i = tid;
    for (; i + 3u * NT < n; i += 4u * NT) {
      const uint4 v[4] = {zv[i], zv[i + NT], zv[i + 2u * NT], zv[i + 3u * NT]};
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u)
        if (i + u * NT < keep) kept[i + u * NT] = v[u];
      run.take<T>(v, c, c2);
    }
    for (; i < n; i += NT) {
      const uint4 v[1] = {zv[i]};
      if (i < keep) kept[i] = v[0];
      run.take<T>(v, c, c2);
    }
    Stat st = run.stat();
    if (extra < vocab) st = join(st, {ze, ex2((ze - base_of(ze)) * c)}, c);
    st = join_lanes<32>(st, c);
    if (lane == 0) warp_stat[warp] = st;
  } else {
    // rank 0 needs every listed logit for the loss
    const bool all = plan.stats != nullptr;  // and every P, where the gradient follows apart
    read_list(a, row, z, s, all ? 0u : lo, all ? s.body : n, rank == 0, rank == 0, a.grad || all, l, c, lane, err);
  }
  __syncthreads();
  Stat st = join_warps<WARPS>(warp_stat, lane, c);
  if (C > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid < C) {
      const uint32_t to = mapa_shared(&cta_stat[rank], tid);
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(st.m), "f"(st.s) : "memory");
    }
    cluster_sync();
    st = cta_stat[0];
    for (uint32_t r = 1; r < C; ++r) st = join(st, cta_stat[r], c);
  }
  const float base = base_of(st.m);
  const bool empty = st.m == -INFINITY && st.s == 0.0f;  // a row of NaN is not
  const bool active = l.sums[1] != 0.0f && !empty;
  if (warp == WARPS && rank == 0) {
    write_loss(a, row, l, st, active, empty, c, lane);
    if (plan.stats) {
      // a row that takes no part: a base and a sum that make every gradient 0
      if (lane == 0) plan.stats[row] = active ? st : Stat{INFINITY, INFINITY};
      for (uint32_t j = lane; j < a.k; j += 32u) {
        plan.ids[row * a.k + j] = active && l.own[j] >= 0.0f ? l.id[j] : kNoEntry;
        plan.terms[row * a.k + j] = make_float2(l.z[j], l.own[j]);
      }
    }
  }
  if (!a.grad) return;

  const float wt = a.temperature * (a.row_weights ? a.row_weights[row] : 1.0f);
  const float f = active ? wt / st.s : 0.0f;
  T* g = static_cast<T*>(a.grad) + row * a.grad_stride;
  T* body = g + s.head + (uint64_t)lo * VE;
  const bool aligned = reinterpret_cast<uintptr_t>(g + s.head) % 16u == 0u;
  if (warp < WARPS) {
    const uint64_t nb = f2_pack(-base, -base), f2 = f2_pack(f, f);
    if (active) {
#pragma unroll 2
      for (uint32_t i = tid; i < keep; i += NT)
        put_vector(body + (uint64_t)i * VE, gradients<T>(kept[i], nb, c2, f2), aligned);
      // what was not kept, by the threads that read it (the gradient may be the logits' place)
#pragma unroll 4
      for (uint32_t i = tid + (keep > tid ? (keep - tid + NT - 1u) / NT * NT : 0u); i < n; i += NT)
        put_vector(body + (uint64_t)i * VE, gradients<T>(zv[i], nb, c2, f2), aligned);
    } else {
      for (uint32_t i = tid; i < n; i += NT) put_vector(body + (uint64_t)i * VE, make_uint4(0u, 0u, 0u, 0u), aligned);
    }
    if (extra < vocab) g[extra] = from_f32<T>(active ? ex2((ze - base) * c) * f : 0.0f);
  }
  if (!active) return;
  __syncthreads();
  for (uint32_t j = tid; j < a.k; j += NT + 32u)
    if (l.own[j] >= 0.0f) g[l.id[j]] = from_f32<T>(ex2((l.z[j] - base) * c) * f - wt * l.own[j]);
}

// The gradient of long rows after the loss' launch: a block takes a piece of a
// row; the listed entries follow in a launch of their own.
constexpr uint32_t kPieceVecs = 4096;  // 64 KB
template <class T>
__global__ void __launch_bounds__(256) dense_gradient_kernel(const tessa_distill_args a, const Stat* stats,
                                                             uint32_t pieces) {
  constexpr uint32_t VE = 16u / sizeof(T);
  const uint64_t row = blockIdx.x / pieces;
  const uint32_t piece = blockIdx.x % pieces, vocab = (uint32_t)a.vocab;
  const float c = 1.44269504088896341f / a.temperature;
  const T* z = static_cast<const T*>(a.logits) + row * a.stride;
  T* g = static_cast<T*>(a.grad) + row * a.grad_stride;
  const Span s = span_of_row(z, vocab);
  const Stat st = stats[row];
  const bool zero = st.m == INFINITY && st.s == INFINITY;
  const float base = base_of(st.m);
  const float f = zero ? 0.0f : a.temperature * (a.row_weights ? a.row_weights[row] : 1.0f) / st.s;
  const uint64_t nb = f2_pack(-base, -base), c2 = f2_pack(c, c), f2 = f2_pack(f, f);
  const uint4* zv = reinterpret_cast<const uint4*>(z + s.head);
  const bool aligned = reinterpret_cast<uintptr_t>(g + s.head) % 16u == 0u;
  const uint32_t end = min(s.body, (piece + 1u) * kPieceVecs);
  auto put = [&](uint32_t i, const uint4& x) {
    put_vector(g + s.head + (uint64_t)i * VE, zero ? make_uint4(0u, 0u, 0u, 0u) : gradients<T>(x, nb, c2, f2), aligned);
  };
  uint32_t i = piece * kPieceVecs + threadIdx.x;
  for (; i + 768u < end; i += 1024u) {
    const uint4 x[4] = {zv[i], zv[i + 256u], zv[i + 512u], zv[i + 768u]};
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) put(i + u * 256u, x[u]);
  }
  for (; i < end; i += 256u) put(i, zv[i]);
  if (piece == 0) {
    uint32_t extra = vocab;
    if (threadIdx.x < s.head) extra = threadIdx.x;
    else if (threadIdx.x >= 32u && threadIdx.x - 32u < vocab - s.tail0) extra = s.tail0 + (threadIdx.x - 32u);
    if (extra < vocab) g[extra] = from_f32<T>(zero ? 0.0f : ex2((to_f32(z[extra]) - base) * c) * f);
  }
}

template <class T>
__global__ void __launch_bounds__(256) listed_gradient_kernel(const tessa_distill_args a, const DistillPlan plan) {
  const uint64_t at = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  if (at >= a.rows * a.k) return;
  const uint32_t id = plan.ids[at];
  if (id == kNoEntry) return;
  const uint64_t row = at / a.k;
  const Stat st = plan.stats[row];
  const float2 t = plan.terms[at];
  const float c = 1.44269504088896341f / a.temperature;
  const float wt = a.temperature * (a.row_weights ? a.row_weights[row] : 1.0f);
  static_cast<T*>(a.grad)[row * a.grad_stride + id] =
      from_f32<T>(ex2((t.x - base_of(st.m)) * c) * (wt / st.s) - wt * t.y);
}

template <class T, int WARPS>
cudaError_t launch_cluster(const tessa_distill_args& a, const DistillPlan& plan, const AsyncCtx& c,
                           cudaStream_t stream) {
  static SmemRaised raised;
  cudaError_t e = raise_smem(distill_kernel<T, WARPS>, c.device, kSmemMost - 1024, raised);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((uint32_t)(a.rows << plan.cluster_log2));
  cfg.blockDim = dim3((WARPS + 1) * 32);
  cfg.dynamicSmemBytes = list_bytes(a.k) + plan.keep_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1u << plan.cluster_log2;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = plan.cluster_log2 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, distill_kernel<T, WARPS>, a, plan, c.err);
}

// Row bytes from which the gradient is launched apart from the loss: a cluster
// keeps less and less of a row, and re-reads the rest when L2 has lost it.
// 1024 x 1M bf16: 0.96 ms apart, 1.10 by clusters; 512 x 200000: 128 us and 112.
constexpr uint64_t kApart = 1024u << 10;
constexpr uint64_t kKeep = 100u << 10;  // of a slice in shared memory: room for two CTAs an SM

}  // namespace train

uint64_t distill_workspace(uint64_t rows, uint64_t vocab, uint32_t dtype, uint32_t k, bool grad) {
  using namespace train;
  return grad && vocab * type_bytes(dtype) >= kApart ? rows * (sizeof(Stat) + k * 12ull) : 0;
}

cudaError_t launch_distill(const tessa_distill_args& a, void* workspace, const AsyncCtx& c, cudaStream_t stream) {
  using namespace train;
  const uint64_t bytes = a.vocab * type_bytes(a.dtype);
  const bool apart = distill_workspace(a.rows, a.vocab, a.dtype, a.k, a.grad != nullptr) != 0;
  DistillPlan plan = {};
  // The fewest CTAs a row that can keep it (a cluster costs: 2048 x 16384 bf16
  // takes 28 us with one CTA a row, 39 with two), more while rows alone do not
  // fill the GPU.
  while (plan.cluster_log2 < 3 &&
         ((a.grad && !apart && bytes >> plan.cluster_log2 > kKeep) ||
          (a.rows << plan.cluster_log2 < (uint64_t)c.sm_count * 2 && bytes >> plan.cluster_log2 > 16384)))
    ++plan.cluster_log2;
  const uint64_t slice = div_up(bytes, 1ull << plan.cluster_log2) + 16;
  tessa_distill_args first = a;
  if (apart) {
    plan.stats = static_cast<Stat*>(workspace);
    plan.terms = reinterpret_cast<float2*>(plan.stats + a.rows);
    plan.ids = reinterpret_cast<uint32_t*>(plan.terms + a.rows * a.k);
    first.grad = nullptr;
  } else if (a.grad) {
    plan.keep_bytes = (uint32_t)(slice < kKeep ? div_up(slice, 16) * 16 : kKeep);
  }
  return with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    // Short rows leave more warps idle than they occupy: 8192 x 2000 f32 takes
    // 43 us with four warps, 56 with eight.  Where shared memory lets two CTAs
    // stand on an SM, they have 16 each; the loss alone keeps nothing (4096 x
    // 50000 bf16: 70 us with eight, 93 with 16), until rows are so long that a
    // CTA's end no longer counts (1024 x 1M bf16: 347 us with eight, 322 with 16).
    const uint32_t w = slice <= 16384 ? 4 : slice <= 65536 || (!plan.keep_bytes && slice < kApart) ? 8 : 16;
    cudaError_t e = w == 4   ? launch_cluster<T, 4>(first, plan, c, stream)
                    : w == 8 ? launch_cluster<T, 8>(first, plan, c, stream)
                             : launch_cluster<T, 16>(first, plan, c, stream);
    if (e != cudaSuccess || !apart) return e;
    const uint32_t pieces = (uint32_t)div_up(bytes, kPieceVecs * 16u);
    dense_gradient_kernel<T><<<(uint32_t)(a.rows * pieces), 256, 0, stream>>>(a, plan.stats, pieces);
    if (a.k) listed_gradient_kernel<T><<<(uint32_t)div_up(a.rows * a.k, 256), 256, 0, stream>>>(a, plan);
    return cudaGetLastError();
  });
}

}  // namespace tessa

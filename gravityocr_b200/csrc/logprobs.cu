// Log probabilities of given tokens with their rank, the distribution's entropy and its best alternatives, from one pass
// over a row of logits l (fp32 or bf16) at temperature T.
//
// With m = max l, d_v = (l_v - m) / T and the sums over every token but the (first) best one
//   R = sum e^{d_v},  W = sum d_v e^{d_v}:   log p_v = d_v - log1p(R),   H = log1p(R) - W / (1 + R).
// Leaving the best token's own 1 out of R keeps a peaked row exact (its log p is -R, not log(1 + 2^-24 ..)), and both terms
// of H are >= 0, so neither cancels.  A thread keeps (m, R, W) of its elements online, 16 of them at a time: their maximum
// first, then one exponential each; two such states join by scaling the lower one by e^{(m_lo - m_hi) / T} after its own
// best token has joined its sums.
//   rank = 1 + the tokens that come before the given one, by logit, then by id.
// Best n: a thread also keeps its best element.  The n-th best of the bests of 64 groups of threads bounds the row's n-th
// best from below, so only threads whose best reaches the bound look at their elements again (a few KB, from L2), and
// what they find above it is ranked by counting.
// Bound: reading the row.  Few rows are shared between the CTAs of a cluster, whose states, counts and best lists the first
// one joins through distributed shared memory.
#include "params.cuh"

namespace gr {

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpGroups = 64;             // groups of threads whose bests bound the n-th best; n <= kLpGroups
constexpr int kLpCand = 1024;             // candidates kept at once
constexpr int kLpMaxCluster = 8;
constexpr float kLpFloor = -1e20f;        // logits count as at least this: e = 0 there, and (l - m) / T stays finite

struct LpState {
  float m, R, W;  // max logit (-inf: no token yet); sums without the max token, W in units of log2
};

// e^{(a - b) / T} with a <= b; 0 for a = -inf.  k = log2(e) / T.
__device__ __forceinline__ float lp_shift(float a, float b, float k, float& d) {
  d = fmaxf((a - b) * k, -1e30f);  // -1e30 instead of -inf: d * 0 stays 0
  return ex2_approx(d);
}
__device__ __forceinline__ LpState lp_join(const LpState& a, const LpState& b, float k) {
  const bool sw = b.m > a.m;
  const LpState hi = sw ? b : a, lo = sw ? a : b;
  if (lo.m == -INFINITY) {  // the lower one is empty, or every token of it is masked; a NaN in its sums stays
    LpState r = hi;
    r.R += lo.R;
    r.W += lo.W;
    return r;
  }
  float d;
  const float f = lp_shift(lo.m, hi.m, k, d);
  LpState r;
  r.m = hi.m;
  r.R = hi.R + f * (lo.R + 1.f);
  r.W = hi.W + f * (lo.W + (lo.R + 1.f) * d);
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Order of (logit, id) pairs as one integer: higher logit first, then the lower id.  0: no token.
__device__ __forceinline__ uint64_t lp_key(float x, int id) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<uint64_t>(o) << 32) | (0xffffffffu - static_cast<uint32_t>(id));
}
__device__ __forceinline__ int lp_key_id(uint64_t k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ float lp_key_logit(uint64_t k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

// 16 logits of a thread: 16-byte loads raw[], their maximum, and their values raised to kLpFloor (NaNs kept).
template <typename T>
struct LpVec;
template <>
struct LpVec<float> {
  static constexpr int N = 4, B = 4;  // elements per load, loads per batch
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ float get(const uint4& v, int i) {
    return __uint_as_float(i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)));
  }
  static __device__ __forceinline__ float max_of(const uint4& v) {
    return fmaxf(fmaxf(get(v, 0), get(v, 1)), fmaxf(get(v, 2), get(v, 3)));
  }
  static __device__ __forceinline__ void values(const uint4& v, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = max_nan(get(v, i), kLpFloor);
  }
  // how many are >= t
  static __device__ __forceinline__ int count(const uint4& v, float t) {
    return (get(v, 0) >= t) + (get(v, 1) >= t) + (get(v, 2) >= t) + (get(v, 3) >= t);
  }
  // the next larger number of the type
  static __device__ __forceinline__ float next(float x) {
    const int b = __float_as_int(x);
    return __int_as_float(b >= 0 ? b + 1 : b - 1);
  }
};
template <>
struct LpVec<__nv_bfloat16> {
  static constexpr int N = 8, B = 2;
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ float get(const uint4& v, int i) {
    const uint32_t w = (i >> 1) == 0 ? v.x : ((i >> 1) == 1 ? v.y : ((i >> 1) == 2 ? v.z : v.w));
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ __nv_bfloat162 pair(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  static __device__ __forceinline__ float max_of(const uint4& v) {
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(pair(v.x), pair(v.y)), __hmax2(pair(v.z), pair(v.w))));
    return fmaxf(m.x, m.y);
  }
  static __device__ __forceinline__ void values(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 c = __hmax2_nan(pair(w[i]), __float2bfloat162_rn(kLpFloor));
      const uint32_t u = *reinterpret_cast<const uint32_t*>(&c);
      x[2 * i] = __uint_as_float(u << 16);
      x[2 * i + 1] = __uint_as_float(u & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ int count(const uint4& v, float t) {
    const __nv_bfloat162 tt = __float2bfloat162_rn(t);  // t is a bf16 number
    const __nv_bfloat162 n = __hadd2(__hadd2(__hge2(pair(v.x), tt), __hge2(pair(v.y), tt)),
                                     __hadd2(__hge2(pair(v.z), tt), __hge2(pair(v.w), tt)));
    const float2 f = __bfloat1622float2(n);
    return static_cast<int>(f.x + f.y);
  }
  static __device__ __forceinline__ float next(float x) {
    const int b = __float_as_int(x);
    return __int_as_float(b >= 0 ? b + 0x10000 : b - 0x10000);
  }
};

struct LpThread {
  LpState s;
  int best_id;
  int before;  // tokens that come before the given one
};
// One element on its own.
__device__ __forceinline__ void lp_one(LpThread& t, float x, int id, float k, float mine, int my_id) {
  t.before += (x > mine || (x == mine && id < my_id)) ? 1 : 0;
  if (x != x) {
    t.s.R = x;
    return;
  }
  if (x > t.s.m || t.best_id < 0) t.best_id = id;
  if (x == -INFINITY) return;
  LpState e;
  e.m = x;
  e.R = e.W = 0.f;
  t.s = lp_join(t.s, e, k);
}
// A batch of loads, id0[u] the id of load u's first element.  Best tokens below kLpFloor are left to lp_one (see the kernel).
template <typename T>
__device__ __forceinline__ void lp_batch(LpThread& t, const uint4 (&raw)[LpVec<T>::B], const int (&id0)[LpVec<T>::B],
                                         float k, float mine, float mine_next, int my_id) {
  using V = LpVec<T>;
  float x[V::B * V::N];
  float bm = V::max_of(raw[0]);
#pragma unroll
  for (int u = 1; u < V::B; ++u) bm = fmaxf(bm, V::max_of(raw[u]));
#pragma unroll
  for (int u = 0; u < V::B; ++u) V::values(raw[u], x + u * V::N);
  if (bm > t.s.m || t.best_id < 0) {  // a new best token: the old one joins the sums, the new one stays out
    int at = -1;
#pragma unroll
    for (int i = V::B * V::N - 1; i >= 0; --i)
      if (V::get(raw[i / V::N], i % V::N) == bm) at = i;
    if (at >= 0) {
      t.best_id = 0;
#pragma unroll
      for (int u = 0; u < V::B; ++u)
        if (at / V::N == u) t.best_id = id0[u] + at % V::N;
      if (bm > -INFINITY) {
        LpState e;
        e.m = bm;
        e.R = e.W = 0.f;
        t.s = lp_join(t.s, e, k);
#pragma unroll
        for (int i = 0; i < V::B * V::N; ++i)
          if (i == at) x[i] = kLpFloor;
      }
    }
  }
  const float m = t.s.m == -INFINITY ? 0.f : fmaxf(t.s.m, kLpFloor);  // nothing but masked tokens yet: e = 0 for each
#pragma unroll
  for (int i = 0; i < V::B * V::N; ++i) {
    const float d = (x[i] - m) * k;
    const float e = ex2_approx(d);
    t.s.R += e;
    t.s.W = fmaf(e, d, t.s.W);
  }
#pragma unroll
  for (int u = 0; u < V::B; ++u) {
    // tokens before the given one count when equal to it
    if (my_id >= id0[u] && my_id < id0[u] + V::N) {
#pragma unroll
      for (int i = 0; i < V::N; ++i) {
        const float y = V::get(raw[u], i);
        t.before += (y > mine || (y == mine && id0[u] + i < my_id)) ? 1 : 0;
      }
    } else {
      t.before += V::count(raw[u], id0[u] < my_id ? mine : mine_next);
    }
  }
}

__device__ __forceinline__ LpState lp_warp_join(LpState s, float k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    LpState t;
    t.m = __shfl_xor_sync(0xffffffffu, s.m, o);
    t.R = __shfl_xor_sync(0xffffffffu, s.R, o);
    t.W = __shfl_xor_sync(0xffffffffu, s.W, o);
    s = lp_join(s, t, k);
  }
  return s;
}

__device__ __forceinline__ uint32_t lp_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t lp_cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void lp_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint64_t lp_peer_u64(const void* p, uint32_t rank) {
  uint32_t a;
  uint64_t v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}

struct LpPart {  // a CTA's part of the row
  float m, R, W;
  int before;
};

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 2) token_logprobs_kernel(const LogprobParams p) {
  using V = LpVec<T>;
  __shared__ LpState s_state[kLpWarps];
  __shared__ int s_before[kLpWarps];
  __shared__ uint64_t s_group[kLpGroups];
  __shared__ uint64_t s_cand[kLpCand];
  __shared__ uint64_t s_top[kLpGroups];
  __shared__ __align__(16) LpPart s_part;
  __shared__ uint64_t s_bound;
  __shared__ int s_n_cand, s_n_hot;
  __shared__ int s_hot[kLpThreads];
  if (threadIdx.x == 0) pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = lp_cluster_rank(), ctas = lp_cluster_size();
  const int64_t row = blockIdx.x / ctas;
  const T* base = static_cast<const T*>(p.logits) + row * p.ld;
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const float k = 1.4426950408889634f / temp;
  const int64_t want = p.ids[row];
  const bool asked = want >= 0 && want < p.vocab;
  const int my_id = asked ? static_cast<int>(want) : -1;
  const float mine = asked ? V::one(base + my_id) + 0.f : INFINITY;  // + 0: one zero
  const float mine_next = V::next(mine);
  const int n = p.n_top;

  // elements [0, head), vectors, elements [tail, vocab): rows need not start on a 16-byte boundary.  The row's first CTA
  // takes both ends; the vectors are cut evenly.
  const int head = min(p.vocab, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / sizeof(T)));
  const int n_vec = (p.vocab - head) / V::N;
  const int tail = head + n_vec * V::N;
  const uint4* vec = reinterpret_cast<const uint4*>(base + head);
  const int per = (n_vec + static_cast<int>(ctas) - 1) / static_cast<int>(ctas);
  const int v_beg = min(n_vec, static_cast<int>(rank) * per), v_end = min(n_vec, v_beg + per);
  const bool ends = rank == 0;

  LpThread t;
  auto clear = [&] {
    t.s.m = -INFINITY;
    t.s.R = t.s.W = 0.f;
    t.best_id = -1;
    t.before = 0;
  };
  clear();
  if (ends && tid < head) lp_one(t, V::one(base + tid), tid, k, mine, my_id);
  {
    constexpr uint32_t hidden = V::N == 4 ? 0xff800000u : 0xff80ff80u;  // -inf: what a load past the end counts as
    uint4 next[V::B];
    auto load = [&](int v0) {
#pragma unroll
      for (int u = 0; u < V::B; ++u) {
        const int v = v0 + u * kLpThreads;
        next[u] = v < v_end ? __ldg(vec + v) : make_uint4(hidden, hidden, hidden, hidden);
      }
    };
    load(v_beg + tid);
    for (int v0 = v_beg + tid; v0 < v_end; v0 += V::B * kLpThreads) {
      uint4 raw[V::B];
      int id0[V::B];
#pragma unroll
      for (int u = 0; u < V::B; ++u) {
        const int v = v0 + u * kLpThreads;
        raw[u] = next[u];
        id0[u] = v < v_end ? head + v * V::N : 0x7fff0000;
      }
      load(v0 + V::B * kLpThreads);
      lp_batch<T>(t, raw, id0, k, mine, mine_next, my_id);
    }
  }
  if (ends && tail + tid < p.vocab) lp_one(t, V::one(base + tail + tid), tail + tid, k, mine, my_id);
  if (__syncthreads_or(t.s.m < 0.1f * kLpFloor && t.s.m > -INFINITY)) {
    // a thread's best logit lies near or below the floor (a mask of the type's lowest value, say): one by one
    clear();
    if (ends && tid < head) lp_one(t, V::one(base + tid), tid, k, mine, my_id);
    for (int v = v_beg + tid; v < v_end; v += kLpThreads)
      for (int i = 0; i < V::N; ++i) {
        const int id = head + v * V::N + i;
        lp_one(t, V::one(base + id), id, k, mine, my_id);
      }
    if (ends && tail + tid < p.vocab) lp_one(t, V::one(base + tail + tid), tail + tid, k, mine, my_id);
  }

  // this CTA's state and rank count, and the bests of its groups of threads
  const LpState ws = lp_warp_join(t.s, k);
  const int wb = __reduce_add_sync(0xffffffffu, t.before);
  if (lane == 0) {
    s_state[warp] = ws;
    s_before[warp] = wb;
  }
  const uint64_t my_best = t.best_id >= 0 ? lp_key(t.s.m, t.best_id) : 0;
  if (tid == 0) s_n_cand = s_n_hot = 0;
  if (tid < kLpGroups) s_top[tid] = 0;
  uint64_t gb = my_best;
#pragma unroll
  for (int o = kLpThreads / kLpGroups / 2; o > 0; o >>= 1) gb = max(gb, __shfl_xor_sync(0xffffffffu, gb, o));
  if (tid % (kLpThreads / kLpGroups) == 0) s_group[tid / (kLpThreads / kLpGroups)] = gb;
  __syncthreads();
  if (warp == kLpWarps - 1) {
    LpState x;
    x.m = -INFINITY;
    x.R = x.W = 0.f;
    if (lane < kLpWarps) x = s_state[lane];
    x = lp_warp_join(x, k);
    const int before = __reduce_add_sync(0xffffffffu, lane < kLpWarps ? s_before[lane] : 0);
    if (lane == 0) {
      s_part.m = x.m;
      s_part.R = x.R;
      s_part.W = x.W;
      s_part.before = before;
    }
  }
  if (n > 0) {
    // the n-th best of the groups' bests
    if (tid < kLpGroups) {
      const uint64_t mineg = s_group[tid];
      int above = 0;
#pragma unroll 16
      for (int i = 0; i < kLpGroups; ++i) above += (s_group[i] > mineg || (s_group[i] == mineg && i < tid)) ? 1 : 0;
      if (above == n - 1) s_bound = mineg;
    }
    __syncthreads();
    uint64_t bound = max(s_bound, static_cast<uint64_t>(1));
    if (my_best >= bound) s_hot[atomicAdd(&s_n_hot, 1)] = tid;
    __syncthreads();
    const int n_hot = s_n_hot;
    while (true) {
      for (int i = warp; i < n_hot; i += kLpWarps) {
        const int h = s_hot[i];
        auto put = [&](float x, int id) {
          const uint64_t key = lp_key(x, id);
          if (x == x && key >= bound) {
            const int at = atomicAdd(&s_n_cand, 1);
            if (at < kLpCand) s_cand[at] = key;
          }
        };
        if (ends && lane == 0 && h < head) put(V::one(base + h), h);
        if (ends && lane == 0 && tail + h < p.vocab) put(V::one(base + tail + h), tail + h);
        for (int v = v_beg + h + lane * kLpThreads; v < v_end; v += 32 * kLpThreads) {
          const uint4 raw = __ldg(vec + v);
#pragma unroll
          for (int e = 0; e < V::N; ++e) put(V::get(raw, e), head + v * V::N + e);
        }
      }
      __syncthreads();
      const int found = s_n_cand;
      const int kept = min(found, kLpCand);
      // rank by counting; keys are distinct
      for (int i = tid; i < kept; i += kLpThreads) {
        const uint64_t key = s_cand[i];
        int above = 0;
        for (int j = 0; j < kept; ++j) above += s_cand[j] > key ? 1 : 0;
        if (found <= kLpCand) {
          if (above < n) s_top[above] = key;
        } else if (above == n - 1) {
          s_bound = key;  // too many: the n-th best of those kept is a higher bound; look again
        }
      }
      __syncthreads();
      if (found <= kLpCand) break;
      bound = s_bound;
      if (tid == 0) s_n_cand = 0;
      __syncthreads();
    }
  } else {
    __syncthreads();
  }

  // the row: its first CTA joins the parts
  if (ctas > 1) {
    lp_cluster_sync();
    if (rank != 0) {
      lp_cluster_sync();  // this CTA's shared memory is read until here
      return;
    }
  }
  LpState s;
  s.m = s_part.m;
  s.R = s_part.R;
  s.W = s_part.W;
  int before = s_part.before;
  for (uint32_t c = 1; c < ctas; ++c) {
    const uint64_t a = lp_peer_u64(&s_part, c), b = lp_peer_u64(&s_part.W, c);
    LpState x;
    x.m = __uint_as_float(static_cast<uint32_t>(a));
    x.R = __uint_as_float(static_cast<uint32_t>(a >> 32));
    x.W = __uint_as_float(static_cast<uint32_t>(b));
    before += static_cast<int>(b >> 32);
    s = lp_join(s, x, k);
  }
  const bool ok = s.m > -INFINITY && s.m < INFINITY && s.R == s.R && temp > 0.f;
  const float lse = log1pf(s.R);
  const float nan = __int_as_float(0x7fc00000);
  if (tid == 0) {
    const bool known = ok && asked;
    p.logprob[row] = known ? (mine - s.m) / temp - lse : nan;
    p.rank[row] = known ? before + 1 : 0;
    p.entropy[row] = ok ? lse - s.W * 0.69314718055994531f / (1.f + s.R) : nan;
    if (!ok) report(p.status, temp > 0.f ? GR_ERR_NO_TOKEN : GR_ERR_ARG);
    else if (!asked && want != -1) report(p.status, GR_ERR_BAD_ID);
  }
  float* top = p.top_logprob + row * n;
  int32_t* top_ids = p.top_ids + row * n;
  auto put_top = [&](int at, uint64_t key) {
    top[at] = ok ? (lp_key_logit(key) - s.m) / temp - lse : nan;
    top_ids[at] = ok ? lp_key_id(key) : -1;
  };
  if (ctas == 1) {
    if (tid < n) put_top(tid, s_top[tid]);
  } else {
    const int total = n * static_cast<int>(ctas);  // at most kLpGroups * kLpMaxCluster = kLpThreads keys
    const uint64_t key = tid < total ? lp_peer_u64(&s_top[tid % n], tid / n) : 0;
    __syncwarp();
    lp_cluster_sync();
    if (tid < total) s_cand[tid] = key;
    __syncthreads();
    if (tid < total && (key || !ok)) {
      int above = 0;
      for (int j = 0; j < total; ++j) above += (s_cand[j] > key || (s_cand[j] == key && j < tid)) ? 1 : 0;
      if (above < n) put_top(above, key);
    }
  }
}

cudaError_t launch_token_logprobs(const LogprobParams& p, bool bf16, cudaStream_t stream, bool pdl) {
  // CTAs a row: as many as keep the launch within two CTAs an SM
  int ctas = 1;
  while (ctas < kLpMaxCluster && p.rows * ctas * 2 <= 2 * p.sms) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.rows * ctas);
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return bf16 ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<__nv_bfloat16>, p)
              : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<float>, p);
}

}  // namespace gr

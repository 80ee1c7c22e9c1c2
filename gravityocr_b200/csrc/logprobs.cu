// Log probabilities of given tokens with their rank, the distribution's entropy and its best alternatives, from one pass
// over a row of logits l (fp32 or bf16) at temperature T.
//
// With m = max l, d_v = (l_v - m) / T and the sums over every token but the (first) best one
//   R = sum e^{d_v},  W = sum d_v e^{d_v}:   log p_v = d_v - log1p(R),   H = log1p(R) - W / (1 + R).
// Leaving the best token's own 1 out of R keeps a peaked row exact (its log p is -R, not log(1 + 2^-24 ..)), and both terms
// of H are >= 0, so neither cancels.
//
// Stream: a thread sums e^{(l - ref) / T} and its product with the exponent, 16 logits at a time, against a reference of its
// own that moves only when a batch's maximum is 2^24 above it; it keeps its largest logit, and counts the tokens that come
// before the given one (rank = 1 + those, by logit, then by id).  About nine instructions a logit; a running maximum with
// its token left out on the way cost twice that.  At the end the thread that holds the best token is left out of the
// sums, and a warp reads that thread's logits again (they are in L2) to sum them without it.
// Best n: every batch's maximum goes to a cell in shared memory (a thread's batches share 16).  The n-th largest of the largest
// logits of 64 groups of threads bounds the row's n-th best from below, so only cells that reach the bound are read
// again, and what is found above it is ranked by counting.  (Cells, not threads, because 592 rows in flight outgrow the L2:
// reading every such thread's logits again cost 20% more DRAM traffic.)
// Bound: reading the row (1,088 rows of 59,392 fp32 logits, the 20 best: 51 us, 55 on another machine; 258 MB, 5.0 TB/s; bf16:
// 45 us, by its instructions).  Few rows (64 bf16: 12 us, one: 9) wait for the chain of phases: stream, maxima, bound, cells,
// ranks.  They are shared between the CTAs of a cluster, whose states, counts and best lists the first one joins through
// distributed shared memory.  Rows with fewer tokens than alternatives are slow, since every masked token is a candidate (three
// of 59,392 left, the 20 best: one row 64 us, 1,088 rows 446).
#include <type_traits>

#include "params.cuh"

namespace gr {

constexpr int kLpMaxThreads = 512;
constexpr int kLpGroups = 64;             // groups of threads whose bests bound the n-th best; n <= kLpGroups
constexpr int kLpCand = 1024;             // candidates kept at once
constexpr uint32_t kLpAhead = 48 << 10;   // bytes of a later row fetched to L2 while this one is finished
constexpr int kLpCells = 16;              // cells of a thread: batch i counts in cell i % kLpCells
constexpr int kLpHot = 512;               // cells read again one by one; more (ties) and every thread scans its own logits
constexpr int kLpMaxCluster = 8;

struct LpState {
  float m, R, W;  // max logit (-inf: no token yet); sums without the max token, W in units of log2
};

// e^{(a - b) / T} with a <= b; 0 for a = -inf.  k = log2(e) / T.
__device__ __forceinline__ float lp_shift(float a, float b, float k, float& d) {
  d = fmaxf((a - b) * k, -1e20f);  // -1e20 instead of -inf: times any sum it stays a number
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
__device__ __forceinline__ float lp_warp_max(float v) {
  float r;
  // NaNs are ignored; volatile: every lane has to take part, wherever the result is used
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Order of logits as integers (one zero), and of (logit, id) pairs: higher logit first, then the lower id.  0: no token.
__device__ __forceinline__ uint32_t lp_order(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ uint64_t lp_key(float x, int id) {
  return (static_cast<uint64_t>(lp_order(x)) << 32) | (0xffffffffu - static_cast<uint32_t>(id));
}
__device__ __forceinline__ int lp_key_id(uint64_t k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ float lp_key_logit(uint64_t k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

// Two fp32 numbers in a register pair (add, mul and fma take both at once).
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// A 16-byte load of logits: its elements, their maximum (NaNs ignored), and how many are >= t.
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
  float ref, S, W;  // reference logit (-inf: none yet), sum of e = 2^d, sum of e d, d = (l - ref) k
  float best;       // largest logit
  int before;       // tokens that come before the given one
};
constexpr float kLpRaise = 24.f;
// The sums of a thread or a warp seen from another reference, at or above its own.
__device__ __forceinline__ void lp_move(float& S, float& W, float ref, float to, float k) {
  if (ref == -INFINITY) return;  // nothing yet (or NaN, which stays)
  float d;
  const float f = lp_shift(ref, to, k, d);
  W = f * fmaf(S, d, W);
  S *= f;
}
__device__ __forceinline__ void lp_add(float x, float ref, float k, float& S, float& W) {
  const float d = max_nan((x - ref) * k, -1e20f);  // a masked token: e = 0, and e d = 0 stays a number
  const float e = ex2_approx(d);
  S += e;
  W = fmaf(e, d, W);
}
__device__ __forceinline__ void lp_raise(LpThread& t, float bm, float k) {
  if (bm == -INFINITY || (bm - t.ref) * k <= kLpRaise) return;
  lp_move(t.S, t.W, t.ref, bm, k);
  t.ref = bm;
}
// One element on its own.
__device__ __forceinline__ void lp_one(LpThread& t, float x, int id, float k, float mine, int my_id) {
  t.before += (x > mine || (x == mine && id < my_id)) ? 1 : 0;
  t.best = fmaxf(t.best, x);
  lp_raise(t, x, k);
  lp_add(x, t.ref == -INFINITY ? 0.f : t.ref, k, t.S, t.W);
}
// A batch of loads NT apart, id0 the id of the first one's first element; the first `valid` hold logits, the rest
// -inf, which adds nothing to the sums and must not be counted.  Returns the batch's maximum.
template <typename T, int NT>
__device__ __forceinline__ float lp_batch(LpThread& t, const uint4 (&raw)[LpVec<T>::B], int id0, int valid, float k,
                                          float mine, float mine_next, int my_id) {
  using V = LpVec<T>;
  float bm = V::max_of(raw[0]);
#pragma unroll
  for (int u = 1; u < V::B; ++u) bm = fmaxf(bm, V::max_of(raw[u]));
  t.best = fmaxf(t.best, bm);
  lp_raise(t, bm, k);
  const float ref = t.ref == -INFINITY ? 0.f : t.ref;  // nothing but masked tokens yet: e = 0 for each
  const uint64_t kk = f2_pack(k, k), minus = f2_pack(-ref, -ref);
  uint64_t S2 = f2_pack(t.S, 0.f), W2 = f2_pack(t.W, 0.f);
#pragma unroll
  for (int u = 0; u < V::B; ++u)
#pragma unroll
    for (int i = 0; i < V::N; i += 2) {
      float d0, d1;
      f2_unpack(f2_mul(f2_add(f2_pack(V::get(raw[u], i), V::get(raw[u], i + 1)), minus), kk), d0, d1);
      d0 = max_nan(d0, -1e20f);  // a masked token: e = 0, and e d = 0 stays a number
      d1 = max_nan(d1, -1e20f);
      const uint64_t e = f2_pack(ex2_approx(d0), ex2_approx(d1));
      S2 = f2_add(S2, e);
      W2 = f2_fma(e, f2_pack(d0, d1), W2);
    }
  float a, b;
  f2_unpack(S2, a, b);
  t.S = a + b;
  f2_unpack(W2, a, b);
  t.W = a + b;
  // tokens before the given one count when equal to it
  if (my_id < id0 || my_id >= id0 + (V::B - 1) * NT * V::N + V::N) {
    const float least = my_id < id0 ? mine_next : mine;
#pragma unroll
    for (int u = 0; u < V::B; ++u)
      if (u < valid) t.before += V::count(raw[u], least);
  } else {
#pragma unroll
    for (int u = 0; u < V::B; ++u)
#pragma unroll
      for (int i = 0; i < V::N; ++i) {
        const float y = V::get(raw[u], i);
        t.before += u < valid && (y > mine || (y == mine && id0 + u * NT * V::N + i < my_id)) ? 1 : 0;
      }
  }
  return bm;
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

template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) token_logprobs_kernel(const LogprobParams p) {
  using V = LpVec<T>;
  constexpr int kWarps = NT / 32;
  __shared__ float s_max[kWarps], s_S[kWarps], s_W[kWarps];
  __shared__ int s_before[kWarps];
  __shared__ uint32_t s_group[kLpGroups];
  __shared__ uint64_t s_cand[kLpCand];
  __shared__ uint64_t s_top[kLpGroups];
  __shared__ __align__(16) LpPart s_part;
  __shared__ uint64_t s_bound;
  __shared__ int s_n_cand, s_n_hot, s_arg;
  __shared__ uint16_t s_hot[kLpHot];
  __shared__ float s_cell[kLpCells][NT];
  if (threadIdx.x == 0) pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = lp_cluster_rank(), ctas = lp_cluster_size();
  const int64_t row = blockIdx.x / ctas;
  const T* base = static_cast<const T*>(p.logits) + row * p.ld;
  // elements [0, head), vectors, elements [tail, vocab): rows need not start on a 16-byte boundary.  The row's first CTA
  // takes both ends; the vectors are cut evenly.
  const int head = min(p.vocab, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / sizeof(T)));
  const int n_vec = (p.vocab - head) / V::N;
  const int tail = head + n_vec * V::N;
  const uint4* vec = reinterpret_cast<const uint4*>(base + head);
  const int per = (n_vec + static_cast<int>(ctas) - 1) / static_cast<int>(ctas);
  const int v_beg = min(n_vec, static_cast<int>(rank) * per), v_end = min(n_vec, v_beg + per);
  const bool ends = rank == 0;

  // the first loads of the stream, then what the sums need: the given token's logit is two latencies away
  constexpr int step = V::B * NT;
  uint4 next[V::B];
  const bool full = v_beg + tid + step - NT < v_end;
  if (full) {
#pragma unroll
    for (int u = 0; u < V::B; ++u) next[u] = __ldg(vec + v_beg + tid + u * NT);
  }
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const bool warm = temp >= 0x1p-126f;  // (log2(e) / T is finite for normal T)
  const float k = fmaxf(1.4426950408889634f / temp, 1e-45f);  // above 0 for T = inf, too: a masked token's -inf stays -inf
  const int64_t want = p.ids[row];
  const bool asked = want >= 0 && want < p.vocab;
  const int my_id = asked ? static_cast<int>(want) : -1;
  const float mine = asked ? V::one(base + my_id) + 0.f : INFINITY;  // + 0: one zero
  const float mine_next = V::next(mine);
  const int n = p.n_top;
  if (tid == 0) {
    s_n_cand = s_n_hot = 0;
    s_arg = NT;
    s_bound = 1;
  }
  LpThread t;
  t.ref = t.best = -INFINITY;
  t.S = t.W = 0.f;
  t.before = 0;
  if (ends && tid < head) lp_one(t, V::one(base + tid), tid, k, mine, my_id);
  {
    constexpr uint32_t hidden = V::N == 4 ? 0xff800000u : 0xff80ff80u;  // -inf: what a load past the end counts as
    int v0 = v_beg + tid, i = 0;
    auto cell = [&](float bm) {
      float& c = s_cell[i % kLpCells][tid];
      c = i < kLpCells ? bm : fmaxf(c, bm);
      ++i;
    };
    // full batches, the next one's loads in flight; then the rest
    for (; v0 + step - NT < v_end; v0 += step) {
      uint4 raw[V::B];
#pragma unroll
      for (int u = 0; u < V::B; ++u) raw[u] = next[u];
      const int ahead = v0 + 2 * step - NT < v_end ? v0 + step : v0;  // the last batch loads itself again
#pragma unroll
      for (int u = 0; u < V::B; ++u) next[u] = __ldg(vec + ahead + u * NT);
      cell(lp_batch<T, NT>(t, raw, head + v0 * V::N, V::B, k, mine, mine_next, my_id));
    }
    if (v0 < v_end) {
      uint4 raw[V::B];
#pragma unroll
      for (int u = 0; u < V::B; ++u) {
        const int v = v0 + u * NT;
        raw[u] = v < v_end ? __ldg(vec + v) : make_uint4(hidden, hidden, hidden, hidden);
      }
      cell(lp_batch<T, NT>(t, raw, head + v0 * V::N, (v_end - v0 + NT - 1) / NT, k, mine, mine_next, my_id));
    }
  }
  if (ends && tail + tid < p.vocab) lp_one(t, V::one(base + tail + tid), tail + tid, k, mine, my_id);
  if (NT < kLpMaxThreads && tid == 0 && row + p.ahead < p.rows) {
    // CTAs that started together reach their selection together: meanwhile the row that will follow on this SM comes to L2
    const T* after = base + p.ahead * p.ld;
    const uintptr_t from = (reinterpret_cast<uintptr_t>(after) + 15) & ~uintptr_t(15);
    const uintptr_t bytes = (reinterpret_cast<uintptr_t>(after + p.vocab) - from) & ~uintptr_t(15);
    if (reinterpret_cast<uintptr_t>(after + p.vocab) > from + 16)
      l2_prefetch(reinterpret_cast<const void*>(from), static_cast<uint32_t>(bytes < kLpAhead ? bytes : kLpAhead));
  }
  const bool any = v_beg + tid < v_end || (ends && (tid < head || tail + tid < p.vocab));
  const uint32_t my_best = any ? lp_order(t.best) : 0;

  // the part's largest logit, the thread that holds it (one of those that do), the groups' largest
  const float wm = lp_warp_max(t.best);
  if (lane == 0) s_max[warp] = wm;
  if (tid < kLpGroups) s_top[tid] = 0;
  uint32_t gb = my_best;
#pragma unroll
  for (int o = NT / kLpGroups / 2; o > 0; o >>= 1) gb = max(gb, __shfl_xor_sync(0xffffffffu, gb, o));
  if (tid % (NT / kLpGroups) == 0) s_group[tid / (NT / kLpGroups)] = gb;
  __syncthreads();
  const float m = lp_warp_max(s_max[lane % kWarps]);
  if (any && t.best == m) atomicMin(&s_arg, tid);
  if (n > 0 && tid < kLpGroups) {
    // the n-th largest of the groups'
    const uint32_t mineg = s_group[tid];
    int above = 0;
#pragma unroll 16
    for (int i = 0; i < kLpGroups; ++i) above += (s_group[i] > mineg || (s_group[i] == mineg && i < tid)) ? 1 : 0;
    if (above == n - 1 && mineg) s_bound = static_cast<uint64_t>(mineg) << 32;
  }
  __syncthreads();
  const int arg = s_arg;
  uint64_t bound = s_bound;
  // sums from m: every thread's but the best token's own, which one warp makes anew without that token
  if (tid == arg && m > -INFINITY) t.S = t.W = 0.f;
  else lp_move(t.S, t.W, t.ref, m, k);
  const float S = warp_sum(t.S), W = warp_sum(t.W);
  const int wb = __reduce_add_sync(0xffffffffu, t.before);
  if (lane == 0) {
    s_S[warp] = S;
    s_W[warp] = W;
    s_before[warp] = wb;
  }
  if (n > 0 && v_beg + tid < v_end && (static_cast<uint64_t>(my_best) << 32 | 0xffffffffu) >= bound) {
    const int cells = min(kLpCells, (v_end - v_beg - tid + V::B * NT - 1) / (V::B * NT));
#pragma unroll
    for (int c = 0; c < kLpCells; ++c)
      if (c < cells && (static_cast<uint64_t>(lp_order(s_cell[c][tid])) << 32 | 0xffffffffu) >= bound) {
        const int at = atomicAdd(&s_n_hot, 1);
        if (at < kLpHot) s_hot[at] = static_cast<uint16_t>(c * NT + tid);
      }
  }
  __syncthreads();
  if (warp == 0) {
    float R = 0.f, Wx = 0.f;
    int equal = 0;
    if (m > -INFINITY) {
      auto add = [&](float x) {
        if (x == m) ++equal;
        else lp_add(x, m, k, R, Wx);
      };
      if (ends && lane == 0 && arg < head) add(V::one(base + arg));
      if (ends && lane == 0 && tail + arg < p.vocab) add(V::one(base + tail + arg));
      for (int v = v_beg + arg + lane * NT; v < v_end; v += 32 * NT) {
        const uint4 raw = __ldg(vec + v);
#pragma unroll
        for (int e = 0; e < V::N; ++e) add(V::get(raw, e));
      }
    }
    if (lane < kWarps) {
      R += s_S[lane];
      Wx += s_W[lane];
    }
    R = warp_sum(R);
    Wx = warp_sum(Wx);
    equal = __reduce_add_sync(0xffffffffu, equal);
    const int before = __reduce_add_sync(0xffffffffu, lane < kWarps ? s_before[lane] : 0);
    if (lane == 0) {
      s_part.m = m;
      s_part.R = R + (equal > 1 ? static_cast<float>(equal - 1) : 0.f);
      s_part.W = Wx;
      s_part.before = before;
    }
  }
  if (n > 0) {
    const int n_hot = s_n_hot;
    while (true) {
      auto put = [&](float x, int id) {
        const uint64_t key = lp_key(x, id);
        if (x == x && key >= bound) {
          const int at = atomicAdd(&s_n_cand, 1);
          if (at < kLpCand) s_cand[at] = key;
        }
      };
      auto put_vec = [&](int v) {
        const uint4 raw = __ldg(vec + v);
#pragma unroll
        for (int e = 0; e < V::N; ++e) put(V::get(raw, e), head + v * V::N + e);
      };
      if (ends && tid < head) put(V::one(base + tid), tid);
      if (ends && tail + tid < p.vocab) put(V::one(base + tail + tid), tail + tid);
      if (n_hot <= kLpHot) {
        // V::B lanes a cell: the loads of its batches
        for (int i = tid / V::B; i < n_hot; i += NT / V::B) {
          const int h = s_hot[i];
          for (int v = v_beg + h % NT + (h / NT * V::B + tid % V::B) * NT; v < v_end; v += kLpCells * V::B * NT) put_vec(v);
        }
      } else {
        for (int v = v_beg + tid; v < v_end; v += NT) put_vec(v);
      }
      __syncthreads();
      const int found = s_n_cand;
      const int kept = min(found, kLpCand);
      // rank by counting; keys are distinct
      for (int i = tid; i < kept; i += NT) {
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
  const bool ok = s.m > -INFINITY && s.m < INFINITY && s.R == s.R && warm;
  const float lse = log1pf(s.R);
  const float nan = __int_as_float(0x7fc00000);
  auto log_p = [&](float x) { return x == -INFINITY ? x : (x - s.m) / temp - lse; };
  if (tid == 0) {
    const bool known = ok && asked;
    p.logprob[row] = known ? log_p(mine) : nan;
    p.rank[row] = known ? before + 1 : 0;
    p.entropy[row] = ok ? lse - s.W * 0.69314718055994531f / (1.f + s.R) : nan;
    if (!ok) report(p.status, warm ? GR_ERR_NO_TOKEN : GR_ERR_ARG);
    else if (!asked && want != -1) report(p.status, GR_ERR_BAD_ID);
  }
  float* top = p.top_logprob + row * n;
  int32_t* top_ids = p.top_ids + row * n;
  auto put_top = [&](int at, uint64_t key) {
    top[at] = ok ? log_p(lp_key_logit(key)) : nan;
    top_ids[at] = ok ? lp_key_id(key) : -1;
  };
  if (ctas == 1) {
    if (tid < n) put_top(tid, s_top[tid]);
  } else {
    // at most kLpGroups * kLpMaxCluster keys: clusters come with as many threads
    const int total = n * static_cast<int>(ctas);
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

template <typename T, int NT>
static cudaError_t launch_token_logprobs_t(const LogprobParams& p, int ctas, cudaStream_t stream, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * ctas);
  cfg.blockDim = dim3(NT);
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
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, NT>, p);
}

// 1,024 threads an SM, in CTAs of 512, 256 or 128, a CTA a row: as many rows in flight as there are, since a row's
// selection (about 6 us) leaves the memory to the other rows' reading.  Rows of 59,392 fp32 logits in CTAs of 128, 256 and 512:
// 1,088 rows 51, 57 and 67 us; 580 rows 39, 31 and 36; 290 rows 36, 25 and 19 (just past a border the larger CTAs would still
// be better: 600 rows 50 and 44).  Fewer rows than SMs are shared by clusters.
cudaError_t launch_token_logprobs(LogprobParams p, bool bf16, cudaStream_t stream, bool pdl) {
  auto go = [&](auto nt, int ctas) {
    constexpr int NT = decltype(nt)::value;
    p.ahead = 1024 / NT * p.sms;
    return bf16 ? launch_token_logprobs_t<__nv_bfloat16, NT>(p, ctas, stream, pdl)
                : launch_token_logprobs_t<float, NT>(p, ctas, stream, pdl);
  };
  if (p.rows > 4 * p.sms) return go(std::integral_constant<int, 128>(), 1);
  if (p.rows > 2 * p.sms) return go(std::integral_constant<int, 256>(), 1);
  int ctas = 1;
  while (ctas < kLpMaxCluster && static_cast<int64_t>(p.rows) * ctas <= p.sms) ctas *= 2;
  return go(std::integral_constant<int, kLpMaxThreads>(), ctas);
}

}  // namespace gr

// Log probabilities of given tokens with their rank, the distribution's entropy and its best alternatives, from one pass
// over a row of logits l (fp32 or bf16) at temperature T.
//
// With m = max l, d_v = (l_v - m) / T and the sums over every token but the (first) best one
//   R = sum e^{d_v},  W = sum d_v e^{d_v}:   log p_v = d_v - log1p(R),   H = log1p(R) - W / (1 + R).
// Leaving the best token's own 1 out of R keeps a peaked row exact (its log p is -R, not log(1 + 2^-24 ..)), and both terms
// of H are >= 0, so neither cancels.  A thread keeps (m, R, W) of its elements online; two such states join by scaling
// the lower one by e^{(m_lo - m_hi) / T} after its own best token has joined its sums.
//   rank = 1 + the tokens that come before the given one, by logit, then by id.
// Best n: a thread also keeps its best element.  The n-th best of the bests of 64 groups of threads bounds the row's n-th
// best from below, so only threads whose best reaches the bound look at their elements again (a few KB, from L2), and
// what they find above it is ranked by counting.
#include "params.cuh"

namespace gr {

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpGroups = 64;             // groups of threads whose bests bound the n-th best; n <= kLpGroups
constexpr int kLpCand = 1024;             // candidates kept at once
constexpr int kLpBatch = 4;               // 16-byte loads in flight per thread

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

template <typename T>
struct LpVec;  // 16 bytes of logits
template <>
struct LpVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(const uint4& v, int i) {
    return __uint_as_float(i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)));
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
};
template <>
struct LpVec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(const uint4& v, int i) {
    const uint32_t w = (i >> 1) == 0 ? v.x : ((i >> 1) == 1 ? v.y : ((i >> 1) == 2 ? v.z : v.w));
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
};

struct LpThread {
  LpState s;
  int best_id;
  int before;  // tokens that come before the given one
};
// One element on its own (row ends, candidates of a vector that holds the given token).
__device__ __forceinline__ void lp_one(LpThread& t, float x, int id, float k, float mine, int my_id) {
  t.before += (x > mine || (x == mine && id < my_id)) ? 1 : 0;
  LpState e;
  e.m = x;
  e.R = e.W = 0.f;
  if (x != x) {
    t.s.R = x;
    return;
  }
  if (x > t.s.m || t.best_id < 0) t.best_id = id;
  if (x != -INFINITY) t.s = lp_join(t.s, e, k);
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

template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const LogprobParams p) {
  using V = LpVec<T>;
  __shared__ LpState s_state[kLpWarps];
  __shared__ int s_before[kLpWarps];
  __shared__ uint64_t s_best[kLpThreads];
  __shared__ uint64_t s_group[kLpGroups];
  __shared__ uint64_t s_cand[kLpCand];
  __shared__ uint64_t s_bound;
  __shared__ int s_n_cand, s_n_hot;
  __shared__ int s_hot[kLpThreads];
  if (threadIdx.x == 0) pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x;
  const T* base = static_cast<const T*>(p.logits) + row * p.ld;
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const float k = 1.4426950408889634f / temp;
  const int64_t want = p.ids[row];
  const bool asked = want >= 0 && want < p.vocab;
  const int my_id = asked ? static_cast<int>(want) : -1;
  const float mine = asked ? V::one(base + my_id) : INFINITY;

  // elements [0, head), vectors, elements [tail, vocab): rows need not start on a 16-byte boundary
  const int head = min(p.vocab, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / sizeof(T)));
  const int n_vec = (p.vocab - head) / V::N;
  const int tail = head + n_vec * V::N;
  const uint4* vec = reinterpret_cast<const uint4*>(base + head);

  LpThread t;
  t.s.m = -INFINITY;
  t.s.R = t.s.W = 0.f;
  t.best_id = -1;
  t.before = 0;
  if (tid < head) lp_one(t, V::one(base + tid), tid, k, mine, my_id);
  for (int v0 = tid; v0 < n_vec; v0 += kLpBatch * kLpThreads) {
    uint4 raw[kLpBatch];
#pragma unroll
    for (int u = 0; u < kLpBatch; ++u)
      if (v0 + u * kLpThreads < n_vec) raw[u] = __ldg(vec + v0 + u * kLpThreads);
#pragma unroll
    for (int u = 0; u < kLpBatch; ++u) {
      const int v = v0 + u * kLpThreads;
      if (v >= n_vec) break;
      const int id0 = head + v * V::N;
#pragma unroll
      for (int i = 0; i < V::N; ++i) lp_one(t, V::get(raw[u], i), id0 + i, k, mine, my_id);
    }
  }
  if (tail + tid < p.vocab) lp_one(t, V::one(base + tail + tid), tail + tid, k, mine, my_id);

  // the row's state, its rank count, and the threads' bests
  const LpState ws = lp_warp_join(t.s, k);
  const int wb = __reduce_add_sync(0xffffffffu, t.before);
  if (lane == 0) {
    s_state[warp] = ws;
    s_before[warp] = wb;
  }
  const uint64_t my_best = t.best_id >= 0 ? lp_key(t.s.m, t.best_id) : 0;
  s_best[tid] = my_best;
  if (tid == 0) s_n_cand = s_n_hot = 0;
  uint64_t gb = my_best;
#pragma unroll
  for (int o = kLpThreads / kLpGroups / 2; o > 0; o >>= 1) gb = max(gb, __shfl_xor_sync(0xffffffffu, gb, o));
  if (tid % (kLpThreads / kLpGroups) == 0) s_group[tid / (kLpThreads / kLpGroups)] = gb;
  __syncthreads();
  LpState s;
  {
    LpState x;
    x.m = -INFINITY;
    x.R = x.W = 0.f;
    if (lane < kLpWarps) x = s_state[lane];
    s = lp_warp_join(x, k);
  }
  const bool ok = s.m > -INFINITY && s.m < INFINITY && s.R == s.R && temp > 0.f;
  const float lse = log1pf(s.R);
  if (tid == 0) {
    int before = 0;
    for (int w = 0; w < kLpWarps; ++w) before += s_before[w];
    const float nan = __int_as_float(0x7fc00000);
    const bool known = ok && asked;
    p.logprob[row] = known ? (mine - s.m) / temp - lse : nan;
    p.rank[row] = known ? before + 1 : 0;
    p.entropy[row] = ok ? lse - s.W * 0.69314718055994531f / (1.f + s.R) : nan;
    if (!ok) report(p.status, temp > 0.f ? GR_ERR_NO_TOKEN : GR_ERR_ARG);
    else if (!asked && want != -1) report(p.status, GR_ERR_BAD_ID);
  }
  const int n = p.n_top;
  if (n <= 0) return;
  float* top = p.top_logprob + row * n;
  int32_t* top_ids = p.top_ids + row * n;
  if (!ok) {
    for (int i = tid; i < n; i += kLpThreads) {
      top[i] = __int_as_float(0x7fc00000);
      top_ids[i] = -1;
    }
    return;
  }
  // the n-th best of the groups' bests
  if (tid < kLpGroups) {
    const uint64_t mineg = s_group[tid];
    int above = 0;
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
      if (lane == 0 && h < head) put(V::one(base + h), h);
      if (lane == 0 && tail + h < p.vocab) put(V::one(base + tail + h), tail + h);
      for (int v = h + lane * kLpThreads; v < n_vec; v += 32 * kLpThreads) {
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
        if (above < n) {
          top[above] = (lp_key_logit(key) - s.m) / temp - lse;
          top_ids[above] = lp_key_id(key);
        }
      } else if (above == n - 1) {
        s_bound = key;  // too many: the n-th best of those kept is a higher bound; look again
      }
    }
    if (found <= kLpCand) break;
    __syncthreads();
    bound = s_bound;
    if (tid == 0) s_n_cand = 0;
    __syncthreads();
  }
}

cudaError_t launch_token_logprobs(const LogprobParams& p, bool bf16, cudaStream_t stream, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.rows);
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return bf16 ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<__nv_bfloat16>, p)
              : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<float>, p);
}

}  // namespace gr

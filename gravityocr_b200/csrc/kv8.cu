// The paged K/V cache written and read back, in bf16, e4m3 or int8 (kv8_dev.cuh has the 8-bit row's definition).
//
// qk_norm_rope_write: one pass over projected rows [q heads | k heads | v heads] x 128.  q and k heads get their RMS norm
// (optional) and the rotation, q goes to q_out in bf16, k and v rows go to the cache at the row's slot.  A warp owns a
// row, or a share of its heads when there are few rows: its lanes compute the row's cos / sin once, in registers, and
// a head is 32 lanes x 4 elements, so norms and row maxima are warp reductions.
// q is computed in fp32 and rounded once to bf16.  An 8-bit k row is computed in fp64 (position angle, norm, rotation) and
// rounded once to its grid: an fp32 result would land on the wrong side of a rounding border about once in 10^6
// elements, and the cached codes would then depend on the kernel's operation order.
// kv_read: rows by slot back to bf16, exact.
#include "kv8_dev.cuh"

namespace gr {

constexpr int kWriteThreads = 128;
constexpr int kReadThreads = 256;

__device__ __forceinline__ double shfl_d(double v, int src) {
  return __hiloint2double(__shfl_sync(0xffffffffu, __double2hiint(v), src),
                          __shfl_sync(0xffffffffu, __double2loint(v), src));
}
__device__ __forceinline__ void load4(const __nv_bfloat16* src, float (&x)[4]) {
  const uint2 raw = *reinterpret_cast<const uint2*>(src);
  x[0] = __uint_as_float(raw.x << 16);
  x[1] = __uint_as_float(raw.x & 0xffff0000u);
  x[2] = __uint_as_float(raw.y << 16);
  x[3] = __uint_as_float(raw.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(__nv_bfloat16* dst, const float (&y)[4]) {
  uint2 pk;
  pk.x = pack_bf16(y[0], y[1]);
  pk.y = pack_bf16(y[2], y[3]);
  *reinterpret_cast<uint2*>(dst) = pk;
}

// Norm and rotation of one head in T (float or double): y = rope(x * rsqrt(mean x^2 + eps) * w).  c / s: this lane's
// four cosines and signed sines; partner elements are x[i ^ 1] (interleaved) or the same i of lane `src` (half-split).
template <typename T, bool HALF>
__device__ __forceinline__ void norm_rotate(const float (&x)[4], const float* w, double eps, bool rot, int src,
                                            const T (&c)[4], const T (&s)[4], T (&y)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = x[i];
  if (w) {
    T ss = y[0] * y[0] + y[1] * y[1] + y[2] * y[2] + y[3] * y[3];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const T r = static_cast<T>(rsqrt(ss * static_cast<T>(1.0 / 128) + static_cast<T>(eps)));
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] *= r * static_cast<T>(w[i]);
  }
  T z[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) z[i] = HALF ? __shfl_sync(0xffffffffu, y[i], src) : y[i ^ 1];
  if (rot) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = y[i] * c[i] + z[i] * s[i];
  }
}

// One 8-bit row: the warp's 128 values to codes and exponent at byte offset `at` (codes) and index `ai` (exponents).
template <int FMT>
__device__ __forceinline__ void put_row(const double (&y)[4], int lane, uint8_t* codes, int8_t* exps) {
  // largest |y| by its bits, the sign shifted out: NaNs rank highest (an fp64 abs may give a NaN a sign)
  unsigned long long b = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) b = max(b, static_cast<unsigned long long>(__double_as_longlong(y[i])) << 1);
  const int raw = __reduce_max_sync(0xffffffffu, kv_exp_of<FMT>(static_cast<long long>(b >> 1)));
  const int e = max(kKvExpMin, min(kKvExpMax, raw));
  const double f = exp2i64(-e);
  double q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = fmin(fmax(y[i] * f, -448.0), 448.0);
  const bool bad = raw >= (1 << 20);
  *reinterpret_cast<uint32_t*>(codes + lane * 4) = bad ? 0u : kv_pack<FMT>(q);
  if (lane == 0) *exps = static_cast<int8_t>(bad ? kKvExpBad : e);
}
template <int FMT>
__device__ __forceinline__ void put_row(const float (&y)[4], int lane, uint8_t* codes, int8_t* exps) {
  uint32_t b = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) b = max(b, __float_as_uint(y[i]) & 0x7fffffffu);
  const int raw = __reduce_max_sync(0xffffffffu, kv_exp_of<FMT>(b));
  const int e = max(kKvExpMin, min(kKvExpMax, raw));
  const float f = exp2i(-e);
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = fminf(fmaxf(y[i] * f, -448.f), 448.f);
  const bool bad = raw >= (1 << 20);
  *reinterpret_cast<uint32_t*>(codes + lane * 4) = bad ? 0u : kv_pack<FMT>(q);
  if (lane == 0) *exps = static_cast<int8_t>(bad ? kKvExpBad : e);
}

template <int FMT, bool HALF>
__global__ void __launch_bounds__(kWriteThreads) qk_norm_rope_write_kernel(const KvWriteParams p) {
  if (threadIdx.x == 0) pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kWriteThreads + threadIdx.x) >> 5;
  const int64_t row = unit / p.groups;
  if (row >= p.m) return;
  const int g = static_cast<int>(unit - row * p.groups);
  const int n_heads = p.n_q_heads + 2 * p.n_kv_heads;
  // this row's angles: lane l computes pairs l and l + 32, then every lane fetches the pairs of its four elements
  const int pairs = p.rotary_dim >> 1;
  double cd[4], sd[4];
  float cf[4], sf[4];
  {
    double c2[2] = {1.0, 1.0}, s2[2] = {0.0, 0.0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = lane + 32 * h;
      if (i < pairs) {
        int pos;
        if (p.row_pos3) pos = p.row_pos3[row * 3 + (i < p.mrope_s0 ? 0 : (i < p.mrope_s0 + p.mrope_s1 ? 1 : 2))];
        else pos = p.row_pos[row];
        sincos(static_cast<double>(pos) * static_cast<double>(p.inv_freq[i]), &s2[h], &c2[h]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane * 4 + i;
      const int pair = HALF ? (d < pairs ? d : d - pairs) : (d >> 1);
      const double ca = shfl_d(c2[0], pair & 31), cb = shfl_d(c2[1], pair & 31);
      const double sa = shfl_d(s2[0], pair & 31), sb = shfl_d(s2[1], pair & 31);
      const bool neg = HALF ? d < pairs : !(i & 1);
      cd[i] = (pair & 32) ? cb : ca;
      sd[i] = (pair & 32) ? sb : sa;
      if (neg) sd[i] = -sd[i];
      cf[i] = static_cast<float>(cd[i]);
      sf[i] = static_cast<float>(sd[i]);
    }
  }
  const bool rot = lane * 4 < p.rotary_dim;
  const int hop = p.rotary_dim >> 3;  // half-split: partner elements are rotary_dim / 2 apart
  const int src = !HALF || !rot ? lane : (lane < hop ? lane + hop : lane - hop);
  float wq[4], wk[4];
  if (p.q_norm) load4(p.q_norm + lane * 4, wq);
  if (p.k_norm) load4(p.k_norm + lane * 4, wk);
  int64_t slot = p.row_slot[row];
  if (slot >= p.n_slots) {
    if (lane == 0) report(p.status, GR_ERR_BAD_PAGE);
    slot = -1;
  }
  const int64_t page = slot >> 4;
  const int off = static_cast<int>(slot & 15);
  const __nv_bfloat16* in = p.qkv + row * p.ld_qkv + lane * 4;
  for (int h = g; h < n_heads; h += p.groups) {
    if (h >= p.n_q_heads && slot < 0) break;
    float x[4];
    load4(in + h * 128, x);
    if (h < p.n_q_heads) {
      float y[4];
      norm_rotate<float, HALF>(x, p.q_norm ? wq : nullptr, p.eps, rot, src, cf, sf, y);
      store4(p.q_out + (row * p.n_q_heads + h) * 128 + lane * 4, y);
      continue;
    }
    const bool is_k = h < p.n_q_heads + p.n_kv_heads;
    const int kvh = h - p.n_q_heads - (is_k ? 0 : p.n_kv_heads);
    const int64_t r = (page * p.n_kv_heads + kvh) * 16 + off;  // the cache row
    if (FMT == GR_KV_BF16) {
      float y[4];
      if (is_k) norm_rotate<float, HALF>(x, p.k_norm ? wk : nullptr, p.eps, rot, src, cf, sf, y);
      store4(static_cast<__nv_bfloat16*>(is_k ? p.k : p.v) + r * 128 + lane * 4, is_k ? y : x);
    } else if (is_k) {
      double y[4];
      norm_rotate<double, HALF>(x, p.k_norm ? wk : nullptr, p.eps, rot, src, cd, sd, y);
      put_row<FMT>(y, lane, static_cast<uint8_t*>(p.k) + r * 128, p.k_exp + r);
    } else {
      put_row<FMT>(x, lane, static_cast<uint8_t*>(p.v) + r * 128, p.v_exp + r);
    }
  }
}

// Sixteen elements per item: item = ((row * 2 + K or V) * heads + head) * 8 + eighth of the head.
template <int FMT>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const KvReadParams p) {
  if (threadIdx.x == 0) pdl_trigger();
  pdl_wait();
  const int per_row = 16 * p.n_kv_heads;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kReadThreads + threadIdx.x;
  const int64_t row = item / per_row;
  if (row >= p.n) return;
  const int rest = static_cast<int>(item - row * per_row);
  const int which = rest / (8 * p.n_kv_heads);
  const int hc = rest - which * 8 * p.n_kv_heads;  // head * 8 + eighth
  const int64_t slot = p.slots[row];
  if (slot < 0) return;
  if (slot >= p.n_slots) {
    report(p.status, GR_ERR_BAD_PAGE);
    return;
  }
  const int64_t r = ((slot >> 4) * p.n_kv_heads + (hc >> 3)) * 16 + (slot & 15);
  uint4* dst = reinterpret_cast<uint4*>((which ? p.v_out : p.k_out) + row * p.n_kv_heads * 128 + hc * 16);
  if (FMT == GR_KV_BF16) {
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(which ? p.v : p.k) + r * 128 +
                                                      (hc & 7) * 16);
    const uint4 a = __ldg(src), b = __ldg(src + 1);
    dst[0] = a;
    dst[1] = b;
    return;
  }
  const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(which ? p.v : p.k) + r * 128 +
                                                    (hc & 7) * 16);
  const float f = kv_scale((which ? p.v_exp : p.k_exp)[r]);
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t a, b;
    kv_unpack<FMT>(w[i], a, b);
    const float2 fa = __half22float2(*reinterpret_cast<__half2*>(&a));
    const float2 fb = __half22float2(*reinterpret_cast<__half2*>(&b));
    o[2 * i] = pack_bf16(fa.x * f, fa.y * f);
    o[2 * i + 1] = pack_bf16(fb.x * f, fb.y * f);
  }
  dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
  dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

cudaError_t launch_qk_norm_rope_write(KvWriteParams p, int format, bool half, cudaStream_t s, bool pdl) {
  const int n_heads = p.n_q_heads + 2 * p.n_kv_heads;
  // a warp per row once that fills the GPU; fewer rows share their heads between warps
  const int64_t want = static_cast<int64_t>(p.sms) * 16;
  int64_t groups = (want + p.m - 1) / p.m;
  p.groups = static_cast<int>(groups < 1 ? 1 : (groups > n_heads ? n_heads : groups));
  const int64_t units = static_cast<int64_t>(p.m) * p.groups;
  const dim3 grid(static_cast<unsigned>((units + kWriteThreads / 32 - 1) / (kWriteThreads / 32)));
  auto go = [&](auto kern) { return launch_dependent(kern, grid, kWriteThreads, 0, s, pdl, p); };
  switch (format) {
    case GR_KV_E4M3:
      return half ? go(qk_norm_rope_write_kernel<GR_KV_E4M3, true>) : go(qk_norm_rope_write_kernel<GR_KV_E4M3, false>);
    case GR_KV_INT8:
      return half ? go(qk_norm_rope_write_kernel<GR_KV_INT8, true>) : go(qk_norm_rope_write_kernel<GR_KV_INT8, false>);
    default:
      return half ? go(qk_norm_rope_write_kernel<GR_KV_BF16, true>) : go(qk_norm_rope_write_kernel<GR_KV_BF16, false>);
  }
}

cudaError_t launch_kv_read(const KvReadParams& p, int format, cudaStream_t s, bool pdl) {
  const int64_t items = p.n * 16 * p.n_kv_heads;
  const dim3 grid(static_cast<unsigned>((items + kReadThreads - 1) / kReadThreads));
  switch (format) {
    case GR_KV_E4M3: return launch_dependent(kv_read_kernel<GR_KV_E4M3>, grid, kReadThreads, 0, s, pdl, p);
    case GR_KV_INT8: return launch_dependent(kv_read_kernel<GR_KV_INT8>, grid, kReadThreads, 0, s, pdl, p);
    default: return launch_dependent(kv_read_kernel<GR_KV_BF16>, grid, kReadThreads, 0, s, pdl, p);
  }
}

}  // namespace gr

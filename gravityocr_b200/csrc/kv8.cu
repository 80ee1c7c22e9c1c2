// The paged K/V cache written and read back, in bf16, e4m3 or int8 (kv8_dev.cuh has the 8-bit row's definition).
//
// qk_norm_rope_write: one pass over projected rows [q heads | k heads | v heads] x 128.  q and k heads get their RMS norm
// (optional) and the rotation, q goes to q_out in bf16, k and v rows go to the cache at the row's slot.  A warp owns a
// row, or a share of its heads when there are few rows.  Its lanes compute the row's cos / sin once, into shared memory; a
// head is 16 lanes x 8 elements (16-byte loads and stores), so a warp works on two heads of a kind at a time and norms
// and row maxima are four shuffles for both.
// q is computed in fp32 and rounded once to bf16.  An 8-bit k row is computed in fp64 (position angle, norm, rotation) and
// rounded once to its grid: an fp32 result would land on the wrong side of a rounding border about once in 10^6
// elements, and the cached codes would then depend on the kernel's operation order.
// kv_read: rows by slot back to bf16, exact.
//
// Measured (16 q and 8 k / v heads, int8, norms, rotation of 128).  Write: 1,088 rows 7 us, 16,496 rows 77 us (237 MB, 3.1
// TB/s), bound by its instructions: 3,562 a row, 394 of them for the 64-bit angles, 139 for each pair of q heads and 514 for
// each pair of k heads with its pair of v heads; 71% of the issue slots.  A warp per row keeps angles, norms and maxima
// within the warp; seven CTAs an SM cover its latencies (six: 82 us).  Read: 66,560 rows 66 us (411 MB, 6.2 TB/s, a copy's
// rate).
#include "kv8_dev.cuh"

namespace gr {

constexpr int kWriteThreads = 128;
constexpr int kReadThreads = 128;
constexpr int kReadItems = 4;

__device__ __forceinline__ void unpack8(const uint4& raw, float (&x)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void store8(__nv_bfloat16* dst, const float (&y)[8]) {
  *reinterpret_cast<uint4*>(dst) =
      make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
}
// Sum / maximum over the 16 lanes of a head.
template <typename T>
__device__ __forceinline__ T head_sum(T v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ int head_max(int v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Where pair i of the row's (cos, sin) lies: lanes that read together read side by side.
template <bool HALF>
__device__ __forceinline__ int pair_slot(int i) {
  return HALF ? (i & 7) * 8 + (i >> 3) : (i & 3) * 16 + (i >> 2);
}
// This lane's k-th pair: of its elements 2k, 2k + 1, or (half-split) of its element k and its partner.
template <bool HALF>
__device__ __forceinline__ int lane_slot(int k, int l16, int hop) {
  return HALF ? k * 8 + (l16 < hop ? l16 : (l16 - hop) & 7) : k * 16 + l16;
}
// Norm and rotation of a head in T (float or double): y = rope(x * w / sqrt(mean x^2 + eps)); cs(k): this lane's k-th pair.
template <typename T, bool HALF, typename F>
__device__ __forceinline__ void norm_rotate(const float (&x)[8], bool norm, const uint4& w, double eps, int rotary_dim,
                                            int l16, T (&y)[8], F cs) {
  if (norm) {
    float wf[8];
    unpack8(w, wf);
    T ss = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += static_cast<T>(x[i]) * static_cast<T>(x[i]);
    ss = head_sum(ss);
    const T r = static_cast<T>(rsqrt(ss * static_cast<T>(1.0 / 128) + static_cast<T>(eps)));
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = static_cast<T>(x[i] * wf[i]) * r;  // a product of two bf16 is exact in fp32
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
  }
  if (rotary_dim == 0) return;
  const bool rot = l16 * 8 < rotary_dim;
  if (HALF) {
    const int hop = rotary_dim >> 4;  // lanes between an element and its partner
    const bool low = l16 < hop;
    const int src = (threadIdx.x & 16) | (!rot ? l16 : (low ? l16 + hop : l16 - hop));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T z = __shfl_sync(0xffffffffu, y[i], src);
      const auto c = cs(i);
      if (rot) y[i] = y[i] * c.x + z * c.y;  // c.y has the sign of the element's half
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T a = y[2 * i], b = y[2 * i + 1];
      const auto c = cs(i);
      if (rot) {
        y[2 * i] = a * c.x - b * c.y;
        y[2 * i + 1] = b * c.x + a * c.y;
      }
    }
  }
}

// One 8-bit row: the head's 128 values to codes and exponent.
template <int FMT, typename T>
__device__ __forceinline__ void put_row(const T (&y)[8], int l16, bool store, uint8_t* codes, int8_t* exps) {
  // the largest |y| by its bits (NaNs rank highest)
  int raw;
  if constexpr (sizeof(T) == 8) {
    // the high words, one up where the low word is not zero: the exponent's border has zeros below the high word
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      b = max(b, (static_cast<uint32_t>(__double2hiint(y[i])) & 0x7fffffffu) + (__double2loint(y[i]) != 0 ? 1u : 0u));
    raw = kv_exp_of<FMT>(static_cast<long long>(static_cast<unsigned long long>(b) << 32));
  } else {
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) b = max(b, __float_as_uint(y[i]) & 0x7fffffffu);
    raw = kv_exp_of<FMT>(b);
  }
  raw = head_max(raw);
  const int e = max(kKvExpMin, min(kKvExpMax, raw));
  T f;
  if constexpr (sizeof(T) == 8) f = exp2i64(-e);
  else f = exp2i(-e);
  T lo[4], hi[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo[i] = y[i] * f;
    hi[i] = y[4 + i] * f;
  }
  if (raw > kKvExpMax) {  // past the exponents' range: saturate (a bad row's codes are dropped below)
    constexpr T top = FMT == GR_KV_E4M3 ? 448 : 127;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = lo[i] > top ? top : (lo[i] < -top ? -top : lo[i]);
      hi[i] = hi[i] > top ? top : (hi[i] < -top ? -top : hi[i]);
    }
  }
  const bool bad = raw >= (1 << 20);
  const uint2 c = bad ? make_uint2(0u, 0u) : make_uint2(kv_pack<FMT>(lo), kv_pack<FMT>(hi));
  if (store) {
    *reinterpret_cast<uint2*>(codes + l16 * 8) = c;
    if (l16 == 0) *exps = static_cast<int8_t>(bad ? kKvExpBad : e);
  }
}

template <int FMT, bool HALF>
__global__ void __launch_bounds__(kWriteThreads, 7) qk_norm_rope_write_kernel(const KvWriteParams p) {
  __shared__ double2 s_cs64[FMT != GR_KV_BF16 ? kWriteThreads / 32 : 1][64];
  __shared__ float2 s_cs32[kWriteThreads / 32][64];
  if (threadIdx.x == 0) pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, l16 = lane & 15, sub = lane >> 4;
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kWriteThreads + threadIdx.x) >> 5;
  const int64_t row = unit / p.groups;
  if (row >= p.m) return;
  const int g = static_cast<int>(unit - row * p.groups);
  // pairs of heads: q, then k, then v; this warp takes g, g + groups, ...
  const int n_qp = (p.n_q_heads + 1) >> 1, n_kp = (p.n_kv_heads + 1) >> 1;
  const bool even = !((p.n_q_heads | p.n_kv_heads) & 1);
  int64_t slot = p.row_slot[row];
  if (slot >= p.n_slots) {
    if (lane == 0 && g == 0) report(p.status, GR_ERR_BAD_PAGE);
    slot = -1;
  }
  const int n_pairs = slot < 0 ? n_qp : n_qp + 2 * n_kp;
  const __nv_bfloat16* in = p.qkv + row * p.ld_qkv + l16 * 8;
  // this lane's head of pair i, from the row's start (an odd count's last pair has one head: its other half repeats it)
  auto head_of = [&](int i) {
    if (i < n_qp) return min(2 * i + sub, p.n_q_heads - 1);
    i -= n_qp;
    if (i < n_kp) return p.n_q_heads + min(2 * i + sub, p.n_kv_heads - 1);
    return p.n_q_heads + p.n_kv_heads + min(2 * (i - n_kp) + sub, p.n_kv_heads - 1);
  };
  auto load = [&](int i) { return __ldg(reinterpret_cast<const uint4*>(in + (even ? 2 * i + sub : head_of(i)) * 128)); };
  uint4 next = make_uint4(0, 0, 0, 0);
  if (g < n_pairs) next = load(g);

  double2* cs64 = s_cs64[FMT != GR_KV_BF16 ? threadIdx.x >> 5 : 0];
  float2* cs32 = s_cs32[threadIdx.x >> 5];
  for (int i = lane; i < (p.rotary_dim >> 1); i += 32) {
    int pos;
    if (p.row_pos3) pos = p.row_pos3[row * 3 + (i < p.mrope_s0 ? 0 : (i < p.mrope_s0 + p.mrope_s1 ? 1 : 2))];
    else pos = p.row_pos[row];
    // sincospi reduces exactly; the multiplication by 1 / pi is off by 2^-53 of the angle
    double c, s;
    sincospi(static_cast<double>(pos) * static_cast<double>(p.inv_freq[i]) * 0.31830988618379067154, &s, &c);
    if (FMT != GR_KV_BF16) cs64[pair_slot<HALF>(i)] = make_double2(c, s);
    cs32[pair_slot<HALF>(i)] = make_float2(static_cast<float>(c), static_cast<float>(s));
  }
  uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;
  if (p.q_norm) wq = __ldg(reinterpret_cast<const uint4*>(p.q_norm) + l16);
  if (p.k_norm) wk = __ldg(reinterpret_cast<const uint4*>(p.k_norm) + l16);
  __syncwarp();
  // q's pairs stay in registers, the fp64 ones are read when a k head comes
  const int hop = p.rotary_dim >> 4;
  float2 csf[HALF ? 8 : 4];
#pragma unroll
  for (int k = 0; k < (HALF ? 8 : 4); ++k) {
    csf[k] = cs32[lane_slot<HALF>(k, l16, hop)];
    if (HALF && l16 < hop) csf[k].y = -csf[k].y;
  }
  auto cs_f = [&](int k) { return csf[k]; };
  auto cs_d = [&](int k) {
    double2 c = cs64[lane_slot<HALF>(k, l16, hop)];
    if (HALF && l16 < hop) c.y = -c.y;
    return c;
  };

  const int64_t cache_row = (slot >> 4) * p.n_kv_heads * 16 + (slot & 15);
  for (int i = g; i < n_pairs; i += p.groups) {
    float x[8];
    unpack8(next, x);
    if (i + p.groups < n_pairs) next = load(i + p.groups);
    if (i < n_qp) {
      const int h = 2 * i + sub;
      float y[8];
      norm_rotate<float, HALF>(x, p.q_norm != nullptr, wq, p.eps, p.rotary_dim, l16, y, cs_f);
      if (h < p.n_q_heads) store8(p.q_out + (row * p.n_q_heads + h) * 128 + l16 * 8, y);
      continue;
    }
    const bool is_k = i < n_qp + n_kp;
    const int kvh = 2 * (i - n_qp - (is_k ? 0 : n_kp)) + sub;
    const bool store = kvh < p.n_kv_heads;
    const int64_t r = cache_row + kvh * 16;
    if (FMT == GR_KV_BF16) {
      float y[8];
      if (is_k) {
        norm_rotate<float, HALF>(x, p.k_norm != nullptr, wk, p.eps, p.rotary_dim, l16, y, cs_f);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[e];
      }
      if (store) store8(static_cast<__nv_bfloat16*>(is_k ? p.k : p.v) + r * 128 + l16 * 8, y);
    } else if (is_k) {
      double y[8];
      norm_rotate<double, HALF>(x, p.k_norm != nullptr, wk, p.eps, p.rotary_dim, l16, y, cs_d);
      put_row<FMT>(y, l16, store, static_cast<uint8_t*>(p.k) + r * 128, p.k_exp + r);
    } else {
      put_row<FMT>(x, l16, store, static_cast<uint8_t*>(p.v) + r * 128, p.v_exp + r);
    }
  }
}

// A warp reads one row's K or V; a lane takes 8 elements (a warp's stores cover whole lines) of kReadItems pairs of heads at a
// time, every load before the first store.
template <int FMT>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const KvReadParams p) {
  if (threadIdx.x == 0) pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kReadThreads / 32) + (threadIdx.x >> 5);
  const int64_t row = unit >> 1;
  if (row >= p.n) return;
  const bool v = unit & 1;
  const int64_t slot = __ldg(p.slots + row);
  if (slot >= p.n_slots && lane == 0) report(p.status, GR_ERR_BAD_PAGE);
  if (slot < 0 || slot >= p.n_slots) return;
  const int64_t row0 = (slot >> 4) * p.n_kv_heads * 16 + (slot & 15);  // cache row of head 0
  const uint8_t* codes = static_cast<const uint8_t*>(v ? p.v : p.k);
  const int8_t* exps = v ? p.v_exp : p.k_exp;
  __nv_bfloat16* out = (v ? p.v_out : p.k_out) + row * p.n_kv_heads * 128 + (lane & 15) * 8;
  for (int h0 = lane >> 4; h0 < p.n_kv_heads; h0 += 2 * kReadItems) {
    uint4 raw[kReadItems];
    int e[kReadItems];
#pragma unroll
    for (int u = 0; u < kReadItems; ++u) {
      const int h = h0 + 2 * u;
      if (h >= p.n_kv_heads) break;
      const int64_t at = (row0 + h * 16) * 128 + (lane & 15) * 8;
      if (FMT == GR_KV_BF16) {
        raw[u] = __ldg(reinterpret_cast<const uint4*>(codes + at * 2));
      } else {
        const uint2 c = __ldg(reinterpret_cast<const uint2*>(codes + at));
        raw[u].x = c.x;
        raw[u].y = c.y;
        e[u] = __ldg(exps + row0 + h * 16);
      }
    }
#pragma unroll
    for (int u = 0; u < kReadItems; ++u) {
      const int h = h0 + 2 * u;
      if (h >= p.n_kv_heads) break;
      if (FMT != GR_KV_BF16) {
        const float f = kv_scale(e[u]);
        const uint32_t w[2] = {raw[u].x, raw[u].y};
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t a, b;
          kv_unpack<FMT>(w[i], a, b);
          const float2 fa = __half22float2(*reinterpret_cast<__half2*>(&a));
          const float2 fb = __half22float2(*reinterpret_cast<__half2*>(&b));
          o[2 * i] = pack_bf16(fa.x * f, fa.y * f);
          o[2 * i + 1] = pack_bf16(fb.x * f, fb.y * f);
        }
        raw[u] = make_uint4(o[0], o[1], o[2], o[3]);
      }
      *reinterpret_cast<uint4*>(out + h * 128) = raw[u];
    }
  }
}

cudaError_t launch_qk_norm_rope_write(KvWriteParams p, int format, bool half, cudaStream_t s, bool pdl) {
  const int n_pairs = (p.n_q_heads + 1) / 2 + 2 * ((p.n_kv_heads + 1) / 2);
  // a warp per row once that fills the GPU; fewer rows share their heads between warps
  const int64_t want = static_cast<int64_t>(p.sms) * 16;
  int64_t groups = (want + p.m - 1) / p.m;
  p.groups = static_cast<int>(groups < 1 ? 1 : (groups > n_pairs ? n_pairs : groups));
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
  const dim3 grid(static_cast<unsigned>((2 * p.n + kReadThreads / 32 - 1) / (kReadThreads / 32)));
  switch (format) {
    case GR_KV_E4M3: return launch_dependent(kv_read_kernel<GR_KV_E4M3>, grid, kReadThreads, 0, s, pdl, p);
    case GR_KV_INT8: return launch_dependent(kv_read_kernel<GR_KV_INT8>, grid, kReadThreads, 0, s, pdl, p);
    default: return launch_dependent(kv_read_kernel<GR_KV_BF16>, grid, kReadThreads, 0, s, pdl, p);
  }
}

}  // namespace gr

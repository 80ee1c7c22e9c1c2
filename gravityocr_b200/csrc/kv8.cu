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
// Measured (16 q and 8 k / v heads, int8, norms, rotation of 128; launches one behind the other in a graph, on inputs in turn).
// Write: one row 2.5 us, 1,088 rows 7.7, 16,496 rows 65 (237 MB, 3.7 TB/s; e4m3 67, a bf16 cache 52), bound by its
// instructions: 3,010 a row, some 500 of them for the 64-bit angles, 120 for each pair of q heads and 380 for each pair of k
// heads with its pair of v heads; 71% of the issue slots.  A warp per row keeps angles, norms and maxima within the warp; at
// 1,088 rows three warps share a row, each with all of its angles.  Read: 66,560 rows 66 us (411 MB, 6.2 TB/s, a copy's rate).
#include "kv8_dev.cuh"

namespace gr {

constexpr int kWriteThreads = 128;
constexpr int kWriteCtas = 7;  // an SM (16,496 rows: six 68 us, seven 65, eight 67)
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
// The slot of this lane's pair 0 (k further pairs at + k * 8 or k * 16): of its elements 2k, 2k + 1, or (half-split, hop lanes
// between an element and its partner) of its element k and its partner.  Lanes past the rotation find (1, 0).
template <bool HALF>
__device__ __forceinline__ int lane_slot(int l16, int hop) {
  return HALF ? (l16 < hop ? l16 : (l16 < 2 * hop ? l16 - hop : hop & 7)) : l16;
}
// mean x^2 + eps of a head.
template <typename T>
__device__ __forceinline__ T head_square(const float (&x)[8], double eps) {
  T ss = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss += static_cast<T>(x[i]) * static_cast<T>(x[i]);
  return head_sum(ss) * static_cast<T>(1.0 / 128) + static_cast<T>(eps);
}

// Norm and rotation of a head in fp32; cs(k): this lane's k-th pair.  x r stays within sqrt(128) whatever the size of x and w,
// its squares may not: true where they leave fp32 or its normal numbers (WIDE: with a norm in fp64, for such heads).
template <bool HALF, bool WIDE, typename F>
__device__ __forceinline__ bool norm_rotate(float (&x)[8], bool norm, const uint4& w, double eps, int rotary_dim, int l16,
                                            F cs) {
  bool odd = false;
  if (norm) {
    float wf[8];
    unpack8(w, wf);
    const float sq = head_square<float>(x, eps);
    odd = !(sq > 0x1p-100f && sq < 0x1p120f);
    if (WIDE) {
      const double r = rsqrt(head_square<double>(x, eps));
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(static_cast<double>(x[i]) * r) * wf[i];
    } else {
      const float r = rsqrtf(sq);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * wf[i];
    }
  }
  if (rotary_dim == 0) return odd;
  const bool rot = l16 * 8 < rotary_dim;
  if (HALF) {
    const int hop = rotary_dim >> 4;
    const int src = (threadIdx.x & 16) | (!rot ? l16 : (l16 < hop ? l16 + hop : l16 - hop));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float z = __shfl_sync(0xffffffffu, x[i], src);
      const float2 c = cs(i);
      if (rot) x[i] = x[i] * c.x + z * c.y;  // c.y has the sign of the element's half
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[2 * i], b = x[2 * i + 1];
      const float2 c = cs(i);
      if (rot) {
        x[2 * i] = a * c.x - b * c.y;
        x[2 * i + 1] = b * c.x + a * c.y;
      }
    }
  }
  return odd;
}

__device__ __forceinline__ int clamp_exp(int raw) { return max(kKvExpMin, min(kKvExpMax, raw)); }
// This lane's eight codes and, once a head, the exponent.
__device__ __forceinline__ void store_row(uint2 c, int raw, int l16, bool store, uint8_t* codes, int8_t* exps) {
  const bool bad = raw >= (1 << 20);
  if (store) {
    *reinterpret_cast<uint2*>(codes) = bad ? make_uint2(0u, 0u) : c;
    if (l16 == 0) *exps = static_cast<int8_t>(bad ? kKvExpBad : clamp_exp(raw));
  }
}
// An 8-bit v row: the head's bf16 values, scaled exactly, to codes and exponent.
template <int FMT>
__device__ __forceinline__ void put_v(const uint4& in, const float (&x)[8], int l16, bool store, uint8_t* codes,
                                      int8_t* exps) {
  // the largest |x| by its bits (NaNs rank highest)
  constexpr uint32_t mag = 0x7fff7fffu;
  const uint32_t m2 = __vmaxu2(__vmaxu2(in.x & mag, in.y & mag), __vmaxu2(in.z & mag, in.w & mag));
  const int raw = kv_exp_of<FMT>(static_cast<uint32_t>(head_max(static_cast<int>(max(m2 << 16, m2 & 0xffff0000u)))));
  const float f = exp2i(-clamp_exp(raw));
  constexpr float top = FMT == GR_KV_E4M3 ? 448.f : 127.f;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = x[i] * f;
  if (raw > kKvExpMax) {  // past the exponents' range: saturate (a bad row's codes are dropped)
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = y[i] > top ? top : (y[i] < -top ? -top : y[i]);
  }
  store_row(make_uint2(kv_pack<FMT>({y[0], y[1], y[2], y[3]}), kv_pack<FMT>({y[4], y[5], y[6], y[7]})), raw, l16, store,
            codes, exps);
}
// The rotation of a k row in fp64; a: fp32 or fp64.
template <bool HALF, typename T>
__device__ __forceinline__ void rotate64(double (&y)[8], const T (&a)[8], int rotary_dim, int l16, const double2* cs) {
  if (rotary_dim == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = a[i];
  } else if (HALF) {
    const int hop = rotary_dim >> 4;
    const int src = (threadIdx.x & 16) | (l16 >= 2 * hop ? l16 : (l16 < hop ? l16 + hop : l16 - hop));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T z = __shfl_sync(0xffffffffu, a[i], src);
      const double2 c = cs[i * 8];  // c.y has the sign of the element's half
      y[i] = static_cast<double>(a[i]) * c.x + static_cast<double>(z) * c.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double u = a[2 * i], v = a[2 * i + 1];
      const double2 c = cs[i * 16];
      y[2 * i] = u * c.x - v * c.y;
      y[2 * i + 1] = v * c.x + u * c.y;
    }
  }
}
// Exponent of the row y r, not clamped from above: from the high words; where their next value up would give another one, from
// the largest |y r| itself.
template <int FMT>
__device__ __forceinline__ int exp_of_row(const double (&y)[8], double r) {
  int hi = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) hi = max(hi, __double2hiint(y[i]) & 0x7fffffff);
  hi = head_max(hi);
  auto exp_of = [](double v) { return max(kv_exp_of<FMT>(__double_as_longlong(fabs(v))), kKvExpMin); };
  int raw = exp_of(__hiloint2double(hi, 0) * r);
  if (__any_sync(0xffffffffu, raw != exp_of(__hiloint2double(hi + 1, 0) * r))) {
    long long m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __double_as_longlong(y[i] * r) & 0x7fffffffffffffffll);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    raw = max(kv_exp_of<FMT>(m), kKvExpMin);
  }
  return raw;
}
// An 8-bit k row: norm, rotation and rounding in fp64.  With a = x w and r = 1 / rms the row is r * (a c + z s): a and the
// partners z are fp32, where a product of two bf16 is exact while it is a normal number; r goes with 2^-e into one factor, and
// the sum with the rounding constant (kv8_dev.cuh) is fused with it: one multiplication an element is left of three.
// A product past fp32 gives a bad row, one below its normal numbers is off by 2^-150, which only an r above 2^40 brings near
// the codes' steps (2^-49 and up): `odd` for such heads (WIDE: fp64 products).
template <int FMT, bool HALF, bool WIDE>
__device__ __forceinline__ void put_k(float (&a)[8], bool norm, const uint4& w, double eps, int rotary_dim, int l16,
                                      const double2* cs, bool store, uint8_t* codes, int8_t* exps, volatile int* odd) {
  double r = 1.0, y[8];
  float wf[8];
  if (norm) {
    r = rsqrt(head_square<double>(a, eps));
    unpack8(w, wf);
  }
  if (WIDE && norm) {
    double d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = static_cast<double>(a[i]) * static_cast<double>(wf[i]);
    rotate64<HALF>(y, d, rotary_dim, l16, cs);
  } else {
    if (norm) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] *= wf[i];
    }
    rotate64<HALF>(y, a, rotary_dim, l16, cs);
  }
  const int raw = exp_of_row<FMT>(y, r);
  if (!WIDE && norm && (raw >= (1 << 20) || r > 0x1p40)) *odd = 1;
  const double f = r * exp2i64(-clamp_exp(raw));
  if (raw > kKvExpMax) {
    constexpr double top = FMT == GR_KV_E4M3 ? 448 : 127;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = y[i] * f > top ? top / f : (y[i] * f < -top ? -top / f : y[i]);
  }
  const uint2 c = make_uint2(kv_pack<FMT>({y[0], y[1], y[2], y[3]}, f), kv_pack<FMT>({y[4], y[5], y[6], y[7]}, f));
  store_row(c, raw, l16, store, codes, exps);
}

// This lane's head of pair i, from the row's start (an odd count's last pair has one head: its other half repeats it).  Pairs
// of heads: n_qp of q, n_kp of k, n_kp of v.
__device__ __forceinline__ int head_of_pair(const KvWriteParams& p, int i, int n_qp, int n_kp, int sub) {
  if (i < n_qp) return min(2 * i + sub, p.n_q_heads - 1);
  i -= n_qp;
  if (i < n_kp) return p.n_q_heads + min(2 * i + sub, p.n_kv_heads - 1);
  return p.n_q_heads + p.n_kv_heads + min(2 * (i - n_kp) + sub, p.n_kv_heads - 1);
}

// A warp's q and k heads once more, those whose norm needs fp64 over what the lanes wrote (the others stay: an 8-bit k row
// comes out the same).  Rare, and out of line behind the warp's loops: within them it costs every row registers (write and
// read of 16,496 rows 88 us, so 82).
template <int FMT, bool HALF>
__device__ __noinline__ void wide_heads(const KvWriteParams& p, const double2* all64, const float2* all32) {
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kWriteThreads + threadIdx.x) >> 5, row = unit / p.groups;
  const int g = static_cast<int>(unit - row * p.groups);
  int64_t slot = p.row_slot[row];
  if (slot >= p.n_slots) slot = -1;
  const double2* cs64 = all64 + (threadIdx.x >> 5) * (HALF ? 128 : 64);
  const float2* cs32 = all32 + (threadIdx.x >> 5) * 64;
  const int l16 = threadIdx.x & 15, sub = (threadIdx.x >> 4) & 1;
  const int hop = p.rotary_dim >> 4, slot0 = lane_slot<HALF>(l16, hop);
  const int n_qp = (p.n_q_heads + 1) >> 1, n_kp = slot < 0 ? 0 : (p.n_kv_heads + 1) >> 1;
  const int64_t cache_row = (slot >> 4) * p.n_kv_heads * 16 + (slot & 15);
  constexpr int row_bytes = FMT == GR_KV_BF16 ? 256 : 128;
  auto cs = [&](int k) {
    float2 c = cs32[slot0 + k * (HALF ? 8 : 16)];
    if (HALF && l16 < hop) c.y = -c.y;
    return c;
  };
#pragma unroll 1
  for (int i = g; i < n_qp + n_kp; i += p.groups) {
    const bool is_q = i < n_qp;
    const __nv_bfloat16* norm = is_q ? p.q_norm : p.k_norm;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (norm) w = __ldg(reinterpret_cast<const uint4*>(norm) + l16);
    float x[8];
    unpack8(__ldg(reinterpret_cast<const uint4*>(p.qkv + row * p.ld_qkv + head_of_pair(p, i, n_qp, n_kp, sub) * 128) + l16), x);
    const int h = 2 * (is_q ? i : i - n_qp) + sub;
    const bool store = h < (is_q ? p.n_q_heads : p.n_kv_heads);
    uint8_t* k_row = static_cast<uint8_t*>(p.k) + (cache_row + h * 16) * row_bytes + l16 * (row_bytes / 16);
    if (is_q || FMT == GR_KV_BF16) {
      const bool odd = norm_rotate<HALF, true>(x, norm != nullptr, w, p.eps, p.rotary_dim, l16, cs);
      __nv_bfloat16* to =
          is_q ? p.q_out + (row * p.n_q_heads + h) * 128 + l16 * 8 : reinterpret_cast<__nv_bfloat16*>(k_row);
      if (store && odd) store8(to, x);
    } else {
      put_k<FMT, HALF, true>(x, norm != nullptr, w, p.eps, p.rotary_dim, l16, cs64 + (HALF && l16 >= hop ? 64 : 0) + slot0,
                             store, k_row, p.k_exp + cache_row + h * 16, nullptr);
    }
  }
}

template <int FMT, bool HALF>
__global__ void __launch_bounds__(kWriteThreads, kWriteCtas) qk_norm_rope_write_kernel(
    const __grid_constant__ KvWriteParams p) {
  // for k: half-split rotations, with -s for the elements of the first half, and with s
  __shared__ double2 s_cs64[FMT != GR_KV_BF16 ? kWriteThreads / 32 : 1][HALF ? 2 : 1][64];
  __shared__ float2 s_cs32[kWriteThreads / 32][64];
  __shared__ int s_odd[kWriteThreads / 32];  // a head of the warp's needs its norm in fp64
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
  auto load = [&](int i) {
    return __ldg(reinterpret_cast<const uint4*>(in + (even ? 2 * i + sub : head_of_pair(p, i, n_qp, n_kp, sub)) * 128));
  };
  uint4 next = make_uint4(0, 0, 0, 0);
  if (g < n_pairs) next = load(g);
  // More rows than run at once: a row's later heads come to L2 at its start, beside other rows' work (16,496 rows: 65 us, 68
  // without).  A single wave only asks for everything at the same time (4,000 rows: 20.7 us, 19.9 without).
  if (lane == 0 && p.m > p.sms * kWriteCtas * (kWriteThreads / 32))
    l2_prefetch(p.qkv + row * p.ld_qkv, static_cast<uint32_t>(p.n_q_heads + 2 * p.n_kv_heads) * 256);

  volatile int* odd = s_odd + (threadIdx.x >> 5);
  if (lane == 0) *odd = 0;
  double2(*cs64)[64] = s_cs64[FMT != GR_KV_BF16 ? threadIdx.x >> 5 : 0];
  float2* cs32 = s_cs32[threadIdx.x >> 5];
  if (p.rotary_dim) {
#pragma unroll 1
    for (int i = lane; i < 64; i += 32) {
      double c = 1.0, s = 0.0;
      if (i < (p.rotary_dim >> 1)) {
        int pos;
        if (p.row_pos3) pos = p.row_pos3[row * 3 + (i < p.mrope_s0 ? 0 : (i < p.mrope_s0 + p.mrope_s1 ? 1 : 2))];
        else pos = p.row_pos[row];
        // sincospi reduces exactly; the multiplication by 1 / pi is off by 2^-53 of the angle
        sincospi(static_cast<double>(pos) * static_cast<double>(p.inv_freq[i]) * 0.31830988618379067154, &s, &c);
      }
      const int at = pair_slot<HALF>(i);
      if (FMT != GR_KV_BF16) {
        cs64[0][at] = make_double2(c, HALF ? -s : s);
        if (HALF) cs64[1][at] = make_double2(c, s);
      }
      cs32[at] = make_float2(static_cast<float>(c), static_cast<float>(s));
    }
  }
  uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;
  if (p.q_norm) wq = __ldg(reinterpret_cast<const uint4*>(p.q_norm) + l16);
  if (p.k_norm) wk = __ldg(reinterpret_cast<const uint4*>(p.k_norm) + l16);
  __syncwarp();
  // q's pairs stay in registers, the fp64 ones are read when a k head comes
  const int hop = p.rotary_dim >> 4, slot0 = lane_slot<HALF>(l16, hop);
  float2 csf[HALF ? 8 : 4];
#pragma unroll
  for (int k = 0; k < (HALF ? 8 : 4); ++k) {
    csf[k] = cs32[slot0 + k * (HALF ? 8 : 16)];
    if (HALF && l16 < hop) csf[k].y = -csf[k].y;
  }
  auto cs_f = [&](int k) { return csf[k]; };
  const double2* cs_d = cs64[HALF && l16 >= hop ? 1 : 0] + slot0;

  int i = g;
  // this lane's values of pair i; the next pair's are on their way
  auto take = [&](float (&x)[8]) {
    const uint4 v = next;
    unpack8(v, x);
    if (i + p.groups < n_pairs) next = load(i + p.groups);
    return v;
  };
  __nv_bfloat16* q_row = p.q_out + row * p.n_q_heads * 128 + l16 * 8;
  for (; i < n_qp; i += p.groups) {
    float x[8];
    take(x);
    if (norm_rotate<HALF, false>(x, p.q_norm != nullptr, wq, p.eps, p.rotary_dim, l16, cs_f)) *odd = 1;
    const int h = 2 * i + sub;
    if (h < p.n_q_heads) store8(q_row + h * 128, x);
  }
  const int64_t cache_row = (slot >> 4) * p.n_kv_heads * 16 + (slot & 15);
  constexpr int row_bytes = FMT == GR_KV_BF16 ? 256 : 128;
  uint8_t* k_row = static_cast<uint8_t*>(p.k) + cache_row * row_bytes + l16 * (row_bytes / 16);
  for (; i < n_qp + n_kp && i < n_pairs; i += p.groups) {
    float x[8];
    take(x);
    const int h = 2 * (i - n_qp) + sub;
    const bool store = h < p.n_kv_heads;
    uint8_t* to = k_row + h * 16 * row_bytes;
    if (FMT == GR_KV_BF16) {
      if (norm_rotate<HALF, false>(x, p.k_norm != nullptr, wk, p.eps, p.rotary_dim, l16, cs_f)) *odd = 1;
      if (store) store8(reinterpret_cast<__nv_bfloat16*>(to), x);
    } else {
      put_k<FMT, HALF, false>(x, p.k_norm != nullptr, wk, p.eps, p.rotary_dim, l16, cs_d, store, to,
                              p.k_exp + cache_row + h * 16, odd);
    }
  }
  uint8_t* v_row = static_cast<uint8_t*>(p.v) + cache_row * row_bytes + l16 * (row_bytes / 16);
  for (; i < n_pairs; i += p.groups) {
    float x[8];
    const uint4 in8 = take(x);
    const int h = 2 * (i - n_qp - n_kp) + sub;
    const bool store = h < p.n_kv_heads;
    uint8_t* to = v_row + h * 16 * row_bytes;
    if (FMT == GR_KV_BF16) {
      if (store) *reinterpret_cast<uint4*>(to) = in8;
    } else {
      put_v<FMT>(in8, x, l16, store, to, p.v_exp + cache_row + h * 16);
    }
  }
  __syncwarp();
  if (s_odd[threadIdx.x >> 5]) wide_heads<FMT, HALF>(p, s_cs64[0][0], s_cs32[0]);
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

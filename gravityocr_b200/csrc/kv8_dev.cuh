// The 8-bit K/V cache row, shared by the kernels that write, read and attend over it.
//
// A row is one (token, K/V head): 128 codes x_i and one exponent e; it stands for x_i * 2^e.  A power of two costs an
// e4m3 code no precision (its relative step does not depend on the scale) and an int8 code half a bit on average; in
// return every scaling here is exact: a row's codes are a pure function of its values, independent of the order in
// which a kernel computes, and reading back (<= 7 significant bits) is exact in bf16.
//   e = the smallest exponent in [-40, 40] with max|x| <= top * 2^e, top = 448 (e4m3) or 127 (int8);
//   code = round-half-even(x * 2^-e) on the code's grid, saturated at +-top.
// A row that holds a NaN or an infinity is stored as e = -128 and zero codes, and reads back as NaN.
// The range of e bounds 2^(e - e') by 2^80 between any two rows of a request: the attention kernel's softmax sum relies
// on it (attention_kv8.cu).
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "params.cuh"

namespace gr {

constexpr int kKvExpMin = -40, kKvExpMax = 40, kKvExpBad = -128;

// Exponent of a row from the bits of its largest |x| (fp32): top = 1.75 * 2^8 or 1.984375 * 2^6, so e is the binade of
// |x| less 8 or 6, one more when the significand is above top's.  Not clamped; `bad` for NaN / infinity.
template <int FMT>
__device__ __forceinline__ int kv_exp_of(uint32_t abs_bits) {
  constexpr uint32_t carry = FMT == GR_KV_E4M3 ? 0x1fffffu : 0x1ffffu;  // 2^23 - 1 - (top's fraction) * 2^23
  constexpr int off = FMT == GR_KV_E4M3 ? 8 : 6;
  if (abs_bits >= 0x7f800000u) return 1 << 20;
  return static_cast<int>((abs_bits + carry) >> 23) - 127 - off;
}
// The same from an fp64 |x|.
template <int FMT>
__device__ __forceinline__ int kv_exp_of(long long abs_bits) {
  constexpr long long carry = FMT == GR_KV_E4M3 ? 0x0003ffffffffffffll : 0x00003fffffffffffll;
  constexpr int off = FMT == GR_KV_E4M3 ? 8 : 6;
  if (abs_bits >= 0x7ff0000000000000ll) return 1 << 20;
  return static_cast<int>((abs_bits + carry) >> 52) - 1023 - off;
}
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }  // 2^e, |e| <= 126
__device__ __forceinline__ double exp2i64(int e) {
  return __hiloint2double((e + 1023) << 20, 0);
}
// Scale of a stored exponent: 2^e, or NaN for a bad row.
__device__ __forceinline__ float kv_scale(int e) {
  return e == kKvExpBad ? __int_as_float(0x7fc00000) : exp2i(e);
}

// Low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Four values, already scaled by 2^-e and within +-top, to four codes (low byte first).  Adding 1.5 * 2^23 (2^52 in fp64)
// rounds to an integer, ties to even, whose low bits are the sum's.
template <int FMT>
__device__ __forceinline__ uint32_t kv_pack(const float (&y)[4]) {
  if (FMT == GR_KV_E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
  constexpr float big = 12582912.f;
  return low_bytes(__float_as_uint(y[0] + big), __float_as_uint(y[1] + big), __float_as_uint(y[2] + big),
                   __float_as_uint(y[3] + big));
}
// Four fp64 values times f, rounded once: to the integer with the addition, or to e4m3 by way of fp32 rounded to odd (towards
// zero, the last bit set where something was cut off), which keeps the second rounding's side.
template <int FMT>
__device__ __forceinline__ uint32_t kv_pack(const double (&y)[4], double f) {
  if (FMT == GR_KV_E4M3) {
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double v = y[i] * f;
      o[i] = __double2float_rz(v);
      if (static_cast<double>(o[i]) != v) o[i] = __int_as_float(__float_as_int(o[i]) | 1);
    }
    return kv_pack<FMT>(o);
  }
  constexpr double big = 6755399441055744.0;
  return low_bytes(__double2loint(__fma_rn(y[0], f, big)), __double2loint(__fma_rn(y[1], f, big)),
                   __double2loint(__fma_rn(y[2], f, big)), __double2loint(__fma_rn(y[3], f, big)));
}

// Two codes in the low 16 bits -> two halves, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffff), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}
// Four int8 codes as two half2 words (codes 0, 1 and 2, 3): the byte x + 128 placed in the low byte of 0x64XX is the half
// 1024 + (x + 128); subtracting 1152 is exact.
__device__ __forceinline__ void int8x4_to_half2x2(uint32_t w, uint32_t& h01, uint32_t& h23) {
  const uint32_t u = w ^ 0x80808080u;
  const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
  uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 ha = __hsub2(*reinterpret_cast<__half2*>(&a), off), hb = __hsub2(*reinterpret_cast<__half2*>(&b), off);
  h01 = *reinterpret_cast<const uint32_t*>(&ha);
  h23 = *reinterpret_cast<const uint32_t*>(&hb);
}
template <int FMT>
__device__ __forceinline__ void kv_unpack(uint32_t w, uint32_t& h01, uint32_t& h23) {
  if (FMT == GR_KV_E4M3) {
    h01 = e4m3x2_to_half2(w);
    h23 = e4m3x2_to_half2(w >> 16);
  } else {
    int8x4_to_half2x2(w, h01, h23);
  }
}

template <typename Kern, typename P>
static inline cudaError_t launch_dependent(Kern kern, dim3 grid, int threads, size_t smem, cudaStream_t stream,
                                           bool pdl, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace gr

// Attention of one to a few new tokens per request over the paged 8-bit K/V cache (rows as kv8_dev.cuh defines them), split
// over the cache's length and joined.
//
// Rows of one request and one K/V head: the GQA group's G query heads x K window rows (row r = g * K + j), in m16 tiles;
// visibility as in attention_dev.cuh (row_limit).  With one new token and G = 2 there are 2 rows: the work is reading
// the cache, 258 bytes a token and head, so everything below serves that stream.
//
// A CTA covers cache positions [split * chunk, (split + 1) * chunk) of one (request, K/V head).  It is made of independent
// warp groups, one warp per m16 tile of rows; a group owns a ring of 32-token stages (two pages: 4 KB of K codes, 4 KB of
// V codes by 2-D TMA in the 128-byte swizzle, 64 bytes of exponents by bulk copies) and its own online softmax over the
// tiles it takes, so no barrier joins the warps until the end.
//
// Codes become halves in registers (exact) right before mma.sync m16n8k16, f16 in, fp32 accumulated.  Which cache element a
// lane holds is a free permutation of the products' inner index, so both operands are read with 16-byte shared loads
// and no transposition beyond byte shuffles:
//   S = Q K^T: the lane with quad index c holds dims 16c..16c+15 and 64+16c..64+16c+15 of its token (and of its two Q rows);
//   O = P V:   it holds tokens c, c+4, c+8, c+12 of a page, exactly the columns of S it has, for 16 dims of one 16-dim chunk.
// Conflict-free: the 8 lanes of a shared-load phase touch 8 different 16-byte chunks of the swizzled tile.
//
// Scales: a row's q is brought to [2^14, 2^15) by a power of two (halves hold it exactly down to 2^-28 of its largest
// element), the key's 2^ek multiplies the score, and the value's 2^ev joins the softmax weight:
//   w = s * scale * log2(e) + ev,  M = max w,  P = 2^(w - M + 15),  O = sum P code_v,  l = sum 2^(w - ev - M + 15),
//   out = O / l.  P <= 2^15 is rounded to half: 2^-12 relative down to 2^-29 of the largest weight, and the tokens that
//   fall below 2^-40 of it add nothing.  l's terms stay within fp32: |ev| <= 40.
#include "kv8_dev.cuh"

namespace gr {

constexpr int kQTile = 32;                                  // tokens per stage: two pages
constexpr int kQStageBytes = 2 * kQTile * 128;              // K codes, V codes
constexpr int kQExpBytes = 2 * kQTile;                      // K exponents, V exponents
constexpr int kQStages = 3;
constexpr int kQMaxWarps = 8;
constexpr size_t kQTicketBytes = 65536;                     // tickets of 16384 (request, K/V head) pairs

__device__ __forceinline__ void mma_16816_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void bulk_load16(void* dst, const void* src, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], 16, [%2];" ::"r"(
                   smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Two codes (bytes 2h, 2h + 1 of w) as a half2.
template <int FMT, int H>
__device__ __forceinline__ uint32_t kv_half2(uint32_t w) {
  if (FMT == GR_KV_E4M3) return e4m3x2_to_half2(H ? w >> 16 : w);
  const uint32_t a = __byte_perm(w, 0x64646464u, H ? 0x4342 : 0x4140);  // w holds x ^ 0x80 bytes
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&a), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <int FMT>
__device__ __forceinline__ uint32_t kv_biased(uint32_t w) {
  return FMT == GR_KV_INT8 ? w ^ 0x80808080u : w;
}

struct KvAttnSmem {  // offsets from the 1024-aligned start
  int ring, exps, scales, bars, total;
};
__host__ __device__ inline KvAttnSmem kv_attn_smem(int groups, int n_mt) {
  KvAttnSmem s;
  const int ring = groups * kQStages * kQStageBytes;
  const int merge = groups * n_mt * 16 * 130 * 4;  // O [rows][128], m and l, of every group (reuses the ring)
  s.ring = 0;
  s.exps = ring > merge ? ring : (merge + 1023) / 1024 * 1024;
  s.scales = s.exps + groups * kQStages * kQExpBytes;
  s.bars = s.scales + groups * n_mt * kQTile * 8;
  s.total = s.bars + groups * kQStages * 16 + 16;
  return s;
}

template <int FMT>
__global__ void __launch_bounds__(32 * kQMaxWarps) kv8_attention_kernel(const __grid_constant__ CUtensorMap tmk,
                                                                       const __grid_constant__ CUtensorMap tmv,
                                                                       const KvAttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int G = p.n_q_heads / p.n_kv_heads;
  const int R = G * p.K;
  const int n_mt = (R + 15) / 16;
  const int R_pad = n_mt * 16;
  const int NG = p.groups;
  const KvAttnSmem lay = kv_attn_smem(NG, n_mt);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = warp / n_mt, mt = warp - grp * n_mt;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + lay.bars) + grp * kQStages;
  uint64_t* empty = full + NG * kQStages;
  int* flag = reinterpret_cast<int*>(smem + lay.bars + NG * kQStages * 16);
  if (mt == 0 && lane == 0) {
    for (int s = 0; s < kQStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, n_mt);
    }
    fence_mbar_init();
  }
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmk);
    tma_prefetch_desc(&tmv);
    pdl_trigger();
  }
  __syncthreads();
  pdl_wait();

  const int64_t base64 = p.seq_lens[b] + p.base_add;
  const int64_t cap = static_cast<int64_t>(p.pt_stride) * 16;
  const int64_t end64 = base64 + p.K;
  if (end64 > cap && threadIdx.x == 0 && split == 0) report(p.status, GR_ERR_BAD_PAGE);
  const int base = static_cast<int>(min(max(base64, static_cast<int64_t>(-p.K)), cap));
  const int L = static_cast<int>(min(max(end64, static_cast<int64_t>(0)), cap));  // the last row's limit
  const int n_active = max(1, (L + p.chunk - 1) / p.chunk);
  if (split >= n_active) return;
  const int kv_beg = split * p.chunk;
  const int kv_end = min(L, kv_beg + p.chunk);
  const int n_tiles = kv_end > kv_beg ? (kv_end - kv_beg + kQTile - 1) / kQTile : 0;
  const int my_tiles = n_tiles > grp ? (n_tiles - grp + NG - 1) / NG : 0;
  const int* pt = p.page_table + static_cast<int64_t>(b) * p.pt_stride;
  const int last_page = (L - 1) >> 4;

  // ---- producer: lanes 0-7 of the group's first warp issue a stage (K and V tiles of two pages, their exponents)
  uint8_t* ring = smem + lay.ring + grp * kQStages * kQStageBytes;
  uint8_t* exps = smem + lay.exps + grp * kQStages * kQExpBytes;
  const bool producer = mt == 0;
  auto page_of = [&](int i) {  // page id of this lane's copy in the group's tile i (in range: checked here)
    if (!producer || lane >= 8 || i >= my_tiles) return 0;
    const int slot = min(((kv_beg + (grp + i * NG) * kQTile) >> 4) + (lane & 1), last_page);
    const int pg = __ldg(pt + slot);
    if (static_cast<unsigned>(pg) >= static_cast<unsigned>(p.n_pages)) {
      report(p.status, GR_ERR_BAD_PAGE);
      return 0;
    }
    return pg;
  };
  auto issue = [&](int i, int pg) {
    const int st = i % kQStages;
    if (lane == 0) mbar_arrive_expect_tx(full + st, kQStageBytes + kQExpBytes);
    __syncwarp();
    uint8_t* stage = ring + st * kQStageBytes;
    const int half = lane & 1;
    const int64_t row = (static_cast<int64_t>(pg) * p.n_kv_heads + kvh) * 16;
    if (lane < 2) tma_load_2d(stage + half * 2048, &tmk, full + st, 0, static_cast<int>(row));
    else if (lane < 4) tma_load_2d(stage + kQTile * 128 + half * 2048, &tmv, full + st, 0, static_cast<int>(row));
    else if (lane < 6) bulk_load16(exps + st * kQExpBytes + half * 16, p.k_exp + row, full + st);
    else if (lane < 8) bulk_load16(exps + st * kQExpBytes + kQTile + half * 16, p.v_exp + row, full + st);
  };
  if (producer) {
    for (int i = 0; i < kQStages - 1; ++i)
      if (i < my_tiles) issue(i, page_of(i));
  }
  int next_page = page_of(kQStages - 1);

  // ---- this lane's two query rows, as halves
  const int c = lane & 3, n = lane >> 2;
  const int j0 = mt * 16 + n;
  uint32_t qf[2][16];   // [row][k-step * 2 + half of the step's 4 dims]
  float coef[2];
  int lim[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = j0 + 8 * h;
    const int g = r / p.K, j = r - g * p.K;
    float x[32];
    if (r < R) {
      const __nv_bfloat16* src = p.q + ((static_cast<int64_t>(b) * p.K + j) * p.n_q_heads + kvh * G + g) * 128;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(src + (u >> 1) * 64 + c * 16) + (u & 1));
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[u * 8 + 2 * e] = __uint_as_float(w[e] << 16);
          x[u * 8 + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
      }
      lim[h] = p.draft ? ((j == 0 && p.draft == 1) ? base + 1 : base + p.K) : base + j + 1;
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) x[e] = 0.f;
      lim[h] = L;
    }
    uint32_t am = 0;
#pragma unroll
    for (int e = 0; e < 32; ++e) am = max(am, __float_as_uint(x[e]) & 0x7fffffffu);
    am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
    am = max(am, __shfl_xor_sync(0xffffffffu, am, 2));
    const int sh = max(-112, min(112, static_cast<int>(am >> 23) - 127 - 14));  // q * 2^-sh lies in [2^14, 2^15)
    const float f = exp2i(-sh);
    coef[h] = exp2i(sh) * p.scale_log2;
#pragma unroll
    for (int e = 0; e < 16; ++e) qf[h][e] = pack_half(x[2 * e] * f, x[2 * e + 1] * f);
  }
  const int min_lim = p.draft == 2 ? base + p.K : base + 1;

  float o[16][4];
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float2* scales = reinterpret_cast<float2*>(smem + lay.scales) + warp * kQTile;
  const int krow = (n >> 1) + (n & 1) * 4;                 // the token (of 8) this lane's K column stands for
  const int vchunk = (n >> 1) | ((n & 1) << 2);            // the 16-dim chunk this lane's V column stands for
  bool dead = false;

  for (int i = 0; i < my_tiles; ++i) {
    const int st = i % kQStages;
    // refill the stage of the tile before this one, once every warp of the group has read it
    if (producer && i + kQStages - 1 < my_tiles) {
      const int nx = i + kQStages - 1;
      if (i > 0 && n_mt > 1 && !mbar_wait(empty + nx % kQStages, ((i - 1) / kQStages) & 1, p.status, GR_ERR_TIMEOUT))
        dead = true;
      __syncwarp();
      issue(nx, next_page);
      next_page = page_of(nx + 1);
    }
    if (!mbar_wait(full + st, (i / kQStages) & 1, p.status, GR_ERR_TIMEOUT)) dead = true;
    const uint8_t* kt = ring + st * kQStageBytes;
    const uint8_t* vt = kt + kQTile * 128;
    const int8_t* et = reinterpret_cast<const int8_t*>(exps + st * kQExpBytes);
    const int t0 = kv_beg + (grp + i * NG) * kQTile;
    const bool partial = t0 + kQTile > min(min_lim, kv_end);
    {
      const int ev = et[kQTile + lane];
      scales[lane] = make_float2(kv_scale(et[lane]), ev == kKvExpBad ? __int_as_float(0x7fc00000) : static_cast<float>(ev));
    }
    __syncwarp();

    // S: 4 column tiles of 8 tokens
    float s[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
      const int row = t * 8 + krow;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 raw = *reinterpret_cast<const uint4*>(kt + sw128(row, c + 4 * h));
        const uint32_t w[4] = {kv_biased<FMT>(raw.x), kv_biased<FMT>(raw.y), kv_biased<FMT>(raw.z),
                               kv_biased<FMT>(raw.w)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int ks = h * 4 + e;
          const uint32_t a[4] = {qf[0][2 * ks], qf[1][2 * ks], qf[0][2 * ks + 1], qf[1][2 * ks + 1]};
          mma_16816_f16(s[t], a, kv_half2<FMT, 0>(w[e]), kv_half2<FMT, 1>(w[e]));
        }
      }
    }
    // weights: w = s * coef * 2^ek + ev; column e of tile t is token t * 8 + c + 4 * (e & 1), row e >> 1
    float ev[4][2];
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 f = scales[t * 8 + c + 4 * e];
        ev[t][e] = f.y;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float w = fmaf(s[t][2 * h + e], coef[h] * f.x, f.y);
          if (partial) {
            const int tok = t0 + t * 8 + c + 4 * e;
            if (tok >= lim[h] || tok >= kv_end) w = -INFINITY;
          }
          s[t][2 * h + e] = w;
          mx[h] = fmaxf(mx[h], w);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
    }
    if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float al = m[h] == -INFINITY ? 0.f : ex2_approx(m[h] - mx[h]);
        m[h] = mx[h];
        l[h] *= al;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          o[x][2 * h] *= al;
          o[x][2 * h + 1] *= al;
        }
      }
    }
    const float r0 = (m[0] == -INFINITY ? 0.f : m[0]) - 15.f, r1 = (m[1] == -INFINITY ? 0.f : m[1]) - 15.f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float w0 = s[t][e] - r0, w1 = s[t][2 + e] - r1;
        float l0 = ex2_approx(w0 - ev[t][e]), l1 = ex2_approx(w1 - ev[t][e]);
        if (partial) {  // a hidden token's exponent may be that of a bad row, or of no row
          if (w0 == -INFINITY) l0 = 0.f;
          if (w1 == -INFINITY) l1 = 0.f;
        }
        l[0] += l0;
        l[1] += l1;
        s[t][e] = ex2_approx(w0);
        s[t][2 + e] = ex2_approx(w1);
      }
    }
    // O += P V, a page (16 tokens) at a time
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      uint32_t a[4];
      a[0] = pack_half(s[2 * pg][0], s[2 * pg][1]);
      a[1] = pack_half(s[2 * pg][2], s[2 * pg][3]);
      a[2] = pack_half(s[2 * pg + 1][0], s[2 * pg + 1][1]);
      a[3] = pack_half(s[2 * pg + 1][2], s[2 * pg + 1][3]);
      uint4 raw[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int row = pg * 16 + u * 4 + c;
        raw[u] = *reinterpret_cast<const uint4*>(vt + sw128(row, vchunk));
        if (partial && t0 + row >= kv_end) raw[u] = make_uint4(0, 0, 0, 0);  // unwritten slots: any bytes, NaN codes too
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t v0 = kv_biased<FMT>(w == 0 ? raw[0].x : (w == 1 ? raw[0].y : (w == 2 ? raw[0].z : raw[0].w)));
        const uint32_t v1 = kv_biased<FMT>(w == 0 ? raw[1].x : (w == 1 ? raw[1].y : (w == 2 ? raw[1].z : raw[1].w)));
        const uint32_t v2 = kv_biased<FMT>(w == 0 ? raw[2].x : (w == 1 ? raw[2].y : (w == 2 ? raw[2].z : raw[2].w)));
        const uint32_t v3 = kv_biased<FMT>(w == 0 ? raw[3].x : (w == 1 ? raw[3].y : (w == 2 ? raw[3].z : raw[3].w)));
        // bytes (dim, token pair): x holds dims 0, 1 of tokens c, c+4, y of tokens c+8, c+12
        const uint32_t x0 = __byte_perm(v0, v1, 0x5140), y0 = __byte_perm(v2, v3, 0x5140);
        const uint32_t x1 = __byte_perm(v0, v1, 0x7362), y1 = __byte_perm(v2, v3, 0x7362);
        mma_16816_f16(o[4 * w], a, kv_half2<FMT, 0>(x0), kv_half2<FMT, 0>(y0));
        mma_16816_f16(o[4 * w + 1], a, kv_half2<FMT, 1>(x0), kv_half2<FMT, 1>(y0));
        mma_16816_f16(o[4 * w + 2], a, kv_half2<FMT, 0>(x1), kv_half2<FMT, 0>(y1));
        mma_16816_f16(o[4 * w + 3], a, kv_half2<FMT, 1>(x1), kv_half2<FMT, 1>(y1));
      }
    }
    __syncwarp();
    if (n_mt > 1 && lane == 0) mbar_arrive(empty + st);
  }
  if (dead && producer) {  // a wait ran out: give the copies in flight another limit each before the ring is reused
    for (int i = max(0, my_tiles - kQStages); i < my_tiles; ++i)
      mbar_wait(full + i % kQStages, (i / kQStages) & 1, p.status, GR_ERR_TIMEOUT);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
  }

  // ---- join the groups through shared memory (the ring is idle)
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem + lay.ring);      // [NG][R_pad][128]
  float* part_ml = part + NG * R_pad * 128;                     // [NG][R_pad][2]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float* dst = part + (grp * R_pad + j0 + 8 * h) * 128;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      *reinterpret_cast<float4*>(dst + c * 16 + u * 4) =
          make_float4(o[4 * u][2 * h], o[4 * u + 1][2 * h], o[4 * u + 2][2 * h], o[4 * u + 3][2 * h]);
      *reinterpret_cast<float4*>(dst + 64 + c * 16 + u * 4) =
          make_float4(o[4 * u][2 * h + 1], o[4 * u + 1][2 * h + 1], o[4 * u + 2][2 * h + 1], o[4 * u + 3][2 * h + 1]);
    }
    if (c == 0) {
      part_ml[(grp * R_pad + j0 + 8 * h) * 2] = m[h];
      part_ml[(grp * R_pad + j0 + 8 * h) * 2 + 1] = l[h];
    }
  }
  __syncthreads();
  const int nthr = blockDim.x;
  const int64_t slot0 = (static_cast<int64_t>(b) * p.n_kv_heads + kvh) * p.max_splits;
  auto store_out = [&](int r, int d4, float4 a, float inv) {
    const int g = r / p.K, j = r - g * p.K;
    __nv_bfloat16* dst = p.out + ((static_cast<int64_t>(b) * p.K + j) * p.n_q_heads + kvh * G + g) * 128 + d4 * 4;
    uint2 pk;
    pk.x = pack_bf16(a.x * inv, a.y * inv);
    pk.y = pack_bf16(a.z * inv, a.w * inv);
    *reinterpret_cast<uint2*>(dst) = pk;
  };
  for (int it = threadIdx.x; it < R * 32; it += nthr) {
    const int r = it >> 5, d4 = it & 31;
    float M = -INFINITY;
    for (int g = 0; g < NG; ++g) M = fmaxf(M, part_ml[(g * R_pad + r) * 2]);
    const float Ms = M == -INFINITY ? 0.f : M;
    float lsum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int g = 0; g < NG; ++g) {
      const float w = ex2_approx(part_ml[(g * R_pad + r) * 2] - Ms);
      const float4 v = *reinterpret_cast<const float4*>(part + (g * R_pad + r) * 128 + d4 * 4);
      lsum += w * part_ml[(g * R_pad + r) * 2 + 1];
      acc.x += w * v.x;
      acc.y += w * v.y;
      acc.z += w * v.z;
      acc.w += w * v.w;
    }
    if (n_active == 1) {
      store_out(r, d4, acc, lsum == 0.f ? 0.f : 1.f / lsum);
    } else {
      __stcg(reinterpret_cast<float4*>(p.ws_o + ((slot0 + split) * R_pad + r) * 128) + d4, acc);
      if (d4 == 0) __stcg(reinterpret_cast<float2*>(p.ws_ml) + (slot0 + split) * R_pad + r, make_float2(M, lsum));
    }
  }
  if (n_active == 1) return;

  // ---- the last split to arrive joins them, in split order
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    int* tk = p.ws_ticket + b * p.n_kv_heads + kvh;
    const bool last = atomicAdd(tk, 1) == n_active - 1;
    if (last) *tk = 0;
    *flag = last;
  }
  __syncthreads();
  if (!*flag) return;
  __threadfence();
  for (int r = warp; r < R; r += nthr >> 5) {
    const float2* ml = reinterpret_cast<const float2*>(p.ws_ml);
    float M = -INFINITY;
    for (int s2 = lane; s2 < n_active; s2 += 32) M = fmaxf(M, __ldcg(ml + (slot0 + s2) * R_pad + r).x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    const float Ms = M == -INFINITY ? 0.f : M;
    float lsum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s2 = 0; s2 < n_active; ++s2) {
      const float2 x = __ldcg(ml + (slot0 + s2) * R_pad + r);
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p.ws_o + ((slot0 + s2) * R_pad + r) * 128) + lane);
      const float w = ex2_approx(x.x - Ms);
      lsum += w * x.y;
      acc.x += w * v.x;
      acc.y += w * v.y;
      acc.z += w * v.z;
      acc.w += w * v.w;
    }
    store_out(r, lane, acc, lsum == 0.f ? 0.f : 1.f / lsum);
  }
}

size_t kv8_attention_ws_bytes(int bs, int rows, int n_kv_heads, int max_splits, size_t* o_off, size_t* ml_off) {
  const size_t r_pad = static_cast<size_t>((rows + 15) / 16) * 16;
  const size_t slots = static_cast<size_t>(bs) * n_kv_heads * max_splits;
  if (o_off) *o_off = kQTicketBytes;
  if (ml_off) *ml_off = kQTicketBytes + slots * r_pad * 512;
  return kQTicketBytes + slots * r_pad * 520;
}

template <int FMT>
static cudaError_t launch_kv8_attention_t(const CUtensorMap& tmk, const CUtensorMap& tmv, const KvAttnParams& p,
                                          int warps, size_t smem, cudaStream_t stream, bool pdl) {
  static PerDeviceOnce configured;
  cudaError_t e = once_per_device(configured, [] {
    cudaError_t r = cudaFuncSetAttribute(kv8_attention_kernel<FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         227 * 1024);
    if (r != cudaSuccess) return r;
    return cudaFuncSetAttribute(kv8_attention_kernel<FMT>, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.max_splits, p.n_kv_heads, p.bs);
  cfg.blockDim = dim3(32 * warps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv8_attention_kernel<FMT>, tmk, tmv, p);
}

// Warp groups of a CTA: as many as fit eight warps, four at most.
int kv8_attention_groups(int rows) {
  const int n_mt = (rows + 15) / 16;
  const int g = kQMaxWarps / n_mt;
  return g > 4 ? 4 : g;
}

cudaError_t launch_kv8_attention(const CUtensorMap& tmk, const CUtensorMap& tmv, KvAttnParams p, int format,
                                 cudaStream_t stream, bool pdl) {
  const int rows = p.n_q_heads / p.n_kv_heads * p.K;
  const int n_mt = (rows + 15) / 16;
  p.groups = kv8_attention_groups(rows);
  const size_t smem = 1024 + kv_attn_smem(p.groups, n_mt).total;
  return format == GR_KV_E4M3 ? launch_kv8_attention_t<GR_KV_E4M3>(tmk, tmv, p, p.groups * n_mt, smem, stream, pdl)
                              : launch_kv8_attention_t<GR_KV_INT8>(tmk, tmv, p, p.groups * n_mt, smem, stream, pdl);
}

}  // namespace gr

// Attention of one to a few new tokens per request over the paged 8-bit K/V cache (rows as kv8_dev.cuh defines them), split
// over the cache's length and joined, on tcgen05 without unpacking a code.
//
// Rows of one request and one K/V head: the GQA group's G query heads x K window rows (row r = g * K + j); visibility as
// in attention_dev.cuh (row_limit).  With one new token there are G rows: the work is reading the cache, 258 bytes per
// token and head, so the kernel is built to add nothing to that stream.  Both products take the codes as they lie in
// shared memory after TMA, as the tensor core's A operand, and the few query rows as its N side:
//   S [128 tokens x N1] = K [128 tokens x 128] Q^T        A: K tile, K-major
//   O [128 dims x N2]   = V^T [128 dims x 128 tokens] P^T  A: V tile, MN-major; P as its threads write it, MN-major
// A TMEM lane is then a token (S) or a dimension (O): one thread per token does that token's softmax for every row, with
// the token's two exponents as plain scalars, and one thread per dimension accumulates O in fp32 registers.
//
// The 8-bit B operands hold a row in several 8-bit parts, one column each, whose products are summed in fp32:
//   e4m3  q = q0 + q1 / 16, exact to 2^-22 of the row's largest element (q has 8 significant bits, a part 4);
//         p = p0 + p1 / 16 + p2 / 256, 2^-12 relative; accumulated in fp32.
//   int8  q and p in two signed digits to base 256, rounded to 2^-16 of the row's largest element and of the tile's largest
//         weight; accumulated exactly in int32, joined as hi * 256 + lo and added in fp32.
//   (bf16 rounding of the output is 2^-9 relative.)
// Scales: a row's q is brought to the parts' range by a factor that coef_r undoes; with a token's 2^ek, 2^ev:
//   w = s * coef_r * 2^ek + ev (base 2),  p = 2^(w - M_r),  O = sum p code_v,  l = sum p 2^-ev,  out = O / l.
// |ev| <= 40 keeps l: a token whose p underflows within a tile, or whose tile lies 2^126 below M_r, has a score at least 46
// binades below the best.  Sums from before a raise of M_r, and those of other splits, may hold most of l although their
// weights lie 2^126 below: they are scaled in two steps of half the factor, and joined by l, not by their references.
//
// P is measured from its own tile's maximum T_r, not the running one: its parts then resolve the tile's weights whatever the
// rest of the sequence holds (a first token that takes most of the attention would otherwise push every later weight
// below int8's two digits), and O and l take a tile in fp32 with the factor 2^(T_r - M_r).  M_r is the first tile's maximum,
// raised only where a tile's is 2^kQRaise above it: fp32 holds the rest, and the sums are hardly ever rescaled.  The largest
// l: a token adds up to 2^15 (its weight in P's units) 2^40 (2^-ev) 2^48, and a split's 2^13 tokens 2^116 together.
//
// CTA: (split, K/V head and block of at most 40 rows, request).  A thread per token (then per dimension) and row group: one
// group of four warps, or two that share the rows (launch_kv8_attention_f).  One warp issues the MMAs, one the TMA copies (8
// pages a 128-token tile, 2 KB of K and 2 KB of V each; ~85 cycles an issue, which on the MMA warp would sit between a
// tile's two products).  Per tile: S -> weights -> P to shared memory -> O -> registers.  K and V have rings of their own,
// so a tile's K half is refilled as soon as its scores exist, and the two or three CTAs of an SM cover each other's
// latencies.
//
// Measured (8 K/V heads of 2 query heads).  One row: 131,071 tokens of one request 50 us, 283 MB, 5.6 TB/s, where a plain
// sum of as many bytes takes 49.5; 64 requests of 288-4,128 tokens 54 us (291 MB): bound by the memory.  17 rows of these 64:
// 100 us int8, 116 e4m3, bound by the softmax threads: their instructions fill half of the issue slots, and a tile's chain
// (scores, maxima, weights, P, O) the time between.
#include <algorithm>
#include <type_traits>

#include "kv8_dev.cuh"

namespace gr {

constexpr int kQTile = 128;                                 // tokens per tile: eight pages
constexpr int kQHalf = kQTile * 128;                        // K or V codes of a tile
constexpr int kQStages = 2;                                 // K and V rings (the product barriers are as many)
constexpr int kQExpStages = 4;                              // tiles' exponents
constexpr int kQMaxRows = 40;                               // rows of a CTA
constexpr float kQRaise = 48.f;                             // binades of a tile's maximum above the sums' reference
static_assert(kKv8MaxChunk <= 1 << 13 && 15 - kKvExpMin + kQRaise + 13 < 127, "the softmax sum stays below 2^127");

// A ticket a (request, K/V head, row block): the fewest blocks that hold the rows, or more of them for at most two CTAs an SM
// in all.  The same place for every shape: a workspace serves calls of different ones, and only tickets are zero between calls.
constexpr size_t kQTicketBytes = static_cast<size_t>(kKv8MaxPairs) * ((kKv8MaxRows + kQMaxRows - 1) / kQMaxRows) * sizeof(int);

// H groups of RH rows, each padded to RP (a multiple of four; the padding has columns, but no arithmetic).  Columns: S has
// part k of a group's row r at group * 2 * RP + k * RP + r, P likewise with every group padded to 16 columns.
template <int FMT, int RH, int H>
struct KvAttnShape {
  static constexpr int RP = (RH + 3) / 4 * 4, RT = RP * H;
  static constexpr int p_parts = FMT == GR_KV_E4M3 ? 3 : 2;
  static constexpr int p_cols = (p_parts * RP + 15) / 16 * 16;
  static constexpr int n1 = (2 * RT + 15) / 16 * 16;
  static constexpr int n2 = p_cols * H;
  static constexpr int tmem_cols = n1 + n2 <= 32 ? 32 : (n1 + n2 <= 64 ? 64 : (n1 + n2 <= 128 ? 128 : 256));
  static constexpr int threads = 128 * H + 64;
  // shared memory, from a 1024-aligned start
  static constexpr int k = 0;
  static constexpr int v = k + kQStages * kQHalf;
  static constexpr int q = v + kQStages * kQHalf;           // [n1][128], 128-byte swizzle
  static constexpr int p = q + n1 * 128;                    // [n2 / 16][128 tokens][16]
  static constexpr int exps = p + n2 * 128;                 // [kQExpStages][K, V][128]
  static constexpr int xm = exps + kQExpStages * 2 * kQTile;  // [4][RT] warp maxima of a tile; at the end, the sums l
  static constexpr int coef = xm + RT * 16;                 // [RT] score scale
  static constexpr int ref = coef + RT * 4;                 // [RT] (weights' top) - T_r
  static constexpr int alpha = ref + RT * 4;                // [RT] root of the factor of the sums so far
  static constexpr int beta = alpha + RT * 4;               // [RT] factor of the tile's sums
  static constexpr int lim = beta + RT * 4;                 // [RT] row limits
  static constexpr int pages = lim + RT * 4;                // [kKv8MaxChunk / 16] first code row of each page
  static constexpr int bars = (pages + kKv8MaxChunk / 4 + 15) / 16 * 16;
  static constexpr int bytes = 1024 + bars + (2 * kQStages + kQExpStages + 5) * 8 + 16;
  static constexpr bool ordered = RH > 8;                   // may take requests by length
  static_assert(n1 + n2 <= 256, "two CTAs share an SM's 512 columns");
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(src))
               : "memory");
}
// Arrives on the barrier once this thread's copies so far have landed (one of the barrier's expected arrivals).
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// One thread of the warp, the same each time; all 32 lanes take part.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
template <int FMT>
__device__ __forceinline__ void tc_mma_codes(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  if (FMT == GR_KV_E4M3)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Instruction descriptor of the 8-bit kinds: fp32 / int32 result, e4m3 or signed 8-bit inputs, M = 128; both operands
// K-major or both MN-major.
template <int FMT>
__device__ constexpr uint32_t idesc_codes(int n, bool mn) {
  return (FMT == GR_KV_E4M3 ? (1u << 4) : ((2u << 4) | (1u << 7) | (1u << 10))) | (mn ? (1u << 15) | (1u << 16) : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}
// N consecutive TMEM columns of this thread's lane (N a multiple of 4); wait with tmem_ld_done.
template <int N>
__device__ __forceinline__ void tmem_ld_cols(uint32_t addr, uint32_t* r) {
  if constexpr (N >= 16) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
    if constexpr (N > 16) tmem_ld_cols<N - 16>(addr + 16, r + 16);
  } else if constexpr (N >= 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
    if constexpr (N > 8) tmem_ld_cols<N - 8>(addr + 8, r + 8);
  } else {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
  }
}
// Completes this thread's TMEM loads; no use of r can be scheduled before it.
template <int N>
__device__ __forceinline__ void tmem_ld_done(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
// f(first row, rows) over a group's RP (padded) rows: at once up to 12, else in two parts, so that a tile's TMEM columns and
// the thread's sums fit the registers together.
template <int RP, typename F>
__device__ __forceinline__ void rows_by_parts(F f) {
  constexpr int first = RP <= 12 ? RP : (RP / 2 + 3) / 4 * 4;
  f(std::integral_constant<int, 0>(), std::integral_constant<int, first>());
  if constexpr (first < RP) f(std::integral_constant<int, first>(), std::integral_constant<int, RP - first>());
}
__device__ __forceinline__ float warp_max(float v) {
  float r;
  // NaNs are ignored; volatile: every lane has to take part, wherever the result is used
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// The exponent of a softmax sum (2^-33 .. 2^116); 0 for none, and for NaN.
__device__ __forceinline__ int sum_exp(float l) {
  const int e = (__float_as_int(l) >> 23 & 0xff) - 127;
  return e == -127 || e == 128 ? 0 : e;
}
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool named_any(int id, int threads, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(x)), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}
// MN-major operand without a swizzle: [16 MN elements][K index] blocks, each K index 16 bytes; 128 bytes to the next 8 K
// indices (leading), block_bytes to the next 16 MN elements (stride).
__device__ __forceinline__ uint64_t smem_desc_mn16(uint32_t addr, uint32_t block_bytes) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | (static_cast<uint64_t>(128 >> 4) << 16) |
         (static_cast<uint64_t>(block_bytes >> 4) << 32) | (static_cast<uint64_t>(1) << 46);
}
// Four scaled q values to two words of four codes, one a part.
template <int FMT>
__device__ __forceinline__ void split_q(const float (&x)[4], uint32_t* part) {
  if (FMT == GR_KV_E4M3) {  // |x| < 256
    part[0] = kv_pack<GR_KV_E4M3>(x);
    float rest[4];
    const uint32_t h01 = e4m3x2_to_half2(part[0]), h23 = e4m3x2_to_half2(part[0] >> 16);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h01));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&h23));
    rest[0] = (x[0] - a.x) * 16.f;
    rest[1] = (x[1] - a.y) * 16.f;
    rest[2] = (x[2] - b.x) * 16.f;
    rest[3] = (x[3] - b.y) * 16.f;
    part[1] = kv_pack<GR_KV_E4M3>(rest);
  } else {  // |x| <= 32639: digits in [-128, 127]
    part[0] = part[1] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t t = (static_cast<uint32_t>(__float2int_rn(x[i])) + 0x8080u) ^ 0x8080u;
      part[0] |= ((t >> 8) & 0xffu) << (8 * i);
      part[1] |= (t & 0xffu) << (8 * i);
    }
  }
}

struct Kv8Place {
  int b, kvh, blk, r0, R, n_active;
};

template <int FMT, int RH, int H>
__global__ void __launch_bounds__(128 * H + 64, H == 2 ? 2 : 3) kv8_attention_kernel(
    const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const KvAttnParams p) {
  using Sh = KvAttnShape<FMT, RH, H>;
  constexpr int RP = Sh::RP, RT = Sh::RT;
  constexpr int kMmaWarp = 4 * H, kCopyWarp = kMmaWarp + 1, kSoft = 128 * H;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + Sh::bars);
  uint64_t* v_full = k_full + kQStages;
  uint64_t* s_full = v_full + kQStages;
  // products completed, one barrier per stage parity: a waiter two tiles behind must not mistake the phase
  uint64_t* o_full = s_full + 2;
  uint64_t* p_full = o_full + 2;
  uint64_t* e_full = p_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(e_full + kQExpStages);
  int* flag = reinterpret_cast<int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < 2 * kQStages; ++s) mbar_init(k_full + s, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full + s, 1);
      mbar_init(o_full + s, 1);
    }
    mbar_init(p_full, kMmaWarp);
    for (int s = 0; s < kQExpStages; ++s) mbar_init(e_full + s, 32);
    fence_mbar_init();
    tma_prefetch_desc(&tmk);
    tma_prefetch_desc(&tmv);
  }
  pdl_wait();

  // x = K/V head and row block, y = request, z = split: the splits that only the longest requests have launch last
  const int split = blockIdx.z;
  int b = blockIdx.y;
  volatile int* request = flag + 1;
  if (Sh::ordered && p.longest_first) {
    // the split's requests by length: the blockIdx.y-th longest (equal ones by index), by counting
    int* keys = reinterpret_cast<int*>(smem + Sh::pages);
    int key = -1;
    if (tid < p.bs) {
      const int64_t n = max(static_cast<int64_t>(0), min(p.seq_lens[tid] + p.base_add + p.K,
                                                         static_cast<int64_t>(kKv8MaxChunk) * kKv8MaxSplits));
      key = static_cast<int>(n) * kKv8MaxSort + kKv8MaxSort - 1 - tid;
    }
    if (tid < kKv8MaxSort) keys[tid] = key;
    // idle splits leave: fewer requests than blockIdx.y reach past the split's start
    const int least = split == 0 ? 0 : (split * p.chunk + 1) * kKv8MaxSort;
    if (b >= __syncthreads_count(key >= least)) return;
    if (tid < p.bs) {
      int before = 0;
#pragma unroll 4
      for (int i = 0; i < (p.bs + 3) >> 2; ++i) {
        const int4 x = reinterpret_cast<const int4*>(keys)[i];
        before += (x.x > key) + (x.y > key) + (x.z > key) + (x.w > key);
      }
      if (before == b) *request = tid;
    }
    __syncthreads();
    b = *request;
  }
  const int kvh = blockIdx.x / p.row_blocks, blk = blockIdx.x - kvh * p.row_blocks;
  const int G = p.group, R_all = p.group * p.K;
  const int r0 = blk * p.rows_per_block;
  const int R = min(p.rows_per_block, R_all - r0);  // this CTA's rows r0 .. r0 + R - 1
  const int64_t base64 = p.seq_lens[b] + p.base_add;
  const int64_t cap = static_cast<int64_t>(p.pt_stride) * 16;
  const int64_t end64 = base64 + p.K;
  if (tid == 0 && split == 0) {
    if (end64 > cap) report(p.status, GR_ERR_BAD_PAGE);
    else if (end64 > static_cast<int64_t>(p.chunk) * p.max_splits) report(p.status, GR_ERR_ARG);
  }
  const int base = static_cast<int>(min(max(base64, static_cast<int64_t>(-p.K)), cap));
  const int L = static_cast<int>(min(max(end64, static_cast<int64_t>(0)), cap));  // the last row's limit
  const int n_active = min(p.max_splits, max(1, (L + p.chunk - 1) / p.chunk));
  if (split >= n_active) return;
  // what the code behind the tile loop needs is found again there, not held in registers through the loop
  if (tid == 0) request[1] = n_active;
  auto where = [&] {
    Kv8Place w;
    uint32_t x;
    asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(x));
    w.b = Sh::ordered && p.longest_first ? request[0] : static_cast<int>(blockIdx.y);
    w.kvh = static_cast<int>(x) / p.row_blocks;
    w.blk = static_cast<int>(x) - w.kvh * p.row_blocks;
    w.r0 = w.blk * p.rows_per_block;
    w.R = min(p.rows_per_block, p.group * p.K - w.r0);
    w.n_active = request[1];
    return w;
  };
  // TMEM is taken before the dependent launch is released: a CTA of a later kernel (which may wait for this grid) can
  // then never hold the columns this CTA is waiting for
  if (warp == kMmaWarp) tmem_alloc(tmem_slot, Sh::tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (tid == 0) pdl_trigger();
  const int kv_beg = split * p.chunk;
  const int kv_end = min(L, kv_beg + p.chunk);
  const int n_tiles = kv_end > kv_beg ? (kv_end - kv_beg + kQTile - 1) / kQTile : 0;

  // ---- first code row of each of the chunk's pages; page ids are checked here
  int* pages = reinterpret_cast<int*>(smem + Sh::pages);
  for (int k = tid; k < n_tiles * 8; k += Sh::threads) {
    int id = (kv_beg >> 4) + k <= (kv_end - 1) >> 4
                 ? __ldg(p.page_table + static_cast<int64_t>(b) * p.pt_stride + (kv_beg >> 4) + k) : 0;
    if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.n_pages)) {
      report(p.status, GR_ERR_BAD_PAGE);
      id = 0;
    }
    pages[k] = (id * p.n_kv_heads + kvh) * 16;
  }
  if (warp < kMmaWarp) {
    // ---- query rows to shared memory, in parts: a warp per row, each step for all of a warp's rows (their latencies overlap)
    float* coef = reinterpret_cast<float*>(smem + Sh::coef);
    int* lim = reinterpret_cast<int*>(smem + Sh::lim);
    constexpr int per_warp = (RT + kMmaWarp - 1) / kMmaWarp;
    uint2 raw[per_warp];
    int limit[per_warp];
    float x[per_warp][4], f[per_warp], back[per_warp];
#pragma unroll
    for (int u = 0; u < per_warp; ++u) {
      const int r = warp + u * kMmaWarp;
      const int row = r / RP * RH + r % RP;  // of the CTA's
      const bool live = r % RP < RH && row < R;
      const int g = (r0 + min(row, R - 1)) / p.K, j = (r0 + min(row, R - 1)) - g * p.K;
      raw[u] = __ldg(reinterpret_cast<const uint2*>(
          p.q + ((static_cast<int64_t>(b) * p.K + j) * p.n_q_heads + kvh * G + g) * 128) + lane);
      limit[u] = live ? min(kv_end, p.draft ? ((j == 0 && p.draft == 1) ? base + 1 : base + p.K) : base + j + 1) : 0;
      if (!live) raw[u] = make_uint2(0u, 0u);
    }
#pragma unroll
    for (int u = 0; u < per_warp; ++u) {
      x[u][0] = __uint_as_float(raw[u].x << 16);
      x[u][1] = __uint_as_float(raw[u].x & 0xffff0000u);
      x[u][2] = __uint_as_float(raw[u].y << 16);
      x[u][3] = __uint_as_float(raw[u].y & 0xffff0000u);
      uint32_t am = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) am = max(am, __float_as_uint(x[u][i]) & 0x7fffffffu);
      am = __reduce_max_sync(0xffffffffu, am);
      // e4m3: the largest |q| to [2^7, 2^8), exactly; int8: to 32639, two digits' largest, rounded with the digits.  A row
      // with a NaN or an infinity scores NaN.
      if (FMT == GR_KV_E4M3) {
        const int sh = max(-120, static_cast<int>(am >> 23) - 127 - 7);  // at most 120
        f[u] = exp2i(-sh);
        back[u] = exp2i(sh);
      } else {
        const float a = fmaxf(__uint_as_float(am), 1e-30f);
        f[u] = 32639.f / a * 0.9999995f;  // not above 32639 after its rounding
        back[u] = 1.f / f[u];
      }
      if (am >= 0x7f800000u) {
        f[u] = 0.f;
        back[u] = __int_as_float(0x7fc00000);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[u][i] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < per_warp; ++u) {
      const int r = warp + u * kMmaWarp;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[u][i] *= f[u];
      uint32_t part[2];
      split_q<FMT>(x[u], part);
      if (RT % kMmaWarp == 0 || r < RT) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int col = r / RP * 2 * RP + k * RP + r % RP;
          *reinterpret_cast<uint32_t*>(smem + Sh::q + sw128(col, lane >> 2) + (lane & 3) * 4) = part[k];
        }
        if (lane == 0) {
          coef[r] = back[u] * p.scale_log2;
          lim[r] = limit[u];
        }
      }
    }
    fence_proxy_async_smem();
  }
  __syncthreads();

  if (warp == kCopyWarp) {
    // ---- copies, by one elected thread (the compiler keeps their operands uniform)
    const int n_pages = (kv_end - kv_beg + 15) >> 4;
    auto copy = [&](const CUtensorMap* map, int at, uint64_t* bars, int i) {
      if (elect_one()) {
        uint64_t* bar = bars + i % kQStages;
        const int n = min(8, n_pages - i * 8);
        mbar_arrive_expect_tx(bar, n * 2048);
        uint8_t* dst = smem + at + (i % kQStages) * kQHalf;
        const int4 a = *reinterpret_cast<const int4*>(pages + i * 8), c = *reinterpret_cast<const int4*>(pages + i * 8 + 4);
        const int row[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < n) tma_load_2d(dst + k * 2048, map, bar, 0, row[k]);
      }
      __syncwarp();
    };
    int nk = 0, nv = 0;  // tiles whose copies are issued
    for (bool ok = true; ok && nv < n_tiles;) {
      // a K stage is free once its tile's scores exist, a V stage once its tile's second product has completed
      if (nk >= kQStages) ok = mbar_wait(s_full + (nk & 1), ((nk - 2) >> 1) & 1, p.status, GR_ERR_TIMEOUT);
      if (ok) copy(&tmk, Sh::k, k_full, nk++);
      if (ok && nv >= kQStages) ok = mbar_wait(o_full + (nv & 1), ((nv - 2) >> 1) & 1, p.status, GR_ERR_TIMEOUT);
      if (ok) copy(&tmv, Sh::v, v_full, nv++);
    }
    // no copy may still be landing in shared memory when the CTA leaves (after a wait that ran out, too)
    for (int i = max(0, nk - kQStages); i < nk; ++i)
      mbar_wait(k_full + i % kQStages, (i / kQStages) & 1, p.status, GR_ERR_TIMEOUT);
    for (int i = max(0, nv - kQStages); i < nv; ++i)
      mbar_wait(v_full + i % kQStages, (i / kQStages) & 1, p.status, GR_ERR_TIMEOUT);
  } else if (warp == kMmaWarp) {
    // ---- MMAs, by one elected thread; the exponents' copies, 16 bytes a lane and two tiles ahead (plain loads by the
    // threads that use them were waited for with the next TMEM load: a memory latency a tile)
    bool ok = true;
    const int n_pages = (kv_end - kv_beg + 15) >> 4;
    auto copy_exps = [&](int i) {
      const int pg = i * 8 + (lane & 7);
      if (lane < 16 && pg < n_pages)
        cp_async16(smem + Sh::exps + (i % kQExpStages) * 2 * kQTile + lane * 16, (lane < 8 ? p.k_exp : p.v_exp) + pages[pg]);
      cp_async_arrive(e_full + i % kQExpStages);
    };
    for (int i = 0; i < min(2, n_tiles); ++i) copy_exps(i);
    constexpr uint32_t id_s = idesc_codes<FMT>(Sh::n1, false), id_o = idesc_codes<FMT>(Sh::n2, true);
    const uint64_t kd = smem_desc_sw128(smem_u32(smem + Sh::k));
    const uint64_t vd = smem_desc_sw128_mn(smem_u32(smem + Sh::v), kQHalf);
    const uint64_t qd = smem_desc_sw128(smem_u32(smem + Sh::q));
    const uint64_t pd = smem_desc_mn16(smem_u32(smem + Sh::p), kQTile * 16);
    for (int i = 0; i < n_tiles; ++i) {
      const uint32_t so = (static_cast<uint32_t>(i % kQStages) * kQHalf) >> 4;
      ok = ok && mbar_wait(k_full + i % kQStages, (i / kQStages) & 1, p.status, GR_ERR_TIMEOUT);
      tc_fence_after();
      if (ok && elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k)  // 32 dims a step: 32 bytes of a row
          tc_mma_codes<FMT>(tmem, kd + so + 2 * k, qd + 2 * k, id_s, k != 0);
        tc_commit(s_full + (i & 1));
      }
      __syncwarp();
      if (i + 2 < n_tiles) copy_exps(i + 2);  // tile i - 2's slot: its weights are long made
      ok = ok && mbar_wait(v_full + i % kQStages, (i / kQStages) & 1, p.status, GR_ERR_TIMEOUT);
      ok = ok && mbar_wait(p_full, i & 1, p.status, GR_ERR_TIMEOUT);
      tc_fence_after();
      if (ok && elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k)  // 32 tokens a step: 4 KB of V rows, 512 bytes of P
          tc_mma_codes<FMT>(tmem + Sh::n1, vd + so + 256 * k, pd + 32 * k, id_o, k != 0);
        tc_commit(o_full + (i & 1));
      }
      __syncwarp();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // ---- one thread per token (weights), then per dimension (output), for the rows of its group
    const int t128 = tid & 127, grp = H == 1 ? 0 : warp >> 2, rb = grp * RP;
    const float* coef = reinterpret_cast<const float*>(smem + Sh::coef) + rb;
    const int* lim = reinterpret_cast<const int*>(smem + Sh::lim) + rb;
    float* refs = reinterpret_cast<float*>(smem + Sh::ref);
    float* alphas = reinterpret_cast<float*>(smem + Sh::alpha);
    float* betas = reinterpret_cast<float*>(smem + Sh::beta);
    float* xm = reinterpret_cast<float*>(smem + Sh::xm);
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane + grp * 2 * RP, t_o = t_lane + Sh::n1 + grp * Sh::p_cols;
    uint8_t* ps = smem + Sh::p + grp * Sh::p_cols * kQTile;
    const int min_lim = min(kv_end, p.draft == 2 ? base + p.K : base + 1);
    float o[RH], l[RH];
#pragma unroll
    for (int r = 0; r < RH; ++r) o[r] = l[r] = 0.f;
    float m_row = -INFINITY;  // threads 0 .. RT - 1: the row's running maximum
    bool ok = true;
    for (int i = 0; i < n_tiles; ++i) {
      const int t0 = kv_beg + i * kQTile, tok = t0 + t128;
      const bool partial = t0 + kQTile > min_lim;
      ok = ok && mbar_wait(s_full + (i & 1), (i >> 1) & 1, p.status, GR_ERR_TIMEOUT);
      tc_fence_after();
      ok = ok && mbar_wait(e_full + i % kQExpStages, (i / kQExpStages) & 1, p.status, GR_ERR_TIMEOUT);
      const int8_t* ex = reinterpret_cast<const int8_t*>(smem + Sh::exps + (i % kQExpStages) * 2 * kQTile);
      const int ek = ex[t128], ve = ex[kQTile + t128];
      const float fk = kv_scale(ek);
      const float ev = ve == kKvExpBad ? __int_as_float(0x7fc00000) : static_cast<float>(ve);
      const float unv = ve == kKvExpBad ? 1.f : exp2i(-ve);
      float w[RH];
      rows_by_parts<RP>([&](auto beg, auto num) {
        constexpr int r0 = decltype(beg)::value, n = decltype(num)::value;
        uint32_t s[2 * n];
        tmem_ld_cols<n>(t_s + r0, s);
        tmem_ld_cols<n>(t_s + RP + r0, s + n);
        tmem_ld_done(s);
#pragma unroll
        for (int r = 0; r < n; r += 4) {
          const float4 c = *reinterpret_cast<const float4*>(coef + r0 + r);
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[e] = FMT == GR_KV_E4M3 ? fmaf(__uint_as_float(s[n + r + e]), 1.f / 16, __uint_as_float(s[r + e]))
                                     : static_cast<float>(static_cast<int>(s[r + e]) * 256 + static_cast<int>(s[n + r + e]));
          const float cf[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (r0 + r + e < RH) w[r0 + r + e] = fmaf(x[e], cf[e] * fk, ev);
        }
      });
      if (partial) {
#pragma unroll
        for (int r = 0; r < RH; ++r)
          if (tok >= lim[r]) w[r] = -INFINITY;
        // an unwritten slot's value codes may be NaN codes: out of the product
        ok = ok && mbar_wait(v_full + i % kQStages, (i / kQStages) & 1, p.status, GR_ERR_TIMEOUT);
        if (grp == 0 && tok >= kv_end) {
          uint4* row = reinterpret_cast<uint4*>(smem + Sh::v + (i % kQStages) * kQHalf + t128 * 128);
#pragma unroll
          for (int k = 0; k < 8; ++k) row[k] = make_uint4(0, 0, 0, 0);
        }
      }
      // row maxima over the tile's 128 tokens: by warp, then one thread per row
#pragma unroll
      for (int r = 0; r < RH; r += 4) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = r + e < RH ? warp_max(w[r + e]) : 0.f;
        if (lane == 0) *reinterpret_cast<float4*>(xm + (warp & 3) * RT + rb + r) = make_float4(x[0], x[1], x[2], x[3]);
      }
      named_sync(1, kSoft);
      bool raised = false;
      if (tid < RT) {
        const float mt = fmaxf(fmaxf(xm[tid], xm[RT + tid]), fmaxf(xm[2 * RT + tid], xm[3 * RT + tid]));
        // mt = -inf: the row sees no token of this tile.  The sums' reference moves only when a tile is 2^kQRaise above it.
        raised = mt > m_row + kQRaise;
        alphas[tid] = raised ? ex2_approx(0.5f * (m_row - mt)) : 1.f;  // 0 from -inf
        if (raised) m_row = mt;
        betas[tid] = mt == -INFINITY ? 1.f : ex2_approx(mt - m_row);
        // e4m3 weights go up to 2^8, which comes with the reference while fp32 holds both (beyond, a score's step is half a
        // binade); int8's up to 1, brought to the digits as they are rounded
        refs[tid] = (FMT == GR_KV_E4M3 && fabsf(mt) < 0x1p22f ? 8.f : 0.f) - (mt == -INFINITY ? 0.f : mt);
      }
      __syncwarp();
      if (named_any(1, kSoft, raised)) {
#pragma unroll
        for (int r = 0; r < RH; ++r) {
          const float a = alphas[rb + r];
          o[r] = o[r] * a * a;
          l[r] = l[r] * a * a;
        }
      }
      // weights; P to shared memory, 16 (part, row) columns of a token in a vector
      uint32_t pw[Sh::p_cols / 4];
#pragma unroll
      for (int k = 0; k < Sh::p_cols / 4; ++k) pw[k] = 0;
#pragma unroll
      for (int r = 0; r < RH; r += 4) {
        const float4 rf = *reinterpret_cast<const float4*>(refs + rb + r);
        const float4 bt = *reinterpret_cast<const float4*>(betas + rb + r);
        const float rfs[4] = {rf.x, rf.y, rf.z, rf.w}, bts[4] = {bt.x, bt.y, bt.z, bt.w};
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (r + e >= RH) break;
          x[e] = ex2_approx(w[r + e] + rfs[e]);
          // a hidden token's exponent may be that of a bad row, or of no row: its weight is 0, and 2^-ev is finite
          l[r + e] = fmaf(x[e] * unv, bts[e], l[r + e]);
        }
        if (FMT == GR_KV_E4M3) {
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
            pw[(k * RP + r) / 4] = __byte_perm(lo, hi, 0x5410);
            if (k < 2) {
              const uint32_t h01 = e4m3x2_to_half2(lo), h23 = e4m3x2_to_half2(hi);
              const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h01));
              const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&h23));
              x[0] = (x[0] - a.x) * 16.f;
              x[1] = (x[1] - a.y) * 16.f;
              x[2] = (x[2] - c.x) * 16.f;
              x[3] = (x[3] - c.y) * 16.f;
            }
          }
        } else {
          // x times 32639 (two digits' largest) to two signed digits: the low 16 bits of that + 2^23 + 0x8080 are that + 0x8080,
          // each byte less 0x80 a digit
          uint32_t t[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) t[k] = __float_as_uint(fmaf(x[k], 32639.f, 8421504.f));
          const uint32_t a = __byte_perm(t[0], t[1], 0x5140), c = __byte_perm(t[2], t[3], 0x5140);  // lo lo hi hi
          pw[r / 4] = __byte_perm(a, c, 0x7632) ^ 0x80808080u;
          pw[(RP + r) / 4] = __byte_perm(a, c, 0x5410) ^ 0x80808080u;
        }
      }
#pragma unroll
      for (int k = 0; k < Sh::p_cols / 16; ++k)
        *reinterpret_cast<uint4*>(ps + (k * kQTile + t128) * 16) =
            make_uint4(pw[4 * k], pw[4 * k + 1], pw[4 * k + 2], pw[4 * k + 3]);
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
      ok = ok && mbar_wait(o_full + (i & 1), (i >> 1) & 1, p.status, GR_ERR_TIMEOUT);
      tc_fence_after();
      rows_by_parts<RP>([&](auto beg, auto num) {
        constexpr int r0 = decltype(beg)::value, n = decltype(num)::value;
        uint32_t x[Sh::p_parts * n];
#pragma unroll
        for (int k = 0; k < Sh::p_parts; ++k) tmem_ld_cols<n>(t_o + k * RP + r0, x + k * n);
        tmem_ld_done(x);
#pragma unroll
        for (int r1 = 0; r1 < n; r1 += 4) {
          const float4 bt = *reinterpret_cast<const float4*>(betas + rb + r0 + r1);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = r1 + e;
            if (r0 + r >= RH) break;
            float y;
            if (FMT == GR_KV_E4M3)
              y = fmaf(fmaf(__uint_as_float(x[2 * n + r]), 1.f / 16, __uint_as_float(x[n + r])), 1.f / 16,
                       __uint_as_float(x[r]));
            else
              y = static_cast<float>(static_cast<int>(x[r]) * 256 + static_cast<int>(x[n + r]));
            o[r0 + r] = fmaf(y, e == 0 ? bt.x : (e == 1 ? bt.y : (e == 2 ? bt.z : bt.w)), o[r0 + r]);
          }
        }
      });
    }
    // ---- l over the 128 tokens, then this split's result
    const auto [b, kvh, blk, r0, R, n_active] = where();
    const int64_t slot0 = (static_cast<int64_t>(b) * p.n_kv_heads + kvh) * p.max_splits;
    float* part = reinterpret_cast<float*>(smem + Sh::k);  // [RT][128]; the last tile's scores are done with the ring
#pragma unroll
    for (int r = 0; r < RH; ++r) part[(rb + r) * kQTile + t128] = FMT == GR_KV_INT8 ? l[r] * 32639.f : l[r];  // O's units
    named_sync(1, kSoft);
    {
      constexpr int per_warp = (RT + kMmaWarp - 1) / kMmaWarp;
      float sum[per_warp];
#pragma unroll
      for (int u = 0; u < per_warp; ++u) {
        const float4 x = *reinterpret_cast<const float4*>(part + min(warp + u * kMmaWarp, RT - 1) * kQTile + lane * 4);
        sum[u] = (x.x + x.y) + (x.z + x.w);
      }
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) {
#pragma unroll
        for (int u = 0; u < per_warp; ++u) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], w);
      }
#pragma unroll
      for (int u = 0; u < per_warp; ++u)
        if (lane == 0 && warp + u * kMmaWarp < RT) xm[warp + u * kMmaWarp] = sum[u];
    }
    named_sync(1, kSoft);
    const int own = tid / RP * RH + tid % RP;  // a row thread's row
    if (n_active > 1 && tid < RT && tid % RP < RH && own < R)
      __stcg(reinterpret_cast<float2*>(p.ws_ml) + (slot0 + split) * R_all + r0 + own, make_float2(m_row, xm[tid]));
    if (n_active == 1) {
#pragma unroll
      for (int r = 0; r < RH; ++r) {
        if (grp * RH + r >= R) break;
        const float sum = xm[rb + r];
        const int g = (r0 + grp * RH + r) / p.K, j = (r0 + grp * RH + r) - g * p.K;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        p.out[((static_cast<int64_t>(b) * p.K + j) * p.n_q_heads + kvh * G + g) * 128 + t128] =
            __float2bfloat16(o[r] * inv);
      }
    } else {
      float* dst = p.ws_o + ((slot0 + split) * R_all + r0 + grp * RH) * 128 + t128;
#pragma unroll
      for (int r = 0; r < RH; ++r)
        if (grp * RH + r < R) __stcg(dst + r * 128, o[r] * exp2i(-sum_exp(xm[rb + r])));
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, Sh::tmem_cols);
  }

  // ---- the last split to arrive joins them, in split order
  const Kv8Place at = where();
  if (at.n_active == 1) return;
  const int64_t slot0 = (static_cast<int64_t>(at.b) * p.n_kv_heads + at.kvh) * p.max_splits;
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    int* tk = p.ws_ticket + (static_cast<int64_t>(at.b) * p.n_kv_heads + at.kvh) * p.row_blocks + at.blk;
    const bool last = atomicAdd(tk, 1) == at.n_active - 1;
    if (last) *tk = 0;
    *flag = last;
  }
  __syncthreads();
  if (!*flag || warp >= kMmaWarp) return;
  __threadfence();
  const float2* ml = reinterpret_cast<const float2*>(p.ws_ml);
  float* wgt = reinterpret_cast<float*>(smem + Sh::k);  // [rows][kKv8MaxSplits] weights / sum of the splits
  constexpr int per_warp = (RT + kMmaWarp - 1) / kMmaWarp;
  constexpr int per_lane = kKv8MaxSplits / 32;
  // A split's softmax sum is y 2^x from its own reference x: with y = f 2^e, 1 <= f < 2, the splits' shares go by x + e, and its
  // O is stored times 2^-e.
  auto weights = [&](int r, float2 (&x)[per_lane]) {
    float M = -INFINITY, sum = 0.f;
    int e[per_lane];
#pragma unroll
    for (int k = 0; k < per_lane; ++k) {
      e[k] = sum_exp(x[k].y);
      M = fmaxf(M, x[k].x + static_cast<float>(e[k]));
    }
    M = warp_max(M);
    if (M == -INFINITY) M = 0.f;
#pragma unroll
    for (int k = 0; k < per_lane; ++k) {
      x[k].x = ex2_approx((x[k].x - M) + static_cast<float>(e[k]));
      sum += x[k].x * (x[k].y * exp2i(-e[k]));
    }
    sum = warp_sum(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int k = 0; k < per_lane; ++k)
      if (lane + 32 * k < at.n_active) wgt[r * kKv8MaxSplits + lane + 32 * k] = x[k].x * inv;
  };
#pragma unroll
  for (int u0 = 0; u0 < per_warp; u0 += 2) {  // two rows' loads at a time
    float2 x[2][per_lane];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = warp + (u0 + u) * kMmaWarp;
#pragma unroll
      for (int k = 0; k < per_lane; ++k) {
        const int s2 = lane + 32 * k;
        x[u][k] = r < at.R && s2 < at.n_active ? __ldcg(ml + (slot0 + s2) * R_all + at.r0 + r) : make_float2(-INFINITY, 0.f);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (warp + (u0 + u) * kMmaWarp < at.R) weights(warp + (u0 + u) * kMmaWarp, x[u]);
  }
  named_sync(1, kSoft);
  auto store4 = [&](int it, float4 a) {
    const int r = at.r0 + (it >> 5);
    const int g = r / p.K, j = r - g * p.K;
    uint2 pk;
    pk.x = pack_bf16(a.x, a.y);
    pk.y = pack_bf16(a.z, a.w);
    *reinterpret_cast<uint2*>(p.out + ((static_cast<int64_t>(at.b) * p.K + j) * p.n_q_heads + at.kvh * G + g) * 128 +
                              (it & 31) * 4) = pk;
  };
  auto add = [&](float4& a, int it, int s2) {
    const float4 v = __ldcg(reinterpret_cast<const float4*>(p.ws_o + ((slot0 + s2) * R_all + at.r0 + (it >> 5)) * 128) +
                            (it & 31));
    const float w = wgt[(it >> 5) * kKv8MaxSplits + s2];
    a.x += w * v.x;
    a.y += w * v.y;
    a.z += w * v.z;
    a.w += w * v.w;
  };
  if (at.R * 32 * 2 <= kSoft) {
    // one or two rows: the splits are shared between the threads, too
    const int parts = kSoft / (at.R * 32), it = tid % (at.R * 32), part = tid / (at.R * 32);
    float4* pool = reinterpret_cast<float4*>(smem + Sh::v);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (part < parts) {
#pragma unroll 8
      for (int s2 = part; s2 < at.n_active; s2 += parts) add(a, it, s2);
    }
    pool[tid] = a;
    named_sync(1, kSoft);
    if (part == 0) {
      for (int k = 1; k < parts; ++k) {
        const float4 v = pool[k * at.R * 32 + it];
        a.x += v.x;
        a.y += v.y;
        a.z += v.z;
        a.w += v.w;
      }
      store4(it, a);
    }
    return;
  }
  for (int it0 = tid; it0 < at.R * 32; it0 += 4 * kSoft) {  // four (row, 4 dims) items' loads at a time
    float4 a[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int s2 = 0; s2 < at.n_active; ++s2) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (it0 + u * kSoft < at.R * 32) add(a[u], it0 + u * kSoft, s2);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (it0 + u * kSoft < at.R * 32) store4(it0 + u * kSoft, a[u]);
  }
}

size_t kv8_attention_ws_bytes(int bs, int rows, int n_kv_heads, int max_splits, size_t* o_off, size_t* ml_off) {
  const size_t n = static_cast<size_t>(bs) * n_kv_heads * max_splits * rows;
  if (o_off) *o_off = kQTicketBytes;
  if (ml_off) *ml_off = kQTicketBytes + n * 512;
  return kQTicketBytes + n * 520;
}

// Row blocks of a head: at least as many as keep kQMaxRows, at most `room` (CTAs that are to spare) down to 8 rows, as even as
// possible.  A block reads the cache again, from L2: for few CTAs that costs less than a long softmax and one CTA's join
// (one request of 3,000 tokens, 34 rows in 4 blocks: 15 us, in one 20).
void kv8_attention_blocks(int rows, int64_t room, int* blocks, int* per_block) {
  const int64_t least = (rows + kQMaxRows - 1) / kQMaxRows, most = (rows + 7) / 8;
  *blocks = static_cast<int>(std::max(least, std::min(room, most)));
  *per_block = (rows + *blocks - 1) / *blocks;
  *blocks = (rows + *per_block - 1) / *per_block;
}

template <int FMT, int RH, int H>
static cudaError_t launch_kv8_attention_t(const CUtensorMap& tmk, const CUtensorMap& tmv, const KvAttnParams& p,
                                          cudaStream_t stream, bool pdl) {
  auto kern = kv8_attention_kernel<FMT, RH, H>;
  using Sh = KvAttnShape<FMT, RH, H>;
  static PerDeviceOnce configured;
  cudaError_t e = once_per_device(configured, [&] {
    cudaError_t r = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::bytes);
    if (r != cudaSuccess) return r;
    return cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.n_kv_heads * p.row_blocks, p.bs, p.max_splits);
  cfg.blockDim = dim3(Sh::threads);
  cfg.dynamicSmemBytes = Sh::bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, tmk, tmv, p);
}
template <int FMT>
static cudaError_t launch_kv8_attention_f(const CUtensorMap& tmk, const CUtensorMap& tmv, const KvAttnParams& p,
                                          cudaStream_t stream, bool pdl) {
  // Two groups halve a thread's share of a tile's chain, but an SM then holds two CTAs, not three.  Up to 8 rows they are
  // for few CTAs (one request of 16,000 tokens, 8 rows: 18 us, one group 20; of 131,071, 2 rows: 50, 52) and one group for
  // many (64 requests of 288-4,128, 8 rows: 59 us, two groups 64; 2 rows: 53).  From 9 rows on two are better everywhere (16
  // rows: 74 us, one group 77).  A group has the rows of the next size up, 2 x 12, 17 or 20 (24 rows: 74 us, as 2 x 20 100;
  // 34 rows: 95, 105).
  if (p.rows_per_block <= 4)
    return p.few ? launch_kv8_attention_t<FMT, 2, 2>(tmk, tmv, p, stream, pdl)
                 : launch_kv8_attention_t<FMT, 4, 1>(tmk, tmv, p, stream, pdl);
  if (p.rows_per_block <= 8)
    return p.few ? launch_kv8_attention_t<FMT, 4, 2>(tmk, tmv, p, stream, pdl)
                 : launch_kv8_attention_t<FMT, 8, 1>(tmk, tmv, p, stream, pdl);
  if (p.rows_per_block <= 16) return launch_kv8_attention_t<FMT, 8, 2>(tmk, tmv, p, stream, pdl);
  if (p.rows_per_block <= 24) return launch_kv8_attention_t<FMT, 12, 2>(tmk, tmv, p, stream, pdl);
  if (p.rows_per_block <= 34) return launch_kv8_attention_t<FMT, 17, 2>(tmk, tmv, p, stream, pdl);
  return launch_kv8_attention_t<FMT, kQMaxRows / 2, 2>(tmk, tmv, p, stream, pdl);
}

cudaError_t launch_kv8_attention(const CUtensorMap& tmk, const CUtensorMap& tmv, const KvAttnParams& p, int format,
                                 cudaStream_t stream, bool pdl) {
  return format == GR_KV_E4M3 ? launch_kv8_attention_f<GR_KV_E4M3>(tmk, tmv, p, stream, pdl)
                              : launch_kv8_attention_f<GR_KV_INT8>(tmk, tmv, p, stream, pdl);
}

}  // namespace gr
